"""What stands where it must not count, and what must not get lost: values at hidden keys, NaN, infinities, very large and
very small numbers in the decoder's operators, against 64-bit references.

The forms of `window_attention` are reached by shape and type: "tc" and "tiles" by many queries, "split" and "rows" by few
(`path_of` asserts which).
"""
import numpy as np
import pytest

import mtorch_b200 as mt
from test_gpu_decoding import U, attention_close, attention_ref, heads, host, i32, path_of, rounded

pytestmark = pytest.mark.gpu

# dtype, heads, key heads, queries, keys -> the kernel that takes it
FORMS = [
    ("tc", "bfloat16", 64, 64, 300, 300),
    ("tc", "float16", 64, 64, 300, 300),
    ("split", "bfloat16", 8, 2, 3, 300),
    ("split", "float16", 8, 2, 3, 300),
    ("tiles", "float32", 64, 64, 300, 300),
    ("rows", "float32", 4, 2, 3, 300),
]
LARGEST = {"bfloat16": 3.3895e38, "float16": 65504.0, "float32": 3.4028e38}


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("form,dtype,H,Hkv,Sq,Sk", FORMS)
def test_hidden_keys_count_nothing(form, dtype, H, Hkv, Sq, Sk, D):
    """The type's largest and lowest values in V at keys that a query does not see (behind it, or past its window)."""
    rng = np.random.default_rng(Sq + D)
    window = 40
    q, qv = heads(rng, 1, H, Sq, D, dtype)
    k, kv = heads(rng, 1, Hkv, Sk, D, dtype)
    vn = rng.standard_normal((1, Hkv, Sk, D))
    far = np.zeros(Sk, bool)
    far[96:104] = far[200:232] = True  # (in 300 queries over 300 keys: behind some of a tile, past the window of others)
    vn[:, :, far] = np.where(np.arange(D) % 2, LARGEST[dtype], -LARGEST[dtype])
    v, vv = rounded(vn, dtype)
    assert path_of(q, k, v, window, 0) == form
    got = host(mt.window_attention(q, k, v, window, 0))
    p = Sk - Sq + np.arange(Sq)
    clean = np.array([not far[max(0, i - window + 1):i + 1].any() for i in p])
    assert clean.any()
    want = attention_ref(qv, kv, np.where(far[:, None], 0, vv), [Sk - Sq], [Sk], window, 0, True)
    np.testing.assert_allclose(got[:, :, clean], want[:, :, clean], rtol=2 * U[dtype], atol=(2 * U[dtype] + 1e-4) * 5)
