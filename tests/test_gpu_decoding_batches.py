"""Batches of more sequences and key heads than one launch's grid holds."""
import numpy as np
import pytest

import mtorch_b200 as mt
from test_gpu_decoding import U, attention_ref, heads, host, i32, path_of, quantised, rounded

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,path", [("bfloat16", "split"), ("float16", "split"), ("float32", "rows")])
@pytest.mark.parametrize("B,Hkv,Sk", [(70000, 1, 5), (33000, 4, 3), (65536, 1, 40)])
def test_window_attention_of_a_large_batch(B, Hkv, Sk, dtype, path):
    rng = np.random.default_rng(B)
    H, D = 2 * Hkv, 8
    q, qv = heads(rng, B, H, 1, D, dtype)
    k, kv = heads(rng, B, Hkv, Sk, D, dtype)
    v, vv = heads(rng, B, Hkv, Sk, D, dtype)
    lengths = rng.integers(0, Sk + 1, B)
    assert path_of(q, k, v, 4, 1) == path
    got = host(mt.window_attention(q, k, v, 4, 1, starts=i32(lengths - 1), lengths=i32(lengths)))
    per = 65535 // Hkv
    some = np.unique(np.r_[0, np.minimum([per - 1, per, per + 1, 2 * per - 1, 2 * per], B - 1), B - 1, rng.integers(0, B, 200)])
    want = attention_ref(qv[some], kv[some], vv[some], lengths[some] - 1, lengths[some], 4, 1, True)
    np.testing.assert_allclose(got[some], want, rtol=2 * U[dtype], atol=(2 * U[dtype] + 1e-4) * np.abs(vv).max())
    assert np.isfinite(got).all()


def test_cache_of_a_large_batch():
    rng = np.random.default_rng(1)
    B, H, Hkv, D, page = 66000, 2, 1, 64, 16
    cache = mt.KVCache4.empty(B, page, Hkv, D)
    table = rng.permutation(B).reshape(B, 1)
    k, kv = heads(rng, B, Hkv, 3, D, "bfloat16")
    v, vv = heads(rng, B, Hkv, 3, D, "bfloat16")
    starts = rng.integers(0, page - 3, B)
    mt.kv_cache_append(cache, k, v, i32(table), i32(starts))
    gk, gv = mt.kv_cache_read(cache, i32(table), i32(starts), 3, dtype="float32")
    np.testing.assert_allclose(host(gk), quantised(kv), rtol=2.0 ** -23, atol=1e-6)
    np.testing.assert_allclose(host(gv), quantised(vv), rtol=2.0 ** -23, atol=1e-6)
    q, qv = heads(rng, B, H, 1, D, "bfloat16")
    got = host(mt.kv_cache_attention(q, cache, i32(table), i32(starts + 3), window=3))
    some = np.unique(np.r_[0, 65534, 65535, 65536, B - 1, rng.integers(0, B, 200)])
    want = attention_ref(qv[some], quantised(kv[some]), quantised(vv[some]), [2] * len(some), [3] * len(some), 3, 0, True)
    np.testing.assert_allclose(got[some], want, rtol=2.0 ** -8, atol=(2.0 ** -8 + 1e-4) * 5)
    assert np.isfinite(got).all()
