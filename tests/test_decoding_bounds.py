"""Bounds of the decoder's operators that are near what their arithmetic gives, so that a lost part of it is seen.

u = 2^-9 for bf16, 2^-12 for f16, 2^-25 for fp32 (half a step of rounding).
* f16 queries over the 4-bit cache: the weights times scale go to bf16 in two parts, which leaves 2^-18 of them, against codes
  of -8..7: 2^-18 of 8 scale, below 2^-17 of the largest |v| (or 5) here; scores of fp32 sums move the result by at most 1e-4 of
  that; the result is rounded.
* 16-bit attention of few queries: the weights go to their 16-bit type in two parts, which leaves 2^-18 of them (bf16, less in
  f16): 2^-17 of the largest |v|, scores move the result by at most 1e-4 of it; the result is rounded.
* products of fp32 rows with 4-bit weights: X goes in three parts of 8 bits.  Where all of X lies between 1 and 2, the codes'
  sums of 16 products are whole multiples of 2^-23 below 2^9 in each part and exact in fp32 (a part has 8 bits, a code 4, 16 of them 4 more);
  what is rounded are the sums over groups (4 to a block of 128 columns), over blocks and the parts: below 8 roundings of 2^-24
  of sum |x w| for one block, 2^-21.
* the same for many rows: 1024 columns are 64 steps of an accumulator that drops what does not fit, 2^-23 each at most: 2^-17
  of sum |x w|, with a rounding of 2^-24 for each pass of 1024 columns.
* attention in fp32: scores of D products are off by at most D 2^-24 sum |q k| scale, an exponential by 2^-22, sums over n keys by n 2^-24:
  together (D sum|q k| scale + n + 8) 2^-24 of the largest |v|.

The tests without a GPU put the mistake into the reference: the bound has to see it.
"""
import itertools

import numpy as np
import pytest

import mtorch_b200 as mt
from test_gpu_decoding import U, attention_ref, filled_cache, heads, host, i32, path_of, quantised, rounded, sees

CACHE = [
    # H, Hkv, Sq, D, page, pages of a sequence, window, sinks
    (1, 1, 1, 64, 16, 1, None, 0),
    (4, 2, 1, 64, 16, 9, None, 0),
    (8, 1, 1, 128, 32, 7, None, 0),
    (16, 2, 1, 128, 64, 5, 100, 4),
    (6, 2, 4, 64, 16, 20, 50, 20),
    (12, 1, 3, 128, 16, 6, 33, 0),
    (3, 1, 2, 192, 16, 5, 7, 3),
    (2, 2, 40, 64, 32, 4, 30, 5),
]


def cache_limit(want, vq):
    return 2 * U["float16"] * np.abs(want) + (2.0 ** -17 + 1e-4) * max(np.abs(vq).max(), 5)


def bf16(a):
    return mt.tensor(np.ascontiguousarray(a, np.float32)).to("bfloat16").numpy().astype(np.float64).reshape(np.shape(a))


@pytest.mark.gpu
@pytest.mark.parametrize("case", CACHE)
def test_f16_queries_over_the_cache(case):
    H, Hkv, Sq, D, page, per, window, sinks = case
    rng = np.random.default_rng(H * 5 + D + per)
    B, cap = 3, page * per
    cache, table, kq, vq = filled_cache(rng, B, Hkv, page, per, D)
    lengths = np.array([cap, 0, max(1, cap - page // 2 - 1)])
    q, qv = heads(rng, B, H, Sq, D, "float16")
    got = host(mt.kv_cache_attention(q, cache, i32(table), i32(lengths), window=window, sinks=sinks))
    want = attention_ref(qv, kq, vq, lengths - Sq, lengths, window, sinks, True)
    assert (np.abs(got - want) <= cache_limit(want, vq)).all()


@pytest.mark.parametrize("parts", [1, 2])
@pytest.mark.parametrize("case", CACHE)
def test_the_cache_bound_sees_weights_of_one_part(case, parts):
    H, Hkv, Sq, D, page, per, window, sinks = case
    rng = np.random.default_rng(H * 5 + D + per)
    B, n = 2, page * per
    k = rng.standard_normal((B, Hkv, n, D)) + rng.standard_normal((Hkv, 1, D))
    v = rng.standard_normal((B, Hkv, n, D)) + rng.standard_normal((Hkv, 1, D))
    kq, vq = quantised(k), quantised(v)
    groups = v.astype(np.float32).reshape(B, Hkv, n, -1, 64)
    zero = groups.min(-1).astype(np.float16).astype(np.float64)
    scale = ((groups.max(-1) - groups.min(-1)) * np.float32(1 / 15)).astype(np.float16).astype(np.float64)
    code = np.rint((vq.reshape(groups.shape) - zero[..., None]) / scale[..., None])
    q = rng.standard_normal((B, H, Sq, D)).astype(np.float16).astype(np.float64)
    lengths = np.array([n, max(1, n - page // 2 - 1)])
    want = attention_ref(q, kq, vq, lengths - Sq, lengths, window, sinks, True)
    got = np.zeros_like(want)
    for b, h in itertools.product(range(B), range(H)):
        hk = h // (H // Hkv)
        m = sees((lengths[b] - Sq + np.arange(Sq))[:, None], np.arange(n)[None], lengths[b], window, sinks, True)
        s = np.where(m, q[b, h] @ kq[b, hk].T / np.sqrt(D), -np.inf)
        top = s.max(1, keepdims=True)
        e = np.exp(s - np.where(np.isinf(top), 0, top)) * m
        total = np.maximum(e.sum(1, keepdims=True), 1e-300)
        for g in range(D // 64):
            w = e * scale[b, hk, :, g]
            r = bf16(w)
            if parts == 2:
                r = r + bf16(w - r)
            rest = (e * (zero[b, hk, :, g] + 8 * scale[b, hk, :, g])).sum(1, keepdims=True)
            got[b, h][:, g * 64:(g + 1) * 64] = (r @ (code[b, hk, :, g] - 8) + rest) / total
    off = np.abs(got.astype(np.float16).astype(np.float64) - want) > cache_limit(want, vq)
    assert off.any() == (parts == 1)


SPLIT = [
    # dtype, H, Hkv, Sq, Sk, D, window
    ("bfloat16", 4, 2, 1, 60, 64, 5),
    ("bfloat16", 8, 1, 2, 300, 128, 12),
    ("bfloat16", 6, 2, 4, 900, 64, 900),
    ("bfloat16", 16, 2, 2, 500, 256, 8),
    ("float16", 4, 2, 1, 60, 64, 5),
    ("float16", 8, 1, 2, 300, 128, 12),
]


def split_limit(want, vv, dtype):
    return 2 * U[dtype] * np.abs(want) + (2.0 ** -17 + 1e-4) * np.abs(vv).max()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,H,Hkv,Sq,Sk,D,window", SPLIT)
def test_16_bit_attention_of_few_queries(dtype, H, Hkv, Sq, Sk, D, window):
    rng = np.random.default_rng(Sk + D)
    q, qv = heads(rng, 2, H, Sq, D, dtype)
    k, kv = heads(rng, 2, Hkv, Sk, D, dtype)
    v, vv = heads(rng, 2, Hkv, Sk, D, dtype)
    assert path_of(q, k, v, window, 0) == "split"
    got = host(mt.window_attention(q, k, v, window))
    want = attention_ref(qv, kv, vv, [Sk - Sq] * 2, [Sk] * 2, window, 0, True)
    assert (np.abs(got - want) <= split_limit(want, vv, dtype)).all()


@pytest.mark.parametrize("parts", [1, 2])
@pytest.mark.parametrize("dtype,H,Hkv,Sq,Sk,D,window", [c for c in SPLIT if c[0] == "bfloat16" and c[6] < 100])
def test_the_attention_bound_sees_weights_of_one_part(dtype, H, Hkv, Sq, Sk, D, window, parts):
    rng = np.random.default_rng(Sk + D)
    q, k, v = (bf16(rng.standard_normal((2, h, s, D))) for h, s in ((H, Sq), (Hkv, Sk), (Hkv, Sk)))
    want = attention_ref(q, k, v, [Sk - Sq] * 2, [Sk] * 2, window, 0, True)
    got = np.zeros_like(want)
    for b, h in itertools.product(range(2), range(H)):
        m = sees((Sk - Sq + np.arange(Sq))[:, None], np.arange(Sk)[None], Sk, window, 0, True)
        s = np.where(m, q[b, h] @ k[b, h * Hkv // H].T / np.sqrt(D), -np.inf)
        e = np.exp(s - s.max(1, keepdims=True))
        w = bf16(e)
        if parts == 2:
            w = w + bf16(e - w)
        got[b, h] = w @ v[b, h * Hkv // H] / e.sum(1, keepdims=True)
    off = np.abs(bf16(got) - want) > split_limit(want, v, dtype)
    assert off.any() == (parts == 1)


def product_inputs(M, N):
    """X of three parts each (1, 2^-9 and below 2^-17, all positive) and a weight of positive codes: what a lost part takes
    does not cancel."""
    rng = np.random.default_rng(M + N)
    x = 1 + 2.0 ** -9 + rng.integers(16, 64, (M, 128)) * 2.0 ** -23
    return x, np.abs(rng.standard_normal((N, 128))) + 0.5


def product_limit(x, w):
    return 2.0 ** -21 * (np.abs(x) @ np.abs(w).T)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N", [(1, 40), (7, 70), (20, 2400)])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_fp32_products_hold_fp32(M, N, group):
    x, w = product_inputs(M, N)
    p = mt.Weight4.pack(rounded(w, "float32")[0], group)
    wv = host(p.unpack("float32"))
    xt, xv = rounded(x, "float32")
    np.testing.assert_array_equal(xv, x)
    assert (np.abs(host(mt.linear_weight4(xt, p)) - xv @ wv.T) <= product_limit(xv, wv)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K,group", [(300, 130, 128, 64), (150, 70, 3449, 64), (100, 300, 8192, 128)])
def test_fp32_products_of_many_rows_hold_fp32(M, N, K, group):
    """All of one sign: what the accumulator drops does not cancel (without passes it grows to 2^-15 at 8192 columns)."""
    rng = np.random.default_rng(K)
    p = mt.Weight4.pack(rounded(np.abs(rng.standard_normal((N, K))) + 0.5, "float32")[0], group)
    w = host(p.unpack("float32"))
    x, xv = rounded(np.abs(rng.standard_normal((M, K))) + 0.5, "float32")
    bias, bv = rounded(rng.standard_normal(N), "float32")
    y = xv @ w.T
    got = host(mt.linear_weight4(x, p, bias))
    assert (np.abs(got - y - bv) <= (2.0 ** -17 + (K // 1024 + 3) * 2.0 ** -24) * y).all()


@pytest.mark.parametrize("parts", [1, 2, 3])
def test_the_product_bound_sees_every_part(parts):
    x, w = product_inputs(7, 70)
    s = bf16(w.max(1, keepdims=True) / 7)
    w = np.clip(np.rint(w / s), -8, 7) * s
    left, kept = x.copy(), np.zeros_like(x)
    for _ in range(parts):
        part = bf16(left)
        kept, left = kept + part, left - part
    off = np.abs(kept @ w.T - x @ w.T) > product_limit(x, w)
    assert off.all() == (parts < 3) and off.any() == (parts < 3)


@pytest.mark.gpu
@pytest.mark.parametrize("form,H,Hkv,Sq,Sk,D", [("tiles", 64, 64, 300, 300, 64), ("tiles", 64, 32, 200, 260, 128),
                                               ("rows", 4, 2, 3, 300, 64), ("rows", 4, 2, 1, 900, 128), ("rows", 2, 1, 40, 200, 40)])
def test_fp32_attention_holds_fp32(form, H, Hkv, Sq, Sk, D):
    rng = np.random.default_rng(Sq + D)
    window, sinks = 60, 4
    q, qv = heads(rng, 1, H, Sq, D, "float32", scale=0.2)
    k, kv = heads(rng, 1, Hkv, Sk, D, "float32")
    v, vv = heads(rng, 1, Hkv, Sk, D, "float32")
    assert path_of(q, k, v, window, sinks) == form
    got = host(mt.window_attention(q, k, v, window, sinks))
    want = attention_ref(qv, kv, vv, [Sk - Sq], [Sk], window, sinks, True)
    mass = (np.abs(qv) @ np.abs(np.repeat(kv, H // Hkv, 1)).swapaxes(-1, -2)).max() / np.sqrt(D)
    assert np.abs(got - want).max() <= (D * mass + window + sinks + 8) * 2.0 ** -24 * np.abs(vv).max()


@pytest.mark.gpu
def test_a_captured_projection_after_larger_calls():
    """A captured step with a projection by copies (its workspace is the largest of the calls) replays the same bits after
    other calls have used and outgrown the workspace."""
    from mtorch_b200.graphs import Graphed

    rng = np.random.default_rng(3)
    p = mt.Weight4.pack(rounded(rng.standard_normal((300, 520)), "float32")[0], 64)
    big = mt.Weight4.pack(rounded(rng.standard_normal((3000, 2048)), "float32")[0], 64)
    x, _ = rounded(rng.standard_normal((130, 520)), "bfloat16")
    y, _ = rounded(rng.standard_normal((700, 2048)), "bfloat16")
    want = host(mt.linear_weight4(x, p))
    g = Graphed(lambda t: mt.linear_weight4(t, p), x)
    first = host(mt.linear_weight4(y, big))
    np.testing.assert_array_equal(host(g(x)), want)
    np.testing.assert_array_equal(host(mt.linear_weight4(y, big)), first)
    np.testing.assert_array_equal(host(g(x)), want)
