"""The decoder's operators on the GPU against plain 64-bit implementations.

Tolerances, derived from the formats (u = 2^-9 for bf16, 2^-12 for f16, 2^-25 for fp32 is half a step of
rounding; sums are fp32):
* rotary: one rounding of the result, and sine / cosine within 2 units of 2^-23 each: |x| + |y| <= 2 max|x|.
* attention: the probabilities are rounded to 16 bits (bf16 over the 4-bit cache for both types) and the
  result once more: |error| <= 2u sum(p |v|) <= 2u max|v|; fp32 scores of D products are off by at most D 2^-24
  sum|q k| scale, below 1e-4 here, and move the result by as much of max|v|.  Over the 4-bit cache the rounded
  factor is p * scale against codes of -8..7, so the bound takes 8 scale in the place of |v|.
* linear: a step of 16 products in fp32 is within 2^-22 of the running sum; 16-bit inputs multiply codes that
  are offset by 128, so a group of 128 columns is off by at most 8 * 2^-22 * 136 scale sum|x|, below
  2^-13 sum(|x| 8 scale); fp32 inputs (no offset) by K / 16 * 2^-22 sum|x w|, below 2^-13 sum|x w| for K <= 8192.
"""
import itertools

import numpy as np
import pytest

import mtorch_b200 as mt
from mtorch_b200 import _lib as L

pytestmark = pytest.mark.gpu

U = {"bfloat16": 2.0 ** -9, "float16": 2.0 ** -12, "float32": 2.0 ** -25}


def dev(a, dtype=None):
    t = mt.tensor(np.ascontiguousarray(a))
    return (t.to(dtype) if dtype is not None else t).cuda()


def rounded(a, dtype):
    """(device tensor of `dtype`, its values in 64 bits)"""
    t = mt.tensor(np.ascontiguousarray(a, np.float32), dtype=dtype)
    return t.cuda(), t.numpy().astype(np.float64)


def i32(a):
    return mt.tensor(np.ascontiguousarray(a, dtype=np.int32), dtype="int32").cuda()


def host(t):
    return t.float().numpy().astype(np.float64) if t.dtype is not mt.float32 else t.numpy().astype(np.float64)


def heads(rng, b, h, s, d, dtype, merged=True, scale=1.0, extra=0):
    """A [b, h, s, d] device view (of merged rows [b, s, h * d + extra], or of [b, h, s, d + extra]) and its values."""
    if merged:
        t, v = rounded(rng.standard_normal((b, s, h * d + extra)) * scale, dtype)
        t = t._view((b, h, s, d), (s * (h * d + extra), d, h * d + extra, 1))
        return t, v[:, :, :h * d].reshape(b, s, h, d).transpose(0, 2, 1, 3)
    t, v = rounded(rng.standard_normal((b, h, s, d + extra)) * scale, dtype)
    return t[..., :d], v[..., :d]


# ---------------------------------------------------------------------------------------------
# rotary


def rotary_ref(x, positions, freq, sections, interleaved, inverse):
    y = x.copy()
    axis = np.repeat(np.arange(len(sections)), sections)
    P = sum(sections)
    for i in range(P):
        ang = (positions[axis[i]].astype(np.float32) * np.float32(freq[i])).astype(np.float64)
        if ang.ndim == 1:
            ang = ang[None]
        c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
        if inverse:
            s = -s
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + P)
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., a] * s + x[..., b] * c
    return y


ROTARY = [
    # B, Hq, Hk, S, D, sections, merged, extra
    (1, 1, 0, 1, 2, (1,), True, 0),
    (4, 12, 12, 1, 64, (8, 12, 12), True, 0),
    (2, 6, 2, 37, 64, (16, 16), True, 0),
    (2, 3, 1, 33, 80, (10, 10, 10), True, 0),
    (1, 2, 2, 130, 128, (16, 24, 24), False, 0),
    (1, 4, 4, 300, 128, (64,), True, 0),
    (2, 2, 1, 19, 40, (7, 6, 4), True, 0),
    (1, 3, 3, 21, 64, (20, 9), False, 3),
    (1, 2, 1, 9, 30, (5, 0, 2, 4), True, 1),
    (1, 2, 2, 16, 64, (0,), True, 0),
    (3, 48, 0, 65, 96, (24, 8, 8), True, 8),
]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", ROTARY)
def test_rotary(case, interleaved, dtype):
    B, Hq, Hk, S, D, sections, merged, extra = case
    rng = np.random.default_rng(S * 7 + D)
    q, qv = heads(rng, B, Hq, S, D, dtype, merged, extra=extra)
    k, kv = heads(rng, B, Hk, S, D, dtype, merged, extra=extra) if Hk else (None, None)
    pos = rng.integers(0, 3000, (len(sections), B, S)).astype(np.int32)
    freq = mt.rotary_frequencies(sections)
    fv = freq.numpy()
    for inverse in (False, True):
        got = mt.rotary_embedding(q, k, i32(pos), freq, sections, interleaved=interleaved, inverse=inverse)
        pairs = [(got, qv)] if k is None else [(got[0], qv), (got[1], kv)]
        for g, v in pairs:
            want = rotary_ref(v, pos, fv, sections, interleaved, inverse)
            np.testing.assert_allclose(host(g), want, rtol=2 * U[dtype], atol=2.0 ** -21 * 2 * np.abs(v).max())


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_in_place_back_and_shared_positions(interleaved):
    """Turned in place and back again gives the input up to two roundings; positions [axes, S] hold for the
    whole batch; the ladder may be shared between the axes."""
    rng = np.random.default_rng(5)
    B, H, S, D, sections = 2, 4, 50, 64, (8, 16, 8)
    q, qv = heads(rng, B, H, S, D, "float32")
    pos = rng.integers(0, 100, (3, S)).astype(np.int32)
    freq = mt.rotary_frequencies(sections, theta=500.0, shared=True)
    assert freq.numpy()[1] == np.float32(500.0 ** (-1 / 32))
    r = mt.rotary_embedding(q, None, i32(pos), freq, sections, interleaved=interleaved, out=q)
    assert r is q
    want = rotary_ref(qv, pos, freq.numpy(), sections, interleaved, False)
    np.testing.assert_allclose(host(q), want, rtol=2.0 ** -23, atol=2.0 ** -20 * np.abs(qv).max())
    mt.rotary_embedding(q, None, i32(pos), freq, sections, interleaved=interleaved, inverse=True, out=q)
    np.testing.assert_allclose(host(q), qv, rtol=2.0 ** -22, atol=2.0 ** -19 * np.abs(qv).max())


def test_rotary_inverse_is_the_gradient():
    """d/dx sum(g * rotary(x)) by differences in 64 bits equals the inverse turn of g."""
    rng = np.random.default_rng(6)
    sections = (5, 3)
    x, g = rng.standard_normal((1, 1, 3, 20)), rng.standard_normal((1, 1, 3, 20))
    pos = rng.integers(0, 50, (2, 3)).astype(np.int32)
    freq = mt.rotary_frequencies(sections)
    gt, gv = rounded(g, "float32")
    got = host(mt.rotary_embedding(gt, None, i32(pos), freq, sections, inverse=True))
    num = np.zeros_like(x)
    for i in np.ndindex(*x.shape):
        e = np.zeros_like(x)
        e[i] = 0.5
        num[i] = (gv * (rotary_ref(x + e, pos, freq.numpy(), sections, False, False)
                        - rotary_ref(x - e, pos, freq.numpy(), sections, False, False))).sum()
    np.testing.assert_allclose(got, num, rtol=0, atol=2.0 ** -20 * np.abs(gv).max())


# ---------------------------------------------------------------------------------------------
# attention with a window and sinks


def sees(p, j, n, window, sinks, causal):
    near = np.ones(np.broadcast(p, j).shape, bool) if window is None else (p - j < window)
    if not causal and window is not None:
        near &= j - p < window
    ok = near | (j < sinks)
    if causal:
        ok &= j <= p
    return ok & (j < n)


def attention_ref(q, k, v, starts, lengths, window, sinks, causal, scale=None):
    B, H, Sq, D = q.shape
    g = H // k.shape[1]
    scale = 1 / np.sqrt(D) if scale is None else scale
    o = np.zeros(q.shape)
    for b, h in itertools.product(range(B), range(H)):
        p = (starts[b] + np.arange(Sq))[:, None]
        m = sees(p, np.arange(k.shape[2])[None], lengths[b], window, sinks, causal)
        kk = np.where(np.arange(k.shape[2])[:, None] < lengths[b], k[b, h // g], 0)
        vv = np.where(np.arange(k.shape[2])[:, None] < lengths[b], v[b, h // g], 0)
        s = np.where(m, q[b, h] @ kk.T * scale, -np.inf)
        top = s.max(1, keepdims=True, initial=-np.inf)
        e = np.where(m, np.exp(s - np.where(np.isinf(top), 0, top)), 0)
        total = e.sum(1, keepdims=True)
        o[b, h] = np.where(total > 0, e @ vv / np.where(total > 0, total, 1), 0)
    return o


def attention_close(got, want, dtype, vmax):
    np.testing.assert_allclose(host(got), want, rtol=2 * U[dtype], atol=(2 * U[dtype] + 1e-4) * vmax)


WINDOW = [
    # B, H, Hkv, Sq, Sk, D, window, sinks, causal
    (1, 1, 1, 1, 1, 8, 1, 0, True),
    (2, 4, 2, 1, 77, 64, 20, 3, True),
    (1, 8, 1, 1, 300, 128, None, 0, True),
    (2, 12, 4, 3, 131, 64, 17, 40, True),
    (1, 3, 3, 8, 1000, 80, 200, 4, True),
    (3, 2, 1, 1, 2100, 40, 1500, 33, True),
    (1, 2, 2, 77, 77, 64, 16, 2, True),
    (2, 4, 2, 129, 129, 128, 50, 0, True),
    (1, 4, 4, 257, 515, 64, 130, 200, True),
    (1, 2, 1, 300, 300, 128, None, 0, True),
    (1, 2, 1, 640, 640, 128, 128, 5, True),
    (1, 2, 2, 200, 333, 64, 31, 7, False),
    (2, 3, 1, 130, 260, 96, None, 0, False),
    (1, 2, 2, 400, 150, 64, 40, 3, True),  # queries before the first key see nothing
    (1, 2, 2, 260, 260, 160, 100, 1, True),
    (1, 1, 1, 140, 140, 256, 33, 0, True),
    (1, 2, 1, 500, 900, 128, 1, 0, True),
]


PATHS = {1: "tc", 2: "split", 3: "tiles", 4: "rows"}


def path_of(q, k, v, window, sinks, causal=True, scale=0.125):
    B, H, Sq, D = q.shape
    return PATHS[L.lib().mt_cuda_window_attention_path(L.pack_window_attention(
        B, H, k.shape[1], Sq, k.shape[2], D, q.dtype.code, causal, window or 0, sinks, 0, 0, q.data_ptr(), *q.stride(),
        k.data_ptr(), *k.stride(), v.data_ptr(), *v.stride(), q.data_ptr(), *q.stride(), scale))]


# many heads and queries: the tensor-core tiles for 16-bit types, the fp32 tiles
LARGE = [
    # B, H, Hkv, Sq, Sk, D, window, sinks, causal
    (1, 32, 32, 257, 257, 64, 100, 5, True),
    (2, 24, 12, 300, 300, 128, 33, 0, True),
    (1, 64, 8, 513, 640, 128, 300, 140, True),
    (1, 48, 16, 400, 400, 40, None, 0, True),
    (2, 32, 32, 129, 500, 80, 64, 3, False),
    (1, 64, 64, 384, 384, 64, 1, 0, True),
    (1, 64, 64, 700, 300, 64, 90, 2, True),  # queries before the first key see nothing
    (3, 30, 10, 260, 131, 96, None, 7, False),
]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("case", LARGE)
def test_window_attention_of_many_queries(case, dtype):
    B, H, Hkv, Sq, Sk, D, window, sinks, causal = case
    rng = np.random.default_rng(Sq * 3 + Sk)
    q, qv = heads(rng, B, H, Sq, D, dtype)
    k, kv = heads(rng, B, Hkv, Sk, D, dtype)
    v, vv = heads(rng, B, Hkv, Sk, D, dtype, merged=False, extra=8)
    assert path_of(q, k, v, window, sinks, causal) == ("tiles" if dtype == "float32" else "tc")
    got = mt.window_attention(q, k, v, window, sinks, causal=causal)
    want = attention_ref(qv, kv, vv, [Sk - Sq] * B, [Sk] * B, window, sinks, causal)
    attention_close(got, want, dtype, np.abs(vv).max())


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("D", [64, 128])
def test_window_attention_of_many_queries_ragged(D, dtype):
    """A padded batch: what stands past the lengths is NaN and infinity; scores that grow with the key (the running
    maximum is raised in every tile) and an out= view that takes no vector stores."""
    rng = np.random.default_rng(D)
    B, H, Hkv, S, window, sinks = 6, 16, 8, 330, 150, 9
    lengths = np.array([S, 0, 1, 129, 128, 200])
    starts = np.zeros(B, np.int64)
    q, qv = heads(rng, B, H, S, D, dtype)
    kn, vn = rng.standard_normal((B, Hkv, S, D)), rng.standard_normal((B, Hkv, S, D))
    kn += np.arange(S)[:, None] * 0.05
    for b in range(B):
        kn[b, :, lengths[b]:] = np.nan
        vn[b, :, lengths[b]:] = [np.nan, np.inf, -np.inf, np.nan, 3, np.inf][b]
    k, kv = rounded(kn, dtype)
    v, vv = rounded(vn, dtype)
    assert path_of(q, k, v, window, sinks) == ("tiles" if dtype == "float32" else "tc")
    store = mt.zeros(B, S, H * D + 3, dtype=dtype, device="cuda")
    out = store._view((B, H, S, D), (S * (H * D + 3), D, H * D + 3, 1))
    mt.window_attention(q, k, v, window, sinks, starts=i32(starts), lengths=i32(lengths), out=out)
    want = attention_ref(qv, kv, vv, starts, lengths, window, sinks, True)
    # keys of up to 16: the fp32 scores of D products of up to 60 move the result by up to 1e-3
    np.testing.assert_allclose(host(out), want, rtol=2 * U[dtype], atol=(2 * U[dtype] + 1e-3) * 5.0)
    assert (host(store)[..., H * D:] == 0).all()


def test_window_attention_paths():
    """Few queries take the split keys, unaligned rows and a negative scale the others."""
    rng = np.random.default_rng(0)
    q, _ = heads(rng, 1, 4, 1, 64, "bfloat16")
    k, _ = heads(rng, 1, 2, 100, 64, "bfloat16")
    assert path_of(q, k, k, 10, 0) == "split"
    odd, _ = heads(rng, 1, 2, 100, 64, "bfloat16", extra=1)
    assert path_of(q, odd, odd, 10, 0) == "rows"
    q, _ = heads(rng, 2, 64, 300, 64, "bfloat16")
    k, _ = heads(rng, 2, 64, 300, 64, "bfloat16")
    assert path_of(q, k, k, 100, 0) == "tc"
    assert path_of(q, k, k, 100, 0, scale=-1.0) == "split"
    odd, _ = heads(rng, 2, 64, 300, 64, "bfloat16", extra=1)
    assert path_of(q, odd, odd, 100, 0) == "tiles"


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("case", WINDOW)
def test_window_attention(case, dtype):
    B, H, Hkv, Sq, Sk, D, window, sinks, causal = case
    rng = np.random.default_rng(Sq * 3 + Sk)
    q, qv = heads(rng, B, H, Sq, D, dtype)
    k, kv = heads(rng, B, Hkv, Sk, D, dtype)
    v, vv = heads(rng, B, Hkv, Sk, D, dtype, merged=False)
    got = mt.window_attention(q, k, v, window, sinks, causal=causal)
    want = attention_ref(qv, kv, vv, [Sk - Sq] * B, [Sk] * B, window, sinks, causal)
    attention_close(got, want, dtype, np.abs(vv).max())


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("Sq,Sk,D", [(1, 200, 64), (2, 500, 128), (300, 300, 64), (140, 420, 128)])
def test_window_attention_ragged(Sq, Sk, D, dtype):
    """Lengths of zero, one and all keys; what stands past them is NaN and infinity."""
    rng = np.random.default_rng(Sq + Sk)
    B, H, Hkv, window, sinks = 5, 4, 2, 60, 6
    lengths = np.array([Sk, 0, 1, Sk // 2 + 1, 63 if Sk > 63 else 1])
    starts = np.array([0] * B if Sq == Sk else np.maximum(lengths - Sq, -3))
    q, qv = heads(rng, B, H, Sq, D, dtype)
    kn, vn = rng.standard_normal((B, Hkv, Sk, D)), rng.standard_normal((B, Hkv, Sk, D))
    for b in range(B):
        kn[b, :, lengths[b]:] = np.nan
        vn[b, :, lengths[b]:] = [np.nan, np.inf, -np.inf, np.nan, 3][b]
    k, kv = rounded(kn, dtype)
    v, vv = rounded(vn, dtype)
    for causal in (True, False):
        got = mt.window_attention(q, k, v, window, sinks, causal=causal, starts=i32(starts), lengths=i32(lengths))
        want = attention_ref(qv, kv, vv, starts, lengths, window, sinks, causal)
        attention_close(got, want, dtype, 5.0)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("Sq", [1, 200])
def test_window_attention_strides_scale_and_large_scores(Sq, dtype):
    """Head dims that are not contiguous or not aligned, a negative scale, scores far apart, out= a view."""
    rng = np.random.default_rng(Sq)
    B, H, Hkv, Sk, D = 1, 4, 2, 260, 64
    qn, kn, vn = (rng.standard_normal((B, h, s, D)) * 6 for h, s in ((H, Sq), (Hkv, Sk), (Hkv, Sk)))
    qt, qv = rounded(qn.transpose(0, 1, 3, 2), dtype)  # tokens innermost
    k, kv = rounded(np.pad(kn, ((0, 0), (0, 0), (0, 0), (1, 2))), dtype)  # rows that start off alignment
    v, vv = rounded(vn, dtype)
    store = mt.zeros(B, Sq, H * D + 5, dtype=dtype, device="cuda")
    out = store._view((B, H, Sq, D), (Sq * (H * D + 5), D, H * D + 5, 1))
    for scale in (0.3, -0.2):
        got = mt.window_attention(qt.transpose(2, 3), k[..., 1:65], v, 100, 3, scale=scale, out=out)
        assert got is out
        want = attention_ref(qv.transpose(0, 1, 3, 2), kv[..., 1:65], vv, [Sk - Sq], [Sk], 100, 3, True, scale)
        # scores of some hundreds: their fp32 rounding (D products of up to 600) moves exp by up to 1e-3
        np.testing.assert_allclose(host(got), want, rtol=2 * U[dtype], atol=(2 * U[dtype] + 2e-3) * np.abs(vv).max())


# ---------------------------------------------------------------------------------------------
# the 4-bit cache


def quantised(x):
    """Values that the cache holds for x [..., D], by its definition."""
    x = x.astype(np.float32)
    g = x.reshape(x.shape[:-1] + (-1, 64))
    lo, hi = g.min(-1), g.max(-1)
    zero = np.clip(lo, -65504, 65504).astype(np.float16).astype(np.float32)
    scale = np.minimum((hi - lo) * np.float32(1 / 15), np.float32(65504)).astype(np.float16).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        code = np.where(scale[..., None] > 0, np.clip(np.rint((g - zero[..., None]) / scale[..., None]), 0, 15), 0)
    return (zero[..., None].astype(np.float64) + code * scale[..., None].astype(np.float64)).reshape(x.shape)


def filled_cache(rng, B, heads_, page, per, D, spare=2):
    cache = mt.KVCache4.empty(B * per + spare, page, heads_, D)
    table = rng.permutation(B * per + spare)[:B * per].reshape(B, per).astype(np.int32)
    level = rng.standard_normal((2, heads_, 1, D))
    k = rng.standard_normal((B, heads_, page * per, D)) + level[0]
    v = rng.standard_normal((B, heads_, page * per, D)) + level[1]
    kt, kv = rounded(k, "float32")
    vt, vv = rounded(v, "float32")
    mt.kv_cache_append(cache, kt, vt, i32(table), i32(np.zeros(B)))
    return cache, table, quantised(kv), quantised(vv)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("B,H,T,D,page,per", [(1, 1, 1, 64, 16, 2), (3, 2, 45, 128, 16, 4), (2, 3, 100, 192, 64, 3),
                                              (1, 2, 33, 256, 1024, 1)])
def test_cache_append_and_read(B, H, T, D, page, per, dtype):
    rng = np.random.default_rng(T)
    cache = mt.KVCache4.empty(B * per, page, H, D)
    table = rng.permutation(B * per).reshape(B, per).astype(np.int32)
    starts = rng.integers(0, page * per - T + 1, B)
    k, kv = heads(rng, B, H, T, D, dtype)
    v, vv = heads(rng, B, H, T, D, dtype, merged=False, extra=1)
    mt.kv_cache_append(cache, k, v, i32(table), i32(starts))
    gk, gv = mt.kv_cache_read(cache, i32(table), i32(starts), T, dtype=dtype)
    for got, x in ((gk, kv), (gv, vv)):
        want = quantised(x)
        np.testing.assert_allclose(host(got), want, rtol=2 * U[dtype], atol=1e-6)
        step = (x.reshape(B, H, T, -1, 64).max(-1) - x.reshape(B, H, T, -1, 64).min(-1)) / 15
        assert (np.abs(want - x).reshape(B, H, T, -1, 64) <= 0.51 * step[..., None] + 2e-3).all()
    # nothing else was written: the token before the first is still zero
    if starts.max() > 0:
        b = int(starts.argmax())
        gk, _ = mt.kv_cache_read(cache, i32(table), i32(np.maximum(starts - 1, 0)), 1)
        assert (host(gk)[b] == 0).all()


def test_cache_places_that_do_not_exist():
    """Tokens before zero, past the table and on pages that are not there: unwritten, read as zero, unseen."""
    rng = np.random.default_rng(9)
    B, H, D, page = 2, 2, 64, 16
    cache, table, kq, vq = filled_cache(rng, B, H, page, 4, D)
    before = [t.numpy().copy() for t in (cache.k_words, cache.k_scales, cache.v_words, cache.v_scales)]
    bad = table.copy()
    bad[0, 1], bad[1, 2] = -1, cache.num_pages
    x = dev(np.full((B, H, 16, D), 7.0, np.float32) * rng.standard_normal((1, 1, 16, D)).astype(np.float32))
    mt.kv_cache_append(cache, x, x, i32(bad), i32([16, 32]))     # exactly the pages that are not there
    mt.kv_cache_append(cache, x, x, i32(table), i32([-16, 64]))  # before the first, past the last token
    for t, was in zip((cache.k_words, cache.k_scales, cache.v_words, cache.v_scales), before):
        np.testing.assert_array_equal(t.numpy(), was)
    gk, gv = mt.kv_cache_read(cache, i32(bad), i32([8, 24]), 24, dtype="float32")
    want = np.stack([kq[0, :, 8:32], kq[1, :, 24:48]])
    want[0, :, 8:24] = 0
    want[1, :, 8:24] = 0
    np.testing.assert_allclose(host(gk), want, rtol=2.0 ** -23, atol=1e-6)
    # attention: the missing pages' tokens are not seen
    q, qv = heads(rng, B, 4, 1, D, "bfloat16")
    got = host(mt.kv_cache_attention(q, cache, i32(bad), i32([60, 64])))
    gone = [np.r_[16:32], np.r_[32:48]]
    for b, n in enumerate((60, 64)):
        keep = np.setdiff1d(np.arange(n), gone[b])
        want = attention_ref(qv[b:b + 1], kq[b:b + 1][:, :, keep], vq[b:b + 1][:, :, keep], [len(keep) - 1],
                             [len(keep)], None, 0, True)
        np.testing.assert_allclose(got[b:b + 1], want, rtol=2.0 ** -8, atol=(2.0 ** -8 + 1e-4) * 10)


CACHE = [
    # H, Hkv, Sq, D, page, per, window, sinks
    (1, 1, 1, 64, 16, 1, None, 0),
    (4, 2, 1, 64, 16, 9, None, 0),
    (8, 1, 1, 128, 32, 7, None, 0),
    (16, 2, 1, 128, 64, 5, 100, 4),
    (6, 2, 4, 64, 16, 20, 50, 20),
    (12, 1, 3, 128, 16, 6, 33, 0),
    (4, 4, 1, 256, 128, 2, None, 0),
    (3, 1, 2, 192, 16, 5, 7, 3),
    (2, 2, 40, 64, 32, 4, 30, 5),
    (4, 2, 1, 128, 128, 20, 1900, 17),
    (32, 1, 1, 64, 16, 4, None, 0),
]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("case", CACHE)
def test_cache_attention(case, dtype):
    H, Hkv, Sq, D, page, per, window, sinks = case
    rng = np.random.default_rng(H * 5 + D + per)
    B = 4
    cache, table, kq, vq = filled_cache(rng, B, Hkv, page, per, D)
    cap = page * per
    lengths = np.array([cap, 0, min(Sq, cap) // 2 + 1, max(1, cap - page // 2 - 1)])
    q, qv = heads(rng, B, H, Sq, D, dtype)
    got = mt.kv_cache_attention(q, cache, i32(table), i32(lengths), window=window, sinks=sinks)
    want = attention_ref(qv, kq, vq, lengths - Sq, lengths, window, sinks, True)
    # 8 scale <= 8 / 15 of a range of at most about 9
    np.testing.assert_allclose(host(got), want, rtol=2 * U[dtype], atol=(2.0 ** -8 + 1e-4) * max(np.abs(vq).max(), 5))


def test_cache_attention_reads_no_pages_outside_the_window():
    """Table entries of tokens that no query sees may be anything, scales of unused slots too."""
    rng = np.random.default_rng(3)
    H, D, page, per, window, sinks = 2, 64, 16, 12, 40, 10
    cache, table, kq, vq = filled_cache(rng, 1, H, page, per, D)
    n = 150  # sees 110..149 and 0..9: pages 0 and 6..9
    bad = table.copy()
    bad[0, 1:6], bad[0, 10:] = 2 ** 30, -5
    sc = cache.v_scales.numpy()
    sc[table[0, 9], :, n % page:] = np.nan  # slots of the last page past the sequence
    cache.v_scales.copy_(mt.tensor(sc, dtype="float16"))
    cache.k_scales.copy_(mt.tensor(np.where(np.isnan(sc), np.inf, cache.k_scales.numpy()), dtype="float16"))
    q, qv = heads(rng, 1, 4, 1, D, "bfloat16")
    got = mt.kv_cache_attention(q, cache, i32(bad), i32([n]), window=window, sinks=sinks)
    want = attention_ref(qv, kq, vq, [n - 1], [n], window, sinks, True)
    np.testing.assert_allclose(host(got), want, rtol=2.0 ** -8, atol=(2.0 ** -8 + 1e-4) * 10)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("H,Sq", [(2, 1), (6, 2), (10, 3)])
@pytest.mark.parametrize("per,D", [(5, 64), (14, 128), (23, 192), (32, 256), (40, 128)])
def test_few_sequences_over_several_chunks_of_keys(per, D, H, Sq, dtype):
    """2 to 9 and more chunks a sequence, of which short sequences leave some or all empty; one call's bits are the next's."""
    rng = np.random.default_rng(per + H)
    B, Hkv, page = 3, 2, 64
    cap = per * page
    lengths = np.array([cap - 7, 0, Sq + 19])
    cache, table, kq, vq = filled_cache(rng, B, Hkv, page, per, D)
    q, qv = heads(rng, B, H, Sq, D, dtype)
    for window, sinks in ((None, 0), (cap // 2, 9)):
        got = mt.kv_cache_attention(q, cache, i32(table), i32(lengths), window=window, sinks=sinks)
        want = attention_ref(qv, kq, vq, lengths - Sq, lengths, window, sinks, True)
        np.testing.assert_allclose(host(got), want, rtol=2 * U[dtype], atol=(2.0 ** -8 + 1e-4) * max(np.abs(vq).max(), 5))
        again = mt.kv_cache_attention(q, cache, i32(table), i32(lengths), window=window, sinks=sinks)
        np.testing.assert_array_equal(host(got), host(again))
    d = D - 24 if D < 256 else D  # channels that end inside a block of 64
    q, qv = heads(rng, B, H, Sq, d, dtype)
    k, kv = heads(rng, B, Hkv, cap, d, dtype)
    v, vv = heads(rng, B, Hkv, cap, d, dtype)
    for window, sinks in ((cap, 0), (cap // 2, 9)):
        got = mt.window_attention(q, k, v, window, sinks, starts=i32(lengths - Sq), lengths=i32(lengths))
        want = attention_ref(qv, kv, vv, lengths - Sq, lengths, window, sinks, True)
        attention_close(got, want, dtype, 5.0)
        again = mt.window_attention(q, k, v, window, sinks, starts=i32(lengths - Sq), lengths=i32(lengths))
        np.testing.assert_array_equal(host(got), host(again))


# ---------------------------------------------------------------------------------------------
# 4-bit weights


def linear_bound(x, w, dtype, y):
    mag = np.abs(x) @ np.abs(w).T if dtype == "float32" else np.abs(x) @ np.full((x.shape[1], w.shape[0]), np.abs(w).max() * 8 / 7)
    return 2 * U[dtype] * np.abs(y) + 2.0 ** -13 * mag


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("M,N,K,group", [(1, 1, 1, 32), (1, 17, 128, 128), (2, 64, 200, 64), (3, 100, 768, 32),
                                         (8, 48, 1000, 128), (9, 33, 640, 64), (16, 130, 129, 32), (31, 70, 300, 128),
                                         (40, 96, 512, 32), (130, 257, 520, 64), (1, 4100, 2050, 64),
                                         (5, 300, 8192, 128)])
def test_linear_weight4(M, N, K, group, dtype):
    rng = np.random.default_rng(N + K)
    w, wv = rounded(rng.standard_normal((N, K)) / np.sqrt(K), "float32")
    p = mt.Weight4.pack(w, group)
    back = host(p.unpack("float32"))
    Kp = (K + group - 1) // group * group
    pad = np.pad(wv.astype(np.float32), ((0, 0), (0, Kp - K))).reshape(N, -1, group)
    top = np.abs(pad).max(-1)
    scale = mt.tensor(top * np.float32(1 / 7)).to("bfloat16").numpy()
    want = (np.clip(np.rint(pad / np.where(scale > 0, scale, 1)[..., None]), -8, 7) * scale[..., None]).reshape(N, -1)[:, :K]
    np.testing.assert_array_equal(back, want)
    x, xv = rounded(rng.standard_normal((M, K)), dtype)
    bias, bv = rounded(rng.standard_normal(N), dtype)
    for bb, add in ((bias, bv), (None, 0.0)):
        y = xv @ back.T + add
        err = np.abs(host(mt.linear_weight4(x, p, bb)) - y)
        assert (err <= linear_bound(xv, back, dtype, y) + 2.0 ** -22 * np.abs(add)).all(), err.max()


@pytest.mark.parametrize("dtype,power", [("float16", -11), ("float16", -16), ("float16", -22), ("float16", 9),
                                         ("bfloat16", -40), ("bfloat16", 40), ("float32", -40), ("float32", 40)])
@pytest.mark.parametrize("M", [1, 13])
def test_linear_weight4_of_small_and_large_rows(M, dtype, power):
    """Rows whose values all lie near 2^power (f16: down to its subnormals) lose nothing to the operands' scaling."""
    rng = np.random.default_rng(power & 63)
    N, K = 70, 96
    p = mt.Weight4.pack(dev(rng.standard_normal((N, K)) * 2.0 ** (-power // 2), "float32"), 32)
    w = host(p.unpack("float32"))
    x, xv = rounded(rng.standard_normal((M, K)) * 2.0 ** power, dtype)
    y = xv @ w.T
    err = np.abs(host(mt.linear_weight4(x, p)) - y)
    floor = 2.0 ** -25 if dtype == "float16" else 0  # half of f16's smallest number
    assert (err <= linear_bound(xv, w, dtype, y) + floor).all(), err.max()


def test_linear_weight4_views():
    """Rows with a pitch, leading dims, out= a view, columns past K that hold anything."""
    rng = np.random.default_rng(1)
    N, K = 40, 200
    p = mt.Weight4.pack(dev(rng.standard_normal((N, K)), "bfloat16"), 64)
    w = host(p.unpack("float32"))
    wide, wv = rounded(np.where(np.arange(260) < K, rng.standard_normal((6, 260)), np.nan), "bfloat16")
    out = mt.zeros(6, 64, dtype="bfloat16", device="cuda")
    mt.linear_weight4(wide[:, :K], p, out=out[:, 3:3 + N])
    got = host(out)
    y = wv[:, :K] @ w.T
    assert (np.abs(got[:, 3:43] - y) <= linear_bound(wv[:, :K], w, "bfloat16", y)).all()
    assert (got[:, :3] == 0).all() and (got[:, 43:] == 0).all()
    z = mt.linear_weight4(wide[:, :K].reshape(2, 3, K), p)
    np.testing.assert_array_equal(host(z).reshape(6, N), got[:, 3:43])
    assert mt.linear_weight4(wide[:0, :K], p).shape == (0, N)


# ---------------------------------------------------------------------------------------------
# sizes of zero, tables and offsets past 32 bits


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_sizes_of_zero(dtype):
    rng = np.random.default_rng(0)
    q, _ = heads(rng, 2, 4, 3, 64, dtype)
    none = mt.zeros(2, 2, 0, 64, dtype=dtype, device="cuda")
    for Sq in (3, 0):
        o = mt.window_attention(q[:, :, :Sq], none, none, 5, 2)
        assert o.shape == (2, 4, Sq, 64) and (host(o) == 0).all()
    many, _ = heads(rng, 1, 64, 300, 64, dtype)
    o = mt.window_attention(many, none[:1], none[:1], 5, 2)
    assert (host(o) == 0).all()
    freq = mt.rotary_frequencies((4,))
    r = mt.rotary_embedding(q[:, :, :0], None, mt.zeros(1, 0, dtype="int32", device="cuda"), freq, (4,))
    assert r.shape == (2, 4, 0, 64)
    cache = mt.KVCache4.empty(2, 16, 2, 64)
    table, zero = i32([[0], [1]]), i32([0, 0])
    mt.kv_cache_append(cache, none, none, table, zero)
    k, v = mt.kv_cache_read(cache, table, zero, 0)
    assert k.shape == (2, 2, 0, 64)
    if dtype == "bfloat16":
        assert (host(mt.kv_cache_attention(q, cache, table, zero)) == 0).all()
        empty = mt.zeros(2, 0, dtype="int32", device="cuda")  # a table of no pages
        assert (host(mt.kv_cache_attention(q, cache, empty, i32([5, 7]))) == 0).all()


def test_table_with_a_row_pitch_and_shared_pages():
    """Two sequences share their first pages (a forked prompt); the table is a view of a wider one."""
    rng = np.random.default_rng(2)
    H, D, page = 2, 128, 16
    cache = mt.KVCache4.empty(8, page, H, D)
    wide = np.full((2, 9), 77, np.int32)
    wide[:, 1:5] = [[0, 1, 2, 3], [0, 1, 4, 5]]
    table = i32(wide)[:, 1:5]
    k, kv = rounded(rng.standard_normal((2, H, 64, D)), "bfloat16")
    v, vv = rounded(rng.standard_normal((2, H, 64, D)), "bfloat16")
    mt.kv_cache_append(cache, k[:1, :, :32], v[:1, :, :32], table[:1], i32([0]))       # the shared prompt
    mt.kv_cache_append(cache, k[:, :, 32:], v[:, :, 32:], table, i32([32, 32]))         # what follows, apart
    kq, vq = quantised(kv), quantised(vv)
    kq[1, :, :32], vq[1, :, :32] = kq[0, :, :32], vq[0, :, :32]
    q, qv = heads(rng, 2, 8, 1, D, "bfloat16")
    got = mt.kv_cache_attention(q, cache, table, i32([64, 50]))
    want = attention_ref(qv, kq, vq, [63, 49], [64, 50], None, 0, True)
    np.testing.assert_allclose(host(got), want, rtol=2.0 ** -8, atol=(2.0 ** -8 + 1e-4) * 5)


def test_cache_past_32_bits():
    """A page whose words begin 4.3 GB into the arrays."""
    rng = np.random.default_rng(4)
    page, D, pages = 1024, 256, 33000  # 128 bytes a token: 4.3e9 bytes of words each for K and V
    words = [mt.empty(pages, 1, page, D // 8, dtype="int32", device="cuda") for _ in range(2)]
    scales = [mt.empty(pages, 1, page, D // 64, 2, dtype="float16", device="cuda") for _ in range(2)]
    cache = mt.KVCache4(words[0], scales[0], words[1], scales[1])
    table = i32([[pages - 1, pages - 2]])
    k, kv = rounded(rng.standard_normal((1, 1, 1100, D)), "bfloat16")
    v, vv = rounded(rng.standard_normal((1, 1, 1100, D)), "bfloat16")
    mt.kv_cache_append(cache, k, v, table, i32([0]))
    gk, gv = mt.kv_cache_read(cache, table, i32([1000]), 100, dtype="float32")
    np.testing.assert_allclose(host(gk), quantised(kv)[:, :, 1000:], rtol=2.0 ** -23, atol=1e-6)
    np.testing.assert_allclose(host(gv), quantised(vv)[:, :, 1000:], rtol=2.0 ** -23, atol=1e-6)
    q, qv = heads(rng, 1, 2, 1, D, "bfloat16")
    got = mt.kv_cache_attention(q, cache, table, i32([1100]))
    want = attention_ref(qv, quantised(kv), quantised(vv), [1099], [1100], None, 0, True)
    np.testing.assert_allclose(host(got), want, rtol=2.0 ** -8, atol=(2.0 ** -8 + 1e-4) * 5)


@pytest.mark.parametrize("Sq,H", [(1, 4), (300, 64)])
def test_strides_past_32_bits(Sq, H):
    """Sequences that lie 2^31 elements apart in one buffer."""
    rng = np.random.default_rng(Sq)
    S, D, far = 320, 64, (1 << 31) + 64
    buf = mt.empty(far + H * S * D, dtype="bfloat16", device="cuda")
    q, qv = heads(rng, 2, H, Sq, D, "bfloat16")
    k, kv = rounded(rng.standard_normal((2, H, S, D)), "bfloat16")
    view = buf._view((2, H, S, D), (far, S * D, D, 1))
    view.copy_(k)
    got = mt.window_attention(q, view, view, 100, 3)
    want = attention_ref(qv, kv, kv, [S - Sq] * 2, [S] * 2, 100, 3, True)
    attention_close(got, want, "bfloat16", np.abs(kv).max())
    freq = mt.rotary_frequencies((16, 16))
    pos = rng.integers(0, 500, (2, S)).astype(np.int32)
    mt.rotary_embedding(view, None, i32(pos), freq, (16, 16), out=view)
    want = rotary_ref(kv, pos, freq.numpy(), (16, 16), False, False)
    np.testing.assert_allclose(host(view[1:]), want[1:], rtol=2 * U["bfloat16"], atol=2.0 ** -20 * np.abs(kv).max())
