"""What stands where it must not count, and what must not get lost: values at hidden keys, NaN, infinities, very large and
very small numbers in the decoder's operators, against 64-bit references.

The forms of `window_attention` are reached by shape and type: "tc" and "tiles" by many queries, "split" and "rows" by few
(`path_of` asserts which).
"""
import ctypes as C

import numpy as np
import pytest

import mtorch_b200 as mt
from mtorch_b200 import _lib as L
from test_gpu_decoding import U, attention_ref, heads, host, i32, path_of, quantised, rounded

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


@pytest.mark.parametrize("what", ["nan query", "nan key", "nan keys", "infinite score"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("form,dtype,H,Hkv,Sq,Sk", FORMS)
def test_nan_is_not_lost(form, dtype, H, Hkv, Sq, Sk, D, what):
    """A query whose scores hold a NaN, or an infinity (whose difference with itself is one), gives NaN; others do not."""
    rng = np.random.default_rng(Sq + D)
    window, sinks = 90, 2
    qn, kn = rng.standard_normal((1, H, Sq, D)), rng.standard_normal((1, Hkv, Sk, D))
    p = Sk - Sq + np.arange(Sq)
    qn[..., 7] = np.abs(qn[..., 7]) + 1
    hit = np.zeros((H, Sq), bool)
    group = np.arange(H) * Hkv // H  # key head of a head
    if what == "nan query":
        qn[0, 1, Sq // 2, 3] = np.nan
        hit[1, Sq // 2] = True
    else:
        at = {"nan key": [242], "nan keys": list(range(Sk)), "infinite score": [243]}[what]
        kn[0, -1, at, 7] = np.inf if what == "infinite score" else np.nan
        sees = np.array([any(a <= i and (i - a < window or a < sinks) for a in at) for i in p])
        hit[group == Hkv - 1] = sees
    q, qv = rounded(qn, dtype)
    k, kv = rounded(kn, dtype)
    v, vv = heads(rng, 1, Hkv, Sk, D, dtype)
    assert path_of(q, k, v, window, sinks) == form
    got = host(mt.window_attention(q, k, v, window, sinks))[0]
    assert np.isnan(got[hit]).all() and hit.any()
    with np.errstate(invalid="ignore"):
        want = attention_ref(qv, np.where(np.isfinite(kv), kv, 0), vv, [Sk - Sq], [Sk], window, sinks, True)[0]
    np.testing.assert_allclose(got[~hit], want[~hit], rtol=2 * U[dtype], atol=(2 * U[dtype] + 1e-4) * 5)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("form,dtype,H,Hkv,Sq,Sk", FORMS)
def test_scores_of_minus_infinity_weigh_nothing(form, dtype, H, Hkv, Sq, Sk, D):
    """Keys whose scores are -infinity count as hidden ones, the first that a query sees among them; a query that sees no
    others gets zeros."""
    rng = np.random.default_rng(Sq + D)
    window = 30
    qn, kn = rng.standard_normal((1, H, Sq, D)), rng.standard_normal((1, Hkv, Sk, D))
    qn[..., 5] = np.abs(qn[..., 5]) + 1
    gone = np.zeros(Sk, bool)
    gone[[0, 1, 100]] = gone[Sk - 5:Sk - 2] = gone[Sk - 34:Sk - 20] = True
    kn[:, :, gone, 5] = -np.inf
    q, qv = rounded(qn, dtype)
    k, kv = rounded(kn, dtype)
    v, vv = heads(rng, 1, Hkv, Sk, D, dtype)
    assert path_of(q, k, v, window, 0) == form
    got = host(mt.window_attention(q, k, v, window, 0))
    want = attention_ref(qv, kv, vv, [Sk - Sq], [Sk], window, 0, True)
    assert Sq < Sk or (want[:, :, :2] == 0).all()
    np.testing.assert_allclose(got, want, rtol=2 * U[dtype], atol=(2 * U[dtype] + 1e-4) * 5)


def filled(rng, B, Hkv, page, per, D):
    """A cache of random keys and values and what it holds, read back: [B, Hkv, page * per, D]."""
    cache = mt.KVCache4.empty(B * per, page, Hkv, D)
    table = i32(rng.permutation(B * per).reshape(B, per))
    k, _ = rounded(rng.standard_normal((B, Hkv, page * per, D)) + rng.standard_normal((Hkv, 1, D)), "float32")
    v, _ = rounded(rng.standard_normal((B, Hkv, page * per, D)) + rng.standard_normal((Hkv, 1, D)), "float32")
    zero = i32(np.zeros(B))
    mt.kv_cache_append(cache, k, v, table, zero)
    kq, vq = mt.kv_cache_read(cache, table, zero, page * per, dtype="float32")
    return cache, table, host(kq), host(vq)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("B,H,Hkv,Sq,Sk,D", [(1, 4, 1, 1, 6000, 64), (1, 8, 2, 2, 900, 128), (24, 16, 8, 1, 3000, 128)])
def test_nan_is_not_lost_in_the_join(B, H, Hkv, Sq, Sk, D, dtype):
    """A query of NaN over keys that are split over CTAs (joined in a cluster, or by a second kernel), and a chunk of keys
    of which all are NaN."""
    rng = np.random.default_rng(Sk)
    qn = rng.standard_normal((B, H, Sq, D))
    qn[0, 1] = np.nan
    kn = rng.standard_normal((B, Hkv, Sk, D))
    q, qv = rounded(qn, dtype)
    k, kv = rounded(kn, dtype)
    v, vv = heads(rng, B, Hkv, Sk, D, dtype)
    assert path_of(q, k, v, None, 0) == ("rows" if dtype == "float32" else "split")
    want = attention_ref(np.nan_to_num(qv), kv, vv, [Sk - Sq] * B, [Sk] * B, None, 0, True)
    got = host(mt.window_attention(q, k, v, None))
    assert np.isnan(got[0, 1]).all()
    got[0, 1], want[0, 1] = 0, 0
    np.testing.assert_allclose(got, want, rtol=2 * U[dtype], atol=(2 * U[dtype] + 1e-4) * 5)
    kn[0, 0, :Sk // 2] = np.nan
    k, _ = rounded(kn, dtype)
    got = host(mt.window_attention(q, k, v, None))
    assert np.isnan(got[0, :H // Hkv]).all() and np.isfinite(got[0, max(2, H // Hkv):]).all()
    if dtype != "float32":
        cache, table, kq, vq = filled(rng, B, Hkv, 64, (Sk + 63) // 64, D)
        lengths = np.full(B, Sk)
        got = host(mt.kv_cache_attention(q, cache, table, i32(lengths)))
        assert np.isnan(got[0, 1]).all()
        want = attention_ref(np.nan_to_num(qv), kq, vq, lengths - Sq, lengths, None, 0, True)
        got[0, 1], want[0, 1] = 0, 0
        np.testing.assert_allclose(got, want, rtol=2 * U[dtype], atol=(2.0 ** -8 + 1e-4) * 8)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
def test_cache_keeps_nan_and_infinities(dtype):
    """Groups with a NaN, of NaN only, with infinities of one or both signs, of one infinity only, next to clean ones; a
    sequence that sees such keys gives NaN, another does not."""
    rng = np.random.default_rng(11)
    B, H, T, D = 2, 2, 40, 128
    x = rng.standard_normal((2, B, H, T, D))
    x[:, 0, 0, 3, 70] = np.nan
    x[:, 0, 0, 4, 64:] = np.nan
    x[:, 0, 1, 5, 9] = np.inf
    x[:, 0, 1, 6, 10] = -np.inf
    x[:, 0, 1, 7, [11, 60]] = [-np.inf, np.inf]
    x[:, 0, 1, 8, :64] = np.inf
    x[:, 0, 1, 9, :64] = -np.inf
    cache = mt.KVCache4.empty(2 * B, 32, H, D)
    table, zero = i32([[3, 1], [0, 2]]), i32([0, 0])
    k, kv = rounded(x[0], dtype)
    v, vv = rounded(x[1], dtype)
    mt.kv_cache_append(cache, k, v, table, zero)
    got = mt.kv_cache_read(cache, table, zero, T, dtype="float32")
    for g, a in zip(got, (kv, vv)):
        with np.errstate(invalid="ignore"):
            want = quantised(a)
        assert np.isnan(want[0, 0, 3, 64:]).all() and np.isnan(want[0, 1, 8, :64]).all() and np.isfinite(want[1]).all()
        np.testing.assert_allclose(host(g), want, rtol=2.0 ** -23, atol=1e-6)
    q, qv = heads(rng, B, 4, 1, D, "bfloat16")
    o = host(mt.kv_cache_attention(q, cache, table, i32([T, T])))
    assert np.isnan(o[0, :2]).all() and np.isfinite(o[1]).all()
    o = host(mt.kv_cache_attention(q, cache, table, i32([T, T]), window=20))  # (the window is past them)
    want = attention_ref(qv, quantised(np.nan_to_num(kv, posinf=0, neginf=0)), quantised(np.nan_to_num(vv, posinf=0, neginf=0)),
                         [T - 1] * 2, [T] * 2, 20, 0, True)
    np.testing.assert_allclose(o, want, rtol=2 * U["bfloat16"], atol=(2.0 ** -8 + 1e-4) * 5)


def cache_close(got, want, dtype, vmax):
    """Over the cache a bf16 query's weights times scale are rounded to bf16 once, 2^-9 against codes of -8..7 (8 scale in the
    place of |v|); an f16 query's carry the rounding's rest, which leaves 2^-18.  Scores move the result by at most 1e-4
    of |v| (fp32 sums of D products), the result is rounded to its type."""
    weights = 2.0 ** -8 if dtype == "bfloat16" else 2.0 ** -17
    np.testing.assert_allclose(got, want, rtol=2 * U[dtype], atol=(weights + 1e-4) * vmax)


@pytest.mark.parametrize("H,Hkv,Sq,D,page", [(4, 2, 1, 64, 16), (8, 2, 3, 128, 32), (2, 2, 1, 256, 16), (12, 1, 2, 64, 64)])
@pytest.mark.parametrize("dtype,power", [("bfloat16", 64), ("bfloat16", 90), ("bfloat16", 122), ("bfloat16", -60),
                                         ("bfloat16", -90), ("float16", -9), ("float16", -14), ("float16", -17),
                                         ("float16", -21), ("float16", 11)])
def test_cache_attention_of_small_and_large_queries(H, Hkv, Sq, D, page, dtype, power):
    """Queries near 2^power with a scale to match see what ordinary ones do; a head of them beside ordinary ones does too."""
    rng = np.random.default_rng(D + abs(power))
    B, per = 2, 6
    cache, table, kq, vq = filled(rng, B, Hkv, page, per, D)
    n = page * per
    lengths = np.array([n, n - 7])
    qn = rng.standard_normal((B, H, Sq, D)) * 2.0 ** power
    scale = 2.0 ** -power / np.sqrt(D)
    for mixed in (False, True):
        if mixed:
            qn[:, 0] *= 2.0 ** (-20 if power > 0 else 20)  # scores near 0, or far apart
        q, qv = rounded(qn, dtype)
        got = host(mt.kv_cache_attention(q, cache, table, i32(lengths), scale=scale))
        want = attention_ref(qv, kq, vq, lengths - Sq, lengths, None, 0, True, scale)
        if mixed and power < 0:
            got, want = got[:, 1:], want[:, 1:]  # (scores of millions: one key takes all, or two are within fp32's rounding)
        cache_close(got, want, dtype, max(np.abs(vq).max(), 5))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_cache_attention_of_an_infinite_query(dtype):
    """It gives NaN (infinity times a value of zero, or scores of both signs) and leaves the others alone."""
    rng = np.random.default_rng(8)
    cache, table, kq, vq = filled(rng, 1, 2, 32, 4, 64)
    qn = rng.standard_normal((1, 8, 2, 64))
    qn[0, 1, 0, 9], qn[0, 6, 1, 10] = np.inf, -np.inf
    q, qv = rounded(qn, dtype)
    got = host(mt.kv_cache_attention(q, cache, table, i32([128])))
    bad = ~np.isfinite(qv).all(-1)
    assert np.isnan(got[bad]).all() and bad.sum() == 2
    want = attention_ref(np.where(np.isfinite(qv), qv, 0), kq, vq, [126], [128], None, 0, True)
    cache_close(got[~bad], want[~bad], dtype, max(np.abs(vq).max(), 5))


def product_close(got, x, w, dtype, add=0.0):
    """Codes and 16-bit X multiply exactly; what is rounded are fp32 sums, of (code and 8) |x| scale <= 23 / 8 of the largest
    |w| of a row times |x| over at most 24 additions of a group and its products (2^-23 each, 2^-18 together), and the result
    to its type.  fp32 X goes in three parts that leave 2^-25."""
    y = x @ w.T + add
    mag = np.abs(x).sum(1)[:, None] * np.abs(w).max(1)[None] * (23 / 8)
    lim = 2 * U[dtype] * np.abs(y) + 2.0 ** -18 * mag + 2.0 ** -24 * np.abs(add) + (2.0 ** -25 if dtype == "float16" else 0)
    assert (np.abs(got - y) <= lim).all(), (np.abs(got - y) / lim).max()


@pytest.mark.parametrize("M,N,K,group", [(1, 70, 96, 32), (3, 2400, 520, 64), (13, 70, 1000, 128), (33, 40, 300, 64),
                                         (70, 40, 300, 64), (200, 130, 520, 32)])
@pytest.mark.parametrize("dtype,power", [("bfloat16", 64), ("bfloat16", 110), ("bfloat16", -70), ("float32", 64),
                                         ("float32", 100), ("float32", -35), ("float32", -60)])
def test_products_of_very_large_and_small_rows(M, N, K, group, dtype, power):
    """Rows near 2^power, alone and among ordinary ones (the weights' scales keep the results in range)."""
    rng = np.random.default_rng(M + abs(power))
    p = mt.Weight4.pack(rounded(rng.standard_normal((N, K)) * 2.0 ** (-power // 2), "float32")[0], group)
    w = host(p.unpack("float32"))
    xn = rng.standard_normal((M, K))
    xn[::2] *= 2.0 ** power
    x, xv = rounded(xn, dtype)
    product_close(host(mt.linear_weight4(x, p)), xv, w, dtype)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("M,N,K,group", [(1, 70, 96, 32), (3, 2400, 520, 64), (13, 70, 1000, 128), (33, 40, 300, 64),
                                         (70, 50, 300, 64)])
def test_products_of_infinities_and_nan(M, N, K, group, dtype):
    """As the definition has it: an infinity times a weight, NaN times a weight of zero and of infinities of both signs;
    the other rows do not notice."""
    rng = np.random.default_rng(M)
    p = mt.Weight4.pack(rounded(rng.standard_normal((N, K)), "float32")[0], group)
    w = host(p.unpack("float32"))
    xn = rng.standard_normal((M, K))
    rows = np.arange(M) % 4
    xn[rows == 0, 5] = np.inf
    xn[rows == 1, K - 1] = -np.inf
    xn[rows == 2, 7] = np.nan
    bias, bv = rounded(rng.standard_normal(N), dtype)
    x, xv = rounded(xn, dtype)
    got = host(mt.linear_weight4(x, p, bias))
    with np.errstate(invalid="ignore"):
        y = np.stack([(r[None] * w).sum(1) for r in xv]) + bv
    fine = np.isfinite(y)
    np.testing.assert_array_equal(got[~fine], y[~fine])
    if M > 3:
        assert fine.any() and np.isinf(y).any() and np.isnan(y).any()
        product_close(got[rows == 3], xv[rows == 3], w, dtype, bv)


@pytest.mark.parametrize("dtype,weights,rows", [("float16", -30, 12), ("float16", 18, -14), ("float16", 0, 0), ("bfloat16", -50, 0),
                                                ("bfloat16", 60, -20), ("bfloat16", 0, 0), ("float32", -30, 10),
                                                ("float32", 50, -20), ("float32", 0, 0)])
@pytest.mark.parametrize("N,K,group", [(130, 200, 32), (70, 1000, 128)])
def test_a_row_gives_the_same_in_a_prompt(N, K, group, dtype, weights, rows):
    """64 rows, the same and one more, and many: the weights enter exactly in all of them, with scales past f16's range and
    of many sizes too."""
    rng = np.random.default_rng(abs(weights) + N)
    wn = rng.standard_normal((N, K)) * 2.0 ** weights * 2.0 ** rng.integers(-6, 1, (N, 1))
    p = mt.Weight4.pack(rounded(wn, "float32")[0], group)
    w = host(p.unpack("float32"))
    x, xv = rounded(rng.standard_normal((300, K)) * 2.0 ** rows / np.sqrt(K), dtype)
    bias, bv = rounded(rng.standard_normal(N) * 2.0 ** (weights + rows), dtype)
    for M in (1, 64, 65, 300):
        product_close(host(mt.linear_weight4(x[:M], p, bias)), xv[:M], w, dtype, bv)
    same = mt.linear_weight4(x[:1].expand(150, K), p, bias)  # one row in memory
    product_close(host(same), np.repeat(xv[:1], 150, 0), w, dtype, bv)


def products_in_one_read(M, N, K, group, dtype):
    """Whether `linear_weight4` reads the packed weight itself (it needs no workspace then)."""
    code = mt.zeros(1, dtype=dtype).dtype.code
    d = L.LinearWeight4Desc(M, N, K, group, code, 16, K, 16, 16, None, 16, N)
    return L.lib().mt_cuda_linear_weight4_workspace_size(C.byref(d)) == 0


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("N,K,group", [(70, 768, 64), (40, 4096, 128), (33, 17000, 32), (20, 28672, 128)])
def test_products_on_both_sides_of_the_switch(N, K, group, dtype):
    """Where the copies take over from the packed weight, by type and columns; a few rows of a wide weight never go through
    them."""
    rows = [M for M in range(1, 200) if products_in_one_read(M, N, K, group, dtype)]
    last = rows[-1]
    assert rows == list(range(1, last + 1)) and 1 <= last < 199
    rng = np.random.default_rng(K)
    p = mt.Weight4.pack(rounded(rng.standard_normal((N, K)), "float32")[0], group)
    w = host(p.unpack("float32"))
    x, xv = rounded(rng.standard_normal((last + 1, K)) / np.sqrt(K), dtype)
    for M in {1, last, last + 1}:
        got = host(mt.linear_weight4(x[:M], p))
        y = xv[:M] @ w.T
        # (sums over more additions than product_close has: K / 16 of them within 2^-23 of the sum of |x w|)
        lim = 2 * U[dtype] * np.abs(y) + (2.0 ** -18 * 8 + K / 16 * 2.0 ** -23) * (np.abs(xv[:M]) @ np.abs(w).T)
        assert (np.abs(got - y) <= lim + (2.0 ** -25 if dtype == "float16" else 0)).all()
