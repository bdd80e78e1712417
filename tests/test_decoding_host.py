"""The decoder's operators refuse what they cannot take (checked on the host, before any launch)."""
import ctypes as C

import numpy as np
import pytest

import mtorch_b200 as mt
from mtorch_b200 import _lib as L


def test_cpu_tensors_are_refused():
    x = mt.randn(1, 2, 3, 8)
    pos = mt.tensor(np.zeros((1, 3), np.int32), dtype="int32")
    with pytest.raises(NotImplementedError):
        mt.rotary_embedding(x, None, pos, mt.randn(4), (4,))
    with pytest.raises(NotImplementedError):
        mt.window_attention(x, x, x, 4)
    with pytest.raises(NotImplementedError):
        mt.Weight4.pack(mt.randn(4, 4))
    with pytest.raises(NotImplementedError):
        mt.KVCache4(x, x, x, x)


def status(fn, *args):
    rc = fn(*args)
    return rc, L.lib().mt_cuda_last_error_string().decode()


def test_rotary_descriptor_errors():
    f = L.lib().mt_cuda_rotary

    def desc(**kw):
        d = L.RotaryDesc(1, 4, 8, 2, 0, L.MT_F32, 0, 0, 1, 4, (4, 0, 0, 0), 16, 4, 4, 16, 16, (64, 8, 16, 1), 16,
                         (64, 8, 16, 1))
        for k, v in kw.items():
            setattr(d, k, v)
        return C.byref(d)

    assert f(None, None) == L.MT_ERR_INVALID
    assert status(f, desc(axes=5), None)[0] == L.MT_ERR_INVALID
    assert status(f, desc(axes=0), None)[0] == L.MT_ERR_INVALID
    assert "pairs" in status(f, desc(pairs=5, axis_end=(5, 0, 0, 0)), None)[1]
    assert status(f, desc(axis_end=(3, 0, 0, 0)), None)[0] == L.MT_ERR_INVALID
    assert status(f, desc(axes=2, axis_end=(4, 2, 0, 0)), None)[0] == L.MT_ERR_INVALID
    assert status(f, desc(q=None), None)[0] == L.MT_ERR_INVALID
    assert status(f, desc(positions=None), None)[0] == L.MT_ERR_INVALID
    assert status(f, desc(dtype=L.MT_I64), None)[0] == L.MT_ERR_UNSUPPORTED
    assert status(f, desc(D=-1), None)[0] == L.MT_ERR_INVALID
    assert f(desc(B=0, q=None), None) == L.MT_OK


def window_desc(**kw):
    st = (4096, 64, 64, 1)
    d = L.WindowAttentionDesc(1, 4, 2, 16, 16, 64, L.MT_BF16, 1, 8, 0, None, None, 16, st, 16, st, 16, st, 16, st, 0.125)
    for k, v in kw.items():
        setattr(d, k, v)
    return C.byref(d)


def test_window_attention_descriptor_errors():
    f = L.lib().mt_cuda_window_attention
    assert f(None, None, 0, None) == L.MT_ERR_INVALID
    for kw in (dict(H=3), dict(window=-1), dict(sinks=-1), dict(D=0), dict(Sq=-1), dict(q=None), dict(k=None),
               dict(scale=float("nan")), dict(Hkv=0)):
        assert f(window_desc(**kw), None, 0, None) == L.MT_ERR_INVALID, kw
    for kw in (dict(D=257), dict(dtype=L.MT_F64), dict(Sk=1 << 40)):
        assert f(window_desc(**kw), None, 0, None) == L.MT_ERR_UNSUPPORTED, kw
    assert f(window_desc(Sq=0, q=None), None, 0, None) == L.MT_OK
    # one query over many keys is split over CTAs and needs a workspace
    d = window_desc(Sq=1, Sk=8192, window=0)
    need = L.lib().mt_cuda_window_attention_workspace_size(d)
    assert need > 0
    assert f(d, None, 0, None) == L.MT_ERR_WORKSPACE


def test_cache_descriptor_errors():
    lib = L.lib()
    st = L.I64_4(64, 64, 64, 1)

    def cache(**kw):
        c = L.KvCache4Desc(4, 16, 2, 64, 16, 16, 16, 16)
        for k, v in kw.items():
            setattr(c, k, v)
        return c

    def append(c, dtype=L.MT_BF16, B=1, starts=16):
        return lib.mt_cuda_kv_cache4_append(C.byref(c), 16, st, 16, st, dtype, B, 1, 16, 4, 4, starts, None)

    for kw in (dict(page_size=8), dict(page_size=24), dict(page_size=2048), dict(D=32), dict(D=100), dict(D=320),
               dict(k_words=None), dict(v_scales=24)):
        assert append(cache(**kw)) == L.MT_ERR_INVALID, kw
    assert append(cache(), dtype=L.MT_I32) == L.MT_ERR_UNSUPPORTED
    assert append(cache(), B=-1) == L.MT_ERR_INVALID
    assert append(cache(), starts=None) == L.MT_ERR_INVALID
    assert append(cache(), B=0) == L.MT_OK

    def attend(dtype=L.MT_BF16, ws=None, **kw):
        d = L.KvCache4AttentionDesc(cache(), 1, 4, 1, dtype, 0, 0, 16, 4, 4, 16, 16, st, 16, st, 0.125)
        for k, v in kw.items():
            setattr(d, k, v)
        return lib.mt_cuda_kv_cache4_attention(C.byref(d), ws, 0, None)

    assert attend(dtype=L.MT_F32) == L.MT_ERR_UNSUPPORTED
    assert attend(H=3) == L.MT_ERR_INVALID
    assert attend(lengths=None) == L.MT_ERR_INVALID
    assert attend(max_pages=-1) == L.MT_ERR_INVALID
    assert attend(max_pages=1024, num_pages=4) == L.MT_ERR_WORKSPACE
    assert attend(B=0) == L.MT_OK


def test_linear_weight4_descriptor_errors():
    f = L.lib().mt_cuda_linear_weight4

    def desc(**kw):
        d = L.LinearWeight4Desc(1, 8, 128, 64, L.MT_BF16, 16, 128, 16, 16, None, 16, 8)
        for k, v in kw.items():
            setattr(d, k, v)
        return C.byref(d)

    assert f(None, None, 0, None) == L.MT_ERR_INVALID
    for kw in (dict(group=16), dict(M=-1), dict(K=-1), dict(x=None), dict(y=None), dict(words=8)):
        assert f(desc(**kw), None, 0, None) == L.MT_ERR_INVALID, kw
    assert f(desc(dtype=L.MT_F64), None, 0, None) == L.MT_ERR_UNSUPPORTED
    assert f(desc(M=0, x=None), None, 0, None) == L.MT_OK
    assert L.lib().mt_cuda_weight4_pack(16, 16, None, L.MT_BF16, 128, 8, 128, 64, None) == L.MT_ERR_INVALID


@pytest.mark.gpu
def test_python_refusals():
    def z(*s, dtype="bfloat16"):
        return mt.zeros(*s, dtype=dtype, device="cuda")

    def idx(*s):
        return mt.zeros(*s, dtype="int32", device="cuda")

    q, k = z(2, 4, 3, 64), z(2, 2, 9, 64)
    freq = mt.rotary_frequencies((8, 8))
    for call, err in [
        (lambda: mt.rotary_embedding(q, z(2, 2, 4, 64), idx(2, 3), freq, (8, 8)), ValueError),
        (lambda: mt.rotary_embedding(q, z(2, 2, 3, 64, dtype="float16"), idx(2, 3), freq, (8, 8)), RuntimeError),
        (lambda: mt.rotary_embedding(q, None, idx(3, 3), freq, (8, 8)), ValueError),
        (lambda: mt.rotary_embedding(q, None, z(2, 3), freq, (8, 8)), ValueError),
        (lambda: mt.rotary_embedding(q, None, idx(2, 3), freq, (8, 30)), ValueError),
        (lambda: mt.rotary_embedding(q, None, idx(2, 3), freq, (8, 9)), ValueError),
        (lambda: mt.rotary_embedding(q, None, idx(2, 3), freq, (8, 8), out=z(2, 4, 3, 32)), RuntimeError),
        (lambda: mt.window_attention(q, k, k, 0), ValueError),
        (lambda: mt.window_attention(q, k, k, 4, -1), ValueError),
        (lambda: mt.window_attention(q, z(2, 3, 9, 64), z(2, 3, 9, 64), 4), ValueError),
        (lambda: mt.window_attention(q, k, z(2, 2, 8, 64), 4), ValueError),
        (lambda: mt.window_attention(q, k, k, 4, lengths=idx(3)), ValueError),
        (lambda: mt.window_attention(q, k, k, 4, starts=z(2)), ValueError),
        (lambda: mt.window_attention(q, k, k, 4, out=z(1, 4, 3, 64).expand(2, 4, 3, 64)), ValueError),
        (lambda: mt.window_attention(z(1, 1, 3, 300), z(1, 1, 3, 300), z(1, 1, 3, 300), 4), NotImplementedError),
        (lambda: mt.KVCache4.empty(4, 24, 2, 64), ValueError),
        (lambda: mt.KVCache4.empty(4, 16, 2, 96), ValueError),
        (lambda: mt.Weight4.pack(z(4, 4), 16), ValueError),
        (lambda: mt.Weight4(idx(4, 16), z(4, 3), 128), ValueError),
    ]:
        with pytest.raises(err):
            call()
    cache = mt.KVCache4.empty(4, 16, 2, 64)
    for call, err in [
        (lambda: mt.kv_cache_append(cache, z(2, 3, 1, 64), z(2, 3, 1, 64), idx(2, 2), idx(2)), ValueError),
        (lambda: mt.kv_cache_append(cache, z(2, 2, 1, 64), z(2, 2, 1, 64), idx(1, 2), idx(2)), ValueError),
        (lambda: mt.kv_cache_append(cache, z(2, 2, 1, 64), z(2, 2, 1, 64), idx(2, 2), idx(1)), ValueError),
        (lambda: mt.kv_cache_read(cache, idx(2, 2), idx(2), 1, dtype="float64"), NotImplementedError),
        (lambda: mt.kv_cache_attention(z(2, 4, 1, 128), cache, idx(2, 2), idx(2)), ValueError),
        (lambda: mt.kv_cache_attention(z(2, 3, 1, 64), cache, idx(2, 2), idx(2)), ValueError),
        (lambda: mt.kv_cache_attention(z(2, 4, 1, 64, dtype="float32"), cache, idx(2, 2), idx(2)), NotImplementedError),
    ]:
        with pytest.raises(err):
            call()
    w = mt.Weight4.pack(z(8, 100))
    with pytest.raises(RuntimeError):
        mt.linear_weight4(z(1, 128), w)
    with pytest.raises(RuntimeError):
        mt.linear_weight4(z(1, 100), w, z(8, dtype="float16"))
    with pytest.raises(RuntimeError):
        mt.linear_weight4(z(1, 100), w, z(7))
