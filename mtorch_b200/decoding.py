"""Operators of a causal decoder that runs beside the image path: rotary positions with several axes,
attention with a sliding window and sinks, a paged key / value cache held in 4 bits, and products
with weights held in 4 bits.  (The reference has none of them; they follow its conventions for
arguments, views and errors.)

Heads come as [batch, heads, tokens, dim] views with any strides, as `scaled_dot_product_attention`
takes them; `out=` takes any view of the right shape and writes the result there.
"""
from __future__ import annotations

import math

import numpy as np

from . import _lib as L
from .ops import _lib, _same_dtype
from .tensor import (_WS, Tensor, _new, _require_cuda, bfloat16, device as _device, float16, float32, int32, stream_ptr,
                     tensor, to_dtype, workspace, zeros)

CACHE_GROUP = 64  # channels of a head that share a scale and a zero point in KVCache4


# These calls take microseconds on the device, so what stands before them on the host is kept short: descriptors are
# packed at once (L.packer) and the shared workspace is asked for only when it is too small.


def _check(rc, what):
    if rc:
        L.check(rc, what)


def _ptr(t):
    return t._buf.ptr + t._offset * t.dtype.itemsize


def _run(fn, size_fn, desc, t, what):
    """fn(desc, workspace, its size, stream), with the device's workspace grown where it does not suffice."""
    idx = t.device.index or 0
    buf, stream = _WS.get(idx), stream_ptr(idx)
    rc = fn(desc, buf.ptr, buf.nbytes, stream) if buf is not None else fn(desc, None, 0, stream)
    if rc == L.MT_ERR_WORKSPACE:
        ws, n = workspace(size_fn(desc), idx)
        rc = fn(desc, ws, n, stream)
    if rc:
        L.check(rc, what)


def _require_int32(what, B, name, t):
    """Index tensors of a batch: int32 on the device, contiguous, one value a sequence."""
    if t.dtype is not int32 or t.device.type != "cuda":
        raise ValueError(f"{what}: {name} has to be an int32 tensor on the cuda device")
    if t._shape != (B,) or (t._strides != (1,) and B > 1):
        raise ValueError(f"{what}: {name} has to be contiguous of shape [{B}], got {list(t._shape)}")


def _check_out(out, shape, like, what):
    if out._shape != shape:
        raise RuntimeError(f"{what}: out has shape {list(out._shape)}, expected {list(shape)}")
    if out.dtype is not like.dtype or out.device.type != "cuda":
        raise ValueError(f"{what}: out has to be a {like.dtype.name} tensor on the cuda device")
    if 0 in out._strides and any(n > 1 and s == 0 for n, s in zip(out._shape, out._strides)):
        raise ValueError(f"{what}: out is an expanded view")
    return out


def _new_heads(b, h, s, d, like):
    """A [b, h, s, d] view of new heads-merged rows [b, s, h * d], which the next projection reads."""
    return _new((b, s, h, d), like.dtype, like.device)._view((b, h, s, d), (s * h * d, d, h * d, 1))


# ---------------------------------------------------------------------------------------------
# rotary positions


def rotary_frequencies(sections, theta: float = 10000.0, shared: bool = False, device="cuda") -> Tensor:
    """float32 frequencies for `rotary_embedding`: `sections[a]` pairs for each axis.  Each axis has a
    ladder theta^(-i / n) of its own, or with `shared` one ladder runs through all the pairs."""
    sections = [int(n) for n in sections]
    ladders = [sum(sections)] if shared else sections
    f = np.concatenate([theta ** (-np.arange(n, dtype=np.float64) / max(n, 1)) for n in ladders])
    return tensor(f.astype(np.float32)).to(device)


def rotary_embedding(q: Tensor, k: Tensor | None, positions: Tensor, frequencies: Tensor, sections, *,
                     interleaved: bool = False, inverse: bool = False, out=None):
    """Turns the heads of `q` [B, Hq, S, D] and `k` [B, Hk, S, D] (or None) by their positions on
    several axes (time, height, width).

    Pair i turns by positions[axis(i)] * frequencies[i] (fp32); `sections[a]` pairs belong to axis a, in
    order.  Pair i is the channels (i, i + P) with P = sum(sections), or (2i, 2i + 1) when
    `interleaved`; channels past 2P are copied.  `positions`: int32 [axes, S] or [axes, B, S];
    `frequencies`: float32 [P] (`rotary_frequencies`).  `inverse` turns back, which is also the
    gradient of the forward turn.  Returns (q', k') (or q' without k); `out` is the tensor(s) to
    write, which may be the inputs themselves."""
    what = "rotary_embedding"
    _require_cuda(q, k, positions, frequencies)
    if q.dim() != 4 or (k is not None and k.dim() != 4):
        raise ValueError(f"{what}: q and k have to be [batch, heads, tokens, dim]")
    B, Hq, S, D = q._shape
    if k is not None:
        _same_dtype(q, k, what=what)
        if k._shape[0] != B or k._shape[2] != S or k._shape[3] != D:
            raise ValueError(f"{what}: q {list(q._shape)} and k {list(k._shape)} differ in batch, tokens or dim")
    else:
        _same_dtype(q, what=what)
    axes = len(sections)
    if not 1 <= axes <= 4 or min(sections) < 0:
        raise ValueError(f"{what}: 1 to 4 sections of pairs, got {list(sections)}")
    pairs = sum(sections)
    if 2 * pairs > D:
        raise ValueError(f"{what}: {pairs} pairs do not fit a head dim of {D}")
    if positions.dtype is not int32 or positions.dim() not in (2, 3) or positions._shape[0] != axes or \
            positions._shape[-1] != S or (positions.dim() == 3 and positions._shape[1] not in (1, B)):
        raise ValueError(f"{what}: positions have to be int32 [{axes}, {S}] or [{axes}, {B}, {S}]")
    if S > 1 and positions._strides[-1] != 1:
        positions = positions.contiguous()
    if frequencies.dtype is not float32 or frequencies._shape != (pairs,) or (pairs > 1 and frequencies._strides != (1,)):
        raise ValueError(f"{what}: frequencies have to be float32 [{pairs}]")
    if out is None:
        oq = _new_heads(B, Hq, S, D, q)
        ok = _new_heads(B, k._shape[1], S, D, k) if k is not None else None
    else:
        oq, ok = (out, None) if isinstance(out, Tensor) else (out[0], out[1] if len(out) > 1 else None)
        _check_out(oq, q._shape, q, what)
        if (ok is None) != (k is None):
            raise ValueError(f"{what}: out has to hold a tensor for each of q and k")
        if k is not None:
            _check_out(ok, k._shape, k, what)
    ends = [0, 0, 0, 0]
    at = 0
    for a, n in enumerate(sections):
        at += n
        ends[a] = at
    pb = positions._strides[1] if positions.dim() == 3 and positions._shape[1] > 1 else 0
    kq = (_ptr(k), *k._strides, _ptr(ok), *ok._strides) if k is not None else (0,) * 10
    d = L.pack_rotary(B, S, D, Hq, k._shape[1] if k is not None else 0, q.dtype.code, bool(interleaved), bool(inverse),
                      axes, pairs, *ends, _ptr(positions), positions._strides[0], pb, _ptr(frequencies), _ptr(q),
                      *q._strides, _ptr(oq), *oq._strides, *kq)
    _check(_lib().mt_cuda_rotary(d, stream_ptr(q.device.index or 0)), what)
    oq._mark_modified()
    if k is None:
        return oq
    ok._mark_modified()
    return oq, ok


# ---------------------------------------------------------------------------------------------
# attention with a sliding window and sinks


def _window_arg(window, sinks, what):
    w = 0 if window is None else int(window)
    if (window is not None and w < 1) or sinks < 0:
        raise ValueError(f"{what}: window has to be at least 1 (or None) and sinks at least 0")
    return w


def window_attention(q: Tensor, k: Tensor, v: Tensor, window: int | None, sinks: int = 0, *, causal: bool = True,
                     starts: Tensor | None = None, lengths: Tensor | None = None, scale: float | None = None,
                     out: Tensor | None = None) -> Tensor:
    """Attention of `q` [B, H, Sq, D] over `k` and `v` [B, Hkv, Sk, D] with a sliding window of `window` keys and
    the first `sinks` keys always visible.

    Query i of sequence b is at position p = starts[b] + i (default Sk - Sq + i).  It sees key j below
    lengths[b] (default Sk) when j <= p and (p - j < window or j < sinks); without `causal` when
    |p - j| < window or j < sinks.  `window=None`: no window.  A query that sees no key gets zeros.
    Keys at lengths[b] and beyond may hold anything; below it the values have to be finite (an infinity or
    NaN can reach neighbouring queries that do not see its key).  H may be a multiple of Hkv (shared key
    heads).  `starts`, `lengths`: int32 [B] on the device."""
    what = "window_attention"
    _require_cuda(q, k, v)
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError(f"{what}: q, k and v have to be [batch, heads, tokens, dim]")
    _same_dtype(q, k, v, what=what)
    B, H, Sq, D = q._shape
    Hkv, Sk = k._shape[1], k._shape[2]
    if k._shape != v._shape or k._shape[0] != B or k._shape[3] != D:
        raise ValueError(f"{what}: q {list(q._shape)}, k {list(k._shape)} and v {list(v._shape)} do not go together")
    if Hkv == 0 or H % Hkv:
        raise ValueError(f"{what}: number of heads in key/value must divide number of heads in query")
    w = _window_arg(window, sinks, what)
    if starts is not None:
        _require_int32(what, B, "starts", starts)
    if lengths is not None:
        _require_int32(what, B, "lengths", lengths)
    if out is None:
        out = _new_heads(B, H, Sq, D, q)
    else:
        _check_out(out, q._shape, q, what)
    d = L.pack_window_attention(
        B, H, Hkv, Sq, Sk, D, q.dtype.code, bool(causal), w, int(sinks), _ptr(starts) if starts is not None else 0,
        _ptr(lengths) if lengths is not None else 0, _ptr(q), *q._strides, _ptr(k), *k._strides, _ptr(v), *v._strides,
        _ptr(out), *out._strides, float(scale) if scale is not None else 1.0 / math.sqrt(D))
    lib = _lib()
    _run(lib.mt_cuda_window_attention, lib.mt_cuda_window_attention_workspace_size, d, q, what)
    out._mark_modified()
    return out


# ---------------------------------------------------------------------------------------------
# the paged cache in 4 bits


class KVCache4:
    """Keys and values of many sequences in pages, held in 4 bits: `k_words`, `v_words` int32
    [pages, heads, page_size, dim / 8] (8 codes a word, the first channel in the lowest bits) and `k_scales`,
    `v_scales` float16 [pages, heads, page_size, dim / 64, 2] (scale and zero of each 64 channels):
    value = zero + scale * code.  Which pages a sequence has is the caller's table, int32 [batch, pages of
    a sequence]: token t is in page table[b, t // page_size]."""

    def __init__(self, k_words: Tensor, k_scales: Tensor, v_words: Tensor, v_scales: Tensor):
        for name, t, dt in (("k_words", k_words, int32), ("v_words", v_words, int32), ("k_scales", k_scales, float16),
                            ("v_scales", v_scales, float16)):
            _require_cuda(t)
            if t.dtype is not dt or not t.is_contiguous():
                raise ValueError(f"KVCache4: {name} has to be a contiguous {dt.name} tensor")
        if k_words.dim() != 4:
            raise ValueError("KVCache4: words have to be [pages, heads, page_size, dim / 8]")
        pages, heads, page, w = k_words._shape
        if v_words._shape != k_words._shape or w % 8 or \
                k_scales._shape != (pages, heads, page, w // 8, 2) or v_scales._shape != k_scales._shape:
            raise ValueError("KVCache4: words [pages, heads, page_size, dim / 8] and scales "
                             "[pages, heads, page_size, dim / 64, 2] do not go together")
        if page < 16 or page > 1024 or page & (page - 1):
            raise ValueError(f"KVCache4: page_size {page} is not a power of two from 16 to 1024")
        if not 1 <= w // 8 <= 4:
            raise ValueError(f"KVCache4: head dim {w * 8} is not a multiple of 64 up to 256")
        self.k_words, self.k_scales, self.v_words, self.v_scales = k_words, k_scales, v_words, v_scales
        self.num_pages, self.heads, self.page_size, self.dim = pages, heads, page, w * 8
        self.device = k_words.device
        self._fields = (pages, page, heads, w * 8, k_words.data_ptr(), k_scales.data_ptr(), v_words.data_ptr(),
                        v_scales.data_ptr())
        self._desc = L.pack_kv_cache4(*self._fields)

    @classmethod
    def empty(cls, num_pages: int, page_size: int, heads: int, dim: int, device="cuda") -> "KVCache4":
        """A cache of `num_pages` pages, zeroed."""
        if dim % CACHE_GROUP:
            raise ValueError(f"KVCache4: head dim {dim} is not a multiple of {CACHE_GROUP} up to 256")
        dev = _device(device)

        def words():
            return zeros(num_pages, heads, page_size, dim // 8, dtype=int32, device=dev)

        def scales():
            return zeros(num_pages, heads, page_size, dim // CACHE_GROUP, 2, dtype=float16, device=dev)

        return cls(words(), scales(), words(), scales())

    @property
    def nbytes(self) -> int:
        return 2 * (self.k_words.numel() * 4 + self.k_scales.numel() * 2)


def _check_table(cache, table, B, what):
    if table.dtype is not int32 or table.dim() != 2 or table._shape[0] != B or table.device.type != "cuda" or \
            (table._shape[1] > 1 and table._strides[1] != 1):
        raise ValueError(f"{what}: block_table has to be int32 [{B}, pages of a sequence] on the cuda device")


def _cache_move(cache, k, v, table, starts, T, fn, what):
    B, H = k._shape[0], k._shape[1]
    if k._shape != (B, cache.heads, T, cache.dim) or v._shape != k._shape:
        raise ValueError(f"{what}: k and v have to be [batch, {cache.heads}, {T}, {cache.dim}], got {list(k._shape)} "
                         f"and {list(v._shape)}")
    _check_table(cache, table, B, what)
    _require_int32(what, B, "starts", starts)
    _check(fn(cache._desc, _ptr(k), L.pack_strides(*k._strides), _ptr(v), L.pack_strides(*v._strides), k.dtype.code, B, T,
              _ptr(table), table._strides[0], table._shape[1], _ptr(starts), stream_ptr(cache.device.index or 0)), what)


def kv_cache_append(cache: KVCache4, k: Tensor, v: Tensor, block_table: Tensor, starts: Tensor) -> None:
    """Writes `k` and `v` [B, heads, T, dim] to the cache as tokens starts[b] .. starts[b] + T - 1 of each
    sequence.  Per 64 channels (fp32): zero = f16(min), scale = f16((max - min) / 15), code =
    clamp(round((x - zero) / scale), 0, 15); a NaN makes its 64 channels NaN.  Tokens without a page in the table are
    not written."""
    what = "kv_cache_append"
    _require_cuda(k, v, block_table, starts)
    if k.dim() != 4:
        raise ValueError(f"{what}: k and v have to be [batch, heads, tokens, dim]")
    _same_dtype(k, v, what=what)
    _cache_move(cache, k, v, block_table, starts, k._shape[2], _lib().mt_cuda_kv_cache4_append, what)
    for t in (cache.k_words, cache.k_scales, cache.v_words, cache.v_scales):
        t._mark_modified()


def kv_cache_read(cache: KVCache4, block_table: Tensor, starts: Tensor, tokens: int, *, dtype=None, out=None):
    """The values of tokens starts[b] .. starts[b] + tokens - 1 of each sequence: (k, v) [B, heads, tokens,
    dim] in `dtype` (bfloat16), or written to the two tensors of `out`.  Tokens without a page read zero."""
    what = "kv_cache_read"
    _require_cuda(block_table, starts)
    B, T = starts._shape[0] if starts.dim() == 1 else -1, int(tokens)
    if out is None:
        dt = bfloat16 if dtype is None else to_dtype(dtype)
        out = tuple(_new((max(B, 0), cache.heads, T, cache.dim), dt, cache.device) for _ in range(2))
    k, v = out
    _require_cuda(k, v)
    _same_dtype(k, v, what=what)
    for t in (k, v):
        _check_out(t, (B, cache.heads, T, cache.dim), k, what)
    _cache_move(cache, k, v, block_table, starts, T, _lib().mt_cuda_kv_cache4_read, what)
    k._mark_modified()
    v._mark_modified()
    return k, v


def kv_cache_attention(q: Tensor, cache: KVCache4, block_table: Tensor, lengths: Tensor, *, window: int | None = None,
                       sinks: int = 0, scale: float | None = None, out: Tensor | None = None) -> Tensor:
    """Causal attention of the last tokens of each sequence, `q` [B, H, Sq, dim] (bfloat16 or float16), over the
    cache: query i is at position lengths[b] - Sq + i and sees the keys up to itself, with `window` and
    `sinks` as in `window_attention`.  `lengths` int32 [B] counts the tokens in the cache, the queries' own
    among them (append first).  Tokens below it that hold NaN can reach neighbouring queries that do not see them.  H may
    be a multiple of the cache's heads."""
    what = "kv_cache_attention"
    _require_cuda(q, block_table, lengths)
    if q.dim() != 4 or q._shape[3] != cache.dim:
        raise ValueError(f"{what}: q has to be [batch, heads, tokens, {cache.dim}], got {list(q._shape)}")
    B, H, Sq, D = q._shape
    if H % cache.heads:
        raise ValueError(f"{what}: number of heads in the cache must divide number of heads in query")
    if q.dtype is not bfloat16 and q.dtype is not float16:
        raise NotImplementedError(f"{what}: dtype {q.dtype.name} is not supported (bfloat16 or float16)")
    w = _window_arg(window, sinks, what)
    _check_table(cache, block_table, B, what)
    _require_int32(what, B, "lengths", lengths)
    if out is None:
        out = _new_heads(B, H, Sq, D, q)
    else:
        _check_out(out, q._shape, q, what)
    d = L.pack_kv_cache4_attention(
        *cache._fields, B, H, Sq, q.dtype.code, w, int(sinks), _ptr(block_table), block_table._strides[0],
        block_table._shape[1], _ptr(lengths), _ptr(q), *q._strides, _ptr(out), *out._strides,
        float(scale) if scale is not None else 1.0 / math.sqrt(D))
    lib = _lib()
    _run(lib.mt_cuda_kv_cache4_attention, lib.mt_cuda_kv_cache4_attention_workspace_size, d, q, what)
    out._mark_modified()
    return out


# ---------------------------------------------------------------------------------------------
# products with weights held in 4 bits


class Weight4:
    """A weight [out, cols] held in 4 bits: value = scale * (code - 8).  `words` int32 [out, P / 8] with P = cols
    rounded up to 128 (in each 16 words word w is stored at place (w % 4) * 4 + w // 4, the order the
    products read), `scales` bfloat16 [out, P / group] with groups of 32, 64 or 128 columns.
    `Weight4.pack(w, group)` makes one from a floating weight."""

    def __init__(self, words: Tensor, scales: Tensor, cols: int):
        _require_cuda(words, scales)
        P = (int(cols) + 127) // 128 * 128
        if words.dtype is not int32 or scales.dtype is not bfloat16 or not words.is_contiguous() or \
                not scales.is_contiguous() or words.dim() != 2 or scales.dim() != 2:
            raise ValueError("Weight4: words have to be int32 and scales bfloat16, contiguous matrices")
        if cols < 1 or words._shape[1] * 8 != P or scales._shape[0] != words._shape[0]:
            raise ValueError(f"Weight4: words {list(words._shape)} and scales {list(scales._shape)} for {cols} columns")
        group = P // scales._shape[1] if scales._shape[1] else 0
        if group not in (32, 64, 128) or group * scales._shape[1] != P:
            raise ValueError(f"Weight4: {scales._shape[1]} scales for {P} columns (groups of 32, 64 or 128)")
        self.words, self.scales, self.cols, self.out, self.group = words, scales, int(cols), words._shape[0], group

    @classmethod
    def pack(cls, w: Tensor, group: int = 128) -> "Weight4":
        """Packs `w` [out, cols]: per group scale = bf16(max|w| / 7), code = clamp(round(w / scale), -8, 7) + 8."""
        _require_cuda(w)
        _same_dtype(w, what="Weight4.pack")
        if w.dim() != 2 or group not in (32, 64, 128):
            raise ValueError("Weight4.pack: a matrix and a group of 32, 64 or 128")
        if w._strides[1] != 1 and w._shape[1] > 1:
            w = w.contiguous()
        n, k = w._shape
        P = (k + 127) // 128 * 128
        words, scales = _new((n, P // 8), int32, w.device), _new((n, P // group), bfloat16, w.device)
        L.check(_lib().mt_cuda_weight4_pack(words.data_ptr(), scales.data_ptr(), w.data_ptr(), w.dtype.code, w._strides[0],
                                            n, k, group, w._stream()), "Weight4.pack")
        return cls(words, scales, k)

    def unpack(self, dtype=bfloat16) -> Tensor:
        """The values [out, cols] in `dtype`."""
        w = _new((self.out, self.cols), to_dtype(dtype), self.words.device)
        _same_dtype(w, what="Weight4.unpack")
        L.check(_lib().mt_cuda_weight4_unpack(w.data_ptr(), w.dtype.code, self.cols, self.words.data_ptr(),
                                              self.scales.data_ptr(), self.out, self.cols, self.group, w._stream()),
                "Weight4.unpack")
        return w

    @property
    def nbytes(self) -> int:
        return self.words.numel() * 4 + self.scales.numel() * 2


def linear_weight4(x: Tensor, weight: Weight4, bias: Tensor | None = None, *, out: Tensor | None = None) -> Tensor:
    """`linear` with a weight held in 4 bits: x [..., cols] -> [..., out].  Made for few rows (a decoder's step);
    many rows go through copies in f16 (exact, rows of both times powers of two) and the tensor-core product."""
    what = "linear_weight4"
    _require_cuda(x, bias)
    _same_dtype(x, bias, what=what) if bias is not None else _same_dtype(x, what=what)
    if x.dim() < 1 or x._shape[-1] != weight.cols:
        raise RuntimeError(f"{what}: input [..., {x._shape[-1] if x.dim() else ''}] and weight "
                           f"[{weight.out}, {weight.cols}] cannot be multiplied")
    if bias is not None and (bias._shape != (weight.out,) or not bias.is_contiguous()):
        raise RuntimeError(f"{what}: bias has to be [{weight.out}]")
    lead = x._shape[:-1]
    if x.dim() != 2 or (x._strides[1] != 1 and weight.cols > 1):
        x = x.reshape(-1, weight.cols)
    if x._strides[1] != 1 and weight.cols > 1:
        x = x.contiguous()
    M = x._shape[0]
    if out is None:
        out = _new(lead + (weight.out,), x.dtype, x.device)
        ldy = weight.out
    else:
        _check_out(out, lead + (weight.out,), x, what)
        if weight.out > 1 and out._strides[-1] != 1 or (out.dim() != 2 and not out.is_contiguous()):
            raise ValueError(f"{what}: out has to have unit-stride rows")
        ldy = out._strides[0] if out.dim() == 2 else weight.out
    d = L.pack_linear_weight4(M, weight.out, weight.cols, weight.group, x.dtype.code, _ptr(x), x._strides[0],
                              _ptr(weight.words), _ptr(weight.scales), _ptr(bias) if bias is not None else 0, _ptr(out), ldy)
    lib = _lib()
    _run(lib.mt_cuda_linear_weight4, lib.mt_cuda_linear_weight4_workspace_size, d, x, what)
    out._mark_modified()
    return out
