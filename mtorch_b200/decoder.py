"""A causal decoder of images and text (captions of a picture, longer prompts for the image path) on the
operators of ``decoding.py``.  (The reference has no such model; the layers are its text tower's
pre-LayerNorm layers, causal over everything that came before.)

Every projection's weight is held in 4 bits (`Linear4`), the keys and values of the past in a paged 4-bit
cache (`KVCache4`).  Tokens have positions on three axes, time, row and column: a text token is at
(i, i, i); the tokens of an image of rows x cols patches share one time and stand at (t, t + row, t + col), and
the text goes on behind the largest of them.  Attention sees a sliding window and the first `sinks` tokens.

A prompt runs through `window_attention` on its own keys and values and is then appended to the cache
(`prefill`); each further token is appended and attends over the cache (`step`), two calls a layer beside the
projections.  In float32 a step reads the cache back first.
"""
from __future__ import annotations

import numpy as np

from . import decoding, ops
from .nn import LayerNorm, Linear, Module, ModuleList, init
from .tensor import Tensor, _new, empty, float32, tensor, zeros


class Linear4(Module):
    """`Linear` with the weight held in 4 bits (`decoding.Weight4`): packed from a floating `Linear`.  Its parameters are
    the packed `words` and `scales`, whose types stay whatever the module is cast to, and the bias; a state dict
    with a floating `weight` in their place is packed as it is loaded."""

    def __init__(self, linear: Linear, group: int = 64):
        super().__init__()
        self.cols, self.group = linear.in_features, group
        w = decoding.Weight4.pack(linear.weight, group)
        self.register_parameter("words", w.words)
        self.register_parameter("scales", w.scales)
        self.register_parameter("bias", linear.bias)
        self._weight4 = w

    @property
    def weight4(self) -> decoding.Weight4:
        w = self._weight4
        if w.words is not self.words or w.scales is not self.scales:  # moved since
            w = self._weight4 = decoding.Weight4(self.words, self.scales, self.cols)
        return w

    def forward(self, x):
        return decoding.linear_weight4(x, self.weight4, self.bias)

    def _apply(self, fn):
        words, scales = self.words, self.scales
        self._parameters.update(words=None, scales=None)
        super()._apply(fn)
        dev = (self.bias if self.bias is not None else fn(scales)).device
        self.register_parameter("words", words.to(dev))
        self.register_parameter("scales", scales.to(dev))
        return self

    def _load_other(self, key, value):
        if key != "weight":
            return super()._load_other(key, value)
        value = value if isinstance(value, Tensor) else tensor(value)
        if tuple(value.shape) != (self.words.shape[0], self.cols):
            raise ValueError(f"Linear4: weight {list(value.shape)}, expected {[self.words.shape[0], self.cols]}")
        w = decoding.Weight4.pack(value.to(self.words.device), self.group)
        self.words.copy_(w.words)
        self.scales.copy_(w.scales)
        return True


class DecoderLayer(Module):
    def __init__(self, width, heads, kv_heads, mlp, group, device, dtype):
        super().__init__()
        kw = dict(device=device, dtype=dtype)
        self.heads, self.kv_heads, self.dim = heads, kv_heads, width // heads
        self.norm1, self.norm2 = LayerNorm(width, **kw), LayerNorm(width, **kw)
        self.qkv = Linear4(Linear(width, (heads + 2 * kv_heads) * self.dim, **kw), group)
        self.out = Linear4(Linear(heads * self.dim, width, **kw), group)
        self.fc1 = Linear4(Linear(width, mlp, **kw), group)
        self.fc2 = Linear4(Linear(mlp, width, **kw), group)

    def forward(self, h, n, s, state, layer):
        """h: [n * s, width] rows of the new tokens -> the same after this layer; `state`: what `Decoder` keeps
        of the call (positions, cache, table, lengths, window)."""
        D, H, G = self.dim, self.heads, self.kv_heads
        qkv = self.qkv(self.norm1(h))
        p = qkv.stride(0)

        def view(first, count):
            return qkv._view((n, count, s, D), (s * p, D, p, 1), qkv._offset + first * D)

        q, k, v = view(0, H), view(H, G), view(H + G, G)
        decoding.rotary_embedding(q, k, state.positions, state.frequencies, state.sections, out=(q, k))
        a = _new((n * s, H * D), h.dtype, h.device)
        av = a._view((n, H, s, D), (s * H * D, D, H * D, 1))
        cache = state.caches[layer]
        decoding.kv_cache_append(cache, k, v, state.table, state.starts)
        if state.prompt:
            decoding.window_attention(q, k, v, state.window, state.sinks, out=av)
        elif h.dtype is float32:  # (the cache's attention takes 16-bit queries)
            k, v = decoding.kv_cache_read(cache, state.table, state.zeros, state.capacity, dtype=float32)
            decoding.window_attention(q, k, v, state.window, state.sinks, starts=state.starts, lengths=state.lengths, out=av)
        else:
            decoding.kv_cache_attention(q, cache, state.table, state.lengths, window=state.window, sinks=state.sinks,
                                        out=av)
        h = self.out(a) + h
        return self.fc2(ops.gelu(self.fc1(self.norm2(h)))) + h


class _Call:
    pass


class Decoder(Module):
    """`prefill(tokens, image)` takes the prompts of a batch (all of one length) and returns the logits behind their
    last tokens; `step(tokens)` one further token of each.  `image` is [n, rows, cols, width] features that stand
    before the text.  Weights are random-init: embeddings N(0, 0.02), projections with the module default."""

    def __init__(self, vocab=49408, width=768, layers=12, heads=12, kv_heads=None, mlp=2048, window=1024, sinks=4,
                 group=64, page_size=64, sections=None, device="cuda", dtype="bfloat16"):
        super().__init__()
        if width % heads:
            raise ValueError(f"Decoder: width {width} is no multiple of {heads} heads")
        kv_heads = heads if kv_heads is None else kv_heads
        self.width, self.heads, self.kv_heads, self.dim = width, heads, kv_heads, width // heads
        if sections is None:  # a quarter of the pairs for time, the others for row and column
            pairs = self.dim // 2
            rc = 3 * pairs // 8
            sections = (pairs - 2 * rc, rc, rc)
        self.window, self.sinks, self.page_size, self.sections = window, sinks, page_size, tuple(sections)
        self.register_parameter("token_embedding", empty(vocab, width, device=device, dtype=dtype))
        init.normal_(self.token_embedding, 0.0, 0.02)
        self.layers = ModuleList([DecoderLayer(width, heads, kv_heads, mlp, group, device, dtype) for _ in range(layers)])
        self.final_norm = LayerNorm(width, device=device, dtype=dtype)
        self.register_buffer("frequencies", decoding.rotary_frequencies(self.sections, device=device))
        self._state = None

    def _apply(self, fn):
        f = self.frequencies
        self._buffers["frequencies"] = None
        super()._apply(fn)
        self.register_buffer("frequencies", f.to(self.token_embedding.device))  # (float32 whatever the module is cast to)
        return self

    def start(self, batch: int, tokens: int) -> None:
        """Makes room for `batch` sequences of up to `tokens` tokens: a cache per layer and the table of pages."""
        dev = self.token_embedding.device
        per = -(-tokens // self.page_size)
        st = self._state = _Call()
        st.batch, st.capacity = batch, per * self.page_size
        st.caches = [decoding.KVCache4.empty(batch * per, self.page_size, self.kv_heads, self.dim, device=dev)
                     for _ in self.layers]
        st.table = tensor(np.arange(batch * per, dtype=np.int32).reshape(batch, per), dtype="int32").to(dev)
        st.zeros = zeros(batch, dtype="int32", device=dev)
        st.frequencies, st.sections, st.window, st.sinks = self.frequencies, self.sections, self.window, self.sinks
        st.count = st.place = 0  # tokens so far; the next text token's position

    def _run(self, h, s, positions, prompt):
        st, dev = self._state, h.device
        n = st.batch
        if st.count + s > st.capacity:
            raise ValueError(f"Decoder: {st.count + s} tokens, room for {st.capacity}")

        def put(a):
            return tensor(np.ascontiguousarray(a, dtype=np.int32), dtype="int32").to(dev)

        st.prompt = prompt
        st.positions = put(positions)  # [3, s]: all sequences advance together
        st.starts = put(np.full(n, st.count))
        st.count += s
        st.lengths = put(np.full(n, st.count))
        for i, layer in enumerate(self.layers):
            h = layer(h, n, s, st, i)
        last = h.reshape(n, s, self.width)[:, s - 1:s].reshape(n, self.width)
        return ops.linear(self.final_norm(last), self.token_embedding)

    def prefill(self, tokens, image=None):
        """tokens [n, s] int64 (host or device), image [n, rows, cols, width] or None -> logits [n, vocab]."""
        st = self._state
        if st is None or st.count:
            raise RuntimeError("Decoder: prefill comes first after start()")
        n, s = tokens.shape
        if n != st.batch:
            raise ValueError(f"Decoder: {n} prompts, started for {st.batch}")
        h = ops.embedding(tokens, self.token_embedding)
        text0, at = 0, []
        if image is not None:
            if image.dim() != 4 or image.shape[0] != n or image.shape[3] != self.width:
                raise ValueError(f"Decoder: image features have to be [{n}, rows, cols, {self.width}]")
            rows, cols = image.shape[1], image.shape[2]
            h = ops.cat([image.reshape(n, rows * cols, self.width), h], dim=1)
            grid = np.indices((rows, cols)).reshape(2, -1)
            at.append(np.concatenate([np.zeros((1, rows * cols), np.int64), grid]))
            text0 = max(rows, cols)
        at.append(np.broadcast_to(text0 + np.arange(s), (3, s)))
        st.place = text0 + s
        positions = np.concatenate(at, axis=1)
        return self._run(h.reshape(-1, self.width), positions.shape[1], positions, True)

    def step(self, tokens):
        """tokens [n] or [n, 1] int64: the next token of each sequence -> logits [n, vocab]."""
        st = self._state
        if st is None or not st.count:
            raise RuntimeError("Decoder: step comes after prefill()")
        h = ops.embedding(tokens.reshape(st.batch, 1), self.token_embedding)
        positions = np.full((3, 1), st.place)
        st.place += 1
        return self._run(h.reshape(st.batch, self.width), 1, positions, False)

    def generate(self, tokens, count: int, image=None):
        """The `count` most likely further tokens (greedy), [n, count] int64 on the host."""
        n, s = tokens.shape
        self.start(n, s + count + (image.shape[1] * image.shape[2] if image is not None else 0))
        logits = self.prefill(tokens, image)
        out = []
        for i in range(count):
            nxt = logits.float().numpy().argmax(1).astype(np.int64)
            out.append(nxt)
            if i + 1 < count:
                logits = self.step(tensor(nxt))
        return np.stack(out, axis=1)
