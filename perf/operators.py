"""The operators of a causal decoder beside the image path: what they compute, on which work, and how exactly.

Four operators, each in its plain form (elementary torch operations in 32 bits) and as the call that a user of
``mtorch_b200`` makes:

``rotary``   rotary positions with several axes (time, height, width) on the query and key heads of a transformer;
``window``   attention with a sliding window and a few first keys that stay visible (sinks);
``cache4``   a paged key / value cache held in 4 bits: appending tokens, and attention over it;
``linear4``  few rows times a weight held in 4 bits with group scales.

``own`` selects the side.  Inputs are torch tensors on the GPU; the package sees their memory through
``from_device_memory``, and its results land in the state's output buffers.  The package works on a stream of its
own, so the inputs have to be complete before a pass (``prepare`` ends with a synchronisation).
"""
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
GROUP = 64  # channels of a head that share a scale and a zero point in the 4-bit cache


# ---------------------------------------------------------------------------------------------------------------
# cases


def listed():
    return [
        # one generated token for each of 4 sequences, 12 heads of 64 as in the text tower: latency
        dict(name="rotary_token", op="rotary", batch=4, tokens=1, heads=12, kv_heads=12, dim=64, sections="8,12,12",
             dtype="bf16", interleaved=False, inverse=False),
        # a clip of 16 frames of 32 x 32 latents through a video transformer's attention
        dict(name="rotary_video", op="rotary", batch=1, tokens=16384, heads=24, kv_heads=24, dim=128,
             sections="16,24,24", dtype="bf16", interleaved=False, inverse=False),
        # the gradient's direction in 32 bits: image tokens and a prompt of 77, rotated back
        dict(name="rotary_image_back", op="rotary", batch=2, tokens=4173, heads=16, kv_heads=4, dim=80,
             sections="10,10,10", dtype="f32", interleaved=True, inverse=True),
        # a long prompt: shared key heads, window and sinks
        dict(name="window_prompt", op="window", batch=1, heads=16, kv_heads=4, queries=8192, keys=8192, dim=128,
             window=2048, sinks=4, causal=True, ragged=False, dtype="bf16"),
        # a padded batch of odd lengths at the text tower's heads
        dict(name="window_ragged", op="window", batch=3, heads=12, kv_heads=12, queries=1031, keys=1031, dim=64,
             window=257, sinks=5, causal=True, ragged=True, dtype="f16"),
        # one token of each of 8 sequences against a 16-bit cache
        dict(name="window_token", op="window", batch=8, heads=32, kv_heads=8, queries=1, keys=6000, dim=128,
             window=4096, sinks=16, causal=True, ragged=True, dtype="bf16"),
        # a prompt written to the cache (and the written values read back)
        dict(name="cache4_append", op="append", batch=3, tokens=1500, kv_heads=8, dim=128, page=32, capacity=2048,
             dtype="bf16"),
        # generation: 24 long sequences of different lengths, one token each
        dict(name="cache4_batch", op="cache4", batch=24, heads=32, kv_heads=8, queries=1, dim=128, page=64,
             capacity=16384, window=0, sinks=0, dtype="bf16"),
        # four drafted tokens of one sequence, sliding window with sinks, small pages
        dict(name="cache4_draft", op="cache4", batch=1, heads=12, kv_heads=4, queries=4, dim=64, page=16,
             capacity=4096, window=1000, sinks=20, dtype="f16"),
        # the text tower's fused projection for one token
        dict(name="linear4_token", op="linear4", rows=1, cols=768, out=2304, group=64, dtype="bf16"),
        # the largest matrix of a generic decoder, one token
        dict(name="linear4_wide", op="linear4", rows=1, cols=8192, out=28672, group=128, dtype="f16"),
        # a small batch, odd sizes
        dict(name="linear4_batch", op="linear4", rows=13, cols=5000, out=4099, group=32, dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "window", "window_token", "append", "cache4", "linear4"])
    if op == "rotary":
        dim = rng.choice([32, 40, 64, 80, 96, 128, 160])
        axes = rng.choice([1, 2, 3])
        pairs = rng.choice([dim // 2, dim // 4, dim // 2 - 3])
        cut = [pairs // axes] * axes
        cut[0] += pairs - sum(cut)
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 3])
        batch = rng.choice([1, 2, 5])
        tokens = _spread(rng, 1, 16384)
        tokens = max(1, min(tokens, 16384 * 48 * 128 // (batch * (heads + kv) * dim)))
        return dict(op="rotary", batch=batch, tokens=tokens, heads=heads, kv_heads=kv, dim=dim,
                    sections=",".join(map(str, cut)), dtype=rng.choice(["bf16", "f16", "f32"]),
                    interleaved=rng.random() < 0.4, inverse=rng.random() < 0.4)
    if op == "window":
        kv = rng.choice([1, 2, 4])
        heads = kv * rng.choice([1, 2, 4])
        batch = rng.choice([1, 2, 3])
        dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
        dim = rng.choice([40, 64, 64, 80, 128, 128])
        keys = _spread(rng, 17, 1500 if dtype == "f32" else 6000)
        keys = min(keys, int(math.sqrt(8192 * 8192 * 16 / (batch * heads))))
        queries = keys if rng.random() < 0.6 else rng.randint(1, keys)
        return dict(op="window", batch=batch, heads=heads, kv_heads=kv, queries=queries, keys=keys, dim=dim,
                    window=_spread(rng, 1, 3000), sinks=rng.choice([0, 1, 4, 130]), causal=rng.random() < 0.75,
                    ragged=rng.random() < 0.5, dtype=dtype)
    if op == "window_token":
        kv = rng.choice([1, 2, 8])
        return dict(op="window", batch=_spread(rng, 1, 16), heads=kv * rng.choice([1, 3, 4, 8]), kv_heads=kv,
                    queries=rng.choice([1, 1, 1, 3, 8]), keys=_spread(rng, 10, 16000), dim=rng.choice([64, 80, 128]),
                    window=_spread(rng, 16, 16000), sinks=rng.choice([0, 4, 33]), causal=True, ragged=True,
                    dtype=rng.choice(["bf16", "f16", "f32"]))
    if op == "append":
        page = rng.choice([16, 32, 64])
        capacity = page * rng.randint(2, 2048 // page)
        return dict(op="append", batch=rng.choice([1, 2, 4]), tokens=_spread(rng, 1, capacity), dim=rng.choice([64, 128]),
                    kv_heads=rng.choice([1, 2, 8]), page=page, capacity=capacity, dtype=rng.choice(["bf16", "f16", "f32"]))
    if op == "cache4":
        kv = rng.choice([1, 4, 8])
        page = rng.choice([16, 32, 64, 128])
        batch = _spread(rng, 1, 24)
        capacity = page * max(1, _spread(rng, 16, 16384) // page)
        return dict(op="cache4", batch=batch, heads=kv * rng.choice([1, 2, 4, 8]), kv_heads=kv,
                    queries=rng.choice([1, 1, 1, 2, 5]), dim=rng.choice([64, 128]), page=page, capacity=capacity,
                    window=rng.choice([0, 0, _spread(rng, 10, 5000)]), sinks=rng.choice([0, 4, 50]),
                    dtype=rng.choice(["bf16", "f16"]))
    cols, out = _spread(rng, 64, 8192), _spread(rng, 64, 28672)
    return dict(op="linear4", rows=_spread(rng, 1, 32), cols=cols, out=out, group=rng.choice([32, 64, 128]),
                dtype=rng.choice(["bf16", "f16", "f32"]))


# ---------------------------------------------------------------------------------------------------------------
# inputs


def _sections(case):
    return [int(n) for n in case["sections"].split(",")]


def _randn(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEVICE) * scale).to(dtype)


def _heads(gen, batch, tokens, heads, dim, dtype, scale=1.0):
    """[batch, heads, tokens, dim] as a view of the [batch, tokens, heads, dim] rows that a projection writes."""
    return _randn(gen, (batch, tokens, heads, dim), dtype, scale).permute(0, 2, 1, 3)


def _int(gen, lo, hi, shape):
    return torch.randint(lo, hi + 1, shape, generator=gen, device=DEVICE, dtype=torch.int32)


def _nibbles(codes):
    """Codes 0..15 of [..., n] packed into int32 words of [..., n / 8], the first code in the lowest bits."""
    c = codes.to(torch.int64).unflatten(-1, (-1, 8))
    w = (c << (4 * torch.arange(8, device=codes.device))).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def _codes(words):
    """The codes of _nibbles, as 32-bit floating values of [..., 8 n]."""
    w = words.unsqueeze(-1) >> (4 * torch.arange(8, device=words.device, dtype=torch.int32))
    return (w & 15).float().flatten(-2)


def _quantise_cache(x):
    """Words [..., dim / 8] and 16-bit (scale, zero) pairs [..., dim / 64, 2] of x [..., dim]."""
    g = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1), g.amax(-1)
    zero = lo.clamp(-65504.0, 65504.0).half()
    scale = ((hi - lo) * (1.0 / 15.0)).clamp(max=65504.0).half()
    s = scale.float().unsqueeze(-1)
    codes = torch.where(s > 0, ((g - zero.float().unsqueeze(-1)) / s).round().clamp(0, 15), torch.zeros_like(g))
    return _nibbles(codes.flatten(-2)), torch.stack([scale, zero], -1)


def _dequantise_cache(words, scales):
    c = _codes(words).unflatten(-1, (-1, GROUP))
    return (c * scales[..., 0].float().unsqueeze(-1) + scales[..., 1].float().unsqueeze(-1)).flatten(-2)


def _to_blocks(words):
    """Words [out, 16 n] of a weight in the order that the products read: in each 16 words (128 columns), word w at
    place (w % 4) * 4 + w / 4."""
    return words.unflatten(-1, (-1, 4, 4)).transpose(-1, -2).flatten(-3).contiguous()


def _paged(case, gen):
    """A cache of pages handed out in random order, more of them than the sequences need, and the table of pages."""
    per = case["capacity"] // case["page"]
    pages = case["batch"] * per + 3
    table = torch.randperm(pages, generator=gen, device=DEVICE)[: case["batch"] * per].view(case["batch"], per)
    shape = (pages, case["kv_heads"], case["page"])
    return shape, table.to(torch.int32).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    op, dtype = case["op"], TYPES[case["dtype"]]
    s = {"op": op, "case": case}
    if op == "rotary":
        sec = _sections(case)
        b, t, dim = case["batch"], case["tokens"], case["dim"]
        s["q"] = _heads(gen, b, t, case["heads"], dim, dtype)
        s["k"] = _heads(gen, b, t, case["kv_heads"], dim, dtype)
        # a grid of frames, rows and columns, each sequence somewhere of its own in time
        at = torch.arange(t, device=DEVICE)
        side = max(1, int(math.sqrt(t / 16)))
        axes = [at // (side * side), at // side % side, at % side][: len(sec)] if len(sec) > 1 else [at]
        first = _int(gen, 0, 500, (b, 1))
        s["positions"] = torch.stack([(a + (first if i == 0 else 0 * first)).to(torch.int32)
                                      for i, a in enumerate(axes)]).contiguous()
        s["frequencies"] = torch.cat([10000.0 ** (-torch.arange(n, device=DEVICE, dtype=torch.float64) / n)
                                      for n in sec]).float()
        s["out"] = [torch.empty_like(s["q"]), torch.empty_like(s["k"])]
    elif op == "window":
        b, dim = case["batch"], case["dim"]
        s["q"] = _heads(gen, b, case["queries"], case["heads"], dim, dtype)
        s["k"] = _heads(gen, b, case["keys"], case["kv_heads"], dim, dtype)
        s["v"] = _heads(gen, b, case["keys"], case["kv_heads"], dim, dtype)
        if case["ragged"]:
            # full keys for the first sequence, less for the others; the queries are the last of what there is, or
            # where as many queries as keys come, the padded prompt itself
            n = _int(gen, max(1, case["keys"] // 3), case["keys"], (b,))
            n[0] = case["keys"]
            s["lengths"] = n
            s["starts"] = (torch.zeros_like(n) if case["queries"] == case["keys"] else n - case["queries"])
        else:
            s["lengths"] = s["starts"] = None
        s["out"] = torch.empty_like(s["q"])
    elif op == "append":
        b, t, dim = case["batch"], case["tokens"], case["dim"]
        shape, s["table"] = _paged(case, gen)
        for n in ("k", "v"):
            # channels have levels of their own, as keys do
            level = torch.randn((1, 1, case["kv_heads"], dim), generator=gen, device=DEVICE)
            s[n] = (torch.randn((b, t, case["kv_heads"], dim), generator=gen, device=DEVICE)
                    + level).to(dtype).permute(0, 2, 1, 3)
            s[n + "_words"] = torch.zeros(shape + (dim // 8,), dtype=torch.int32, device=DEVICE)
            s[n + "_scales"] = torch.zeros(shape + (dim // GROUP, 2), dtype=torch.float16, device=DEVICE)
        s["starts"] = _int(gen, 0, case["capacity"] - t, (b,))
        s["out"] = [torch.empty((b, case["kv_heads"], t, dim), dtype=dtype, device=DEVICE) for _ in range(2)]
    elif op == "cache4":
        b, dim, g = case["batch"], case["dim"], case["queries"]
        shape, s["table"] = _paged(case, gen)
        for n in ("k", "v"):
            words = torch.empty(shape + (dim // 8,), dtype=torch.int32, device=DEVICE)
            scales = torch.empty(shape + (dim // GROUP, 2), dtype=torch.float16, device=DEVICE)
            level = torch.randn((1, shape[1], 1, dim), generator=gen, device=DEVICE)
            step = max(1, (1 << 26) // max(1, shape[1] * shape[2] * dim))
            for at in range(0, shape[0], step):  # a part of the pages at a time: the codes are wide while they are made
                x = torch.randn((min(step, shape[0] - at),) + shape[1:] + (dim,), generator=gen, device=DEVICE) + level
                words[at:at + step], scales[at:at + step] = _quantise_cache(x)
            s[n + "_words"], s[n + "_scales"] = words, scales
        s["q"] = _heads(gen, b, g, case["heads"], dim, dtype)
        s["lengths"] = _int(gen, min(case["capacity"], max(g, case["capacity"] // 4)), case["capacity"], (b,))
        s["lengths"][0] = case["capacity"]
        s["out"] = torch.empty((b, case["heads"], g, dim), dtype=dtype, device=DEVICE)
    else:
        cols, out, group = case["cols"], case["out"], case["group"]
        padded = (cols + 127) // 128 * 128
        w = torch.zeros((out, padded), device=DEVICE)
        w[:, :cols] = torch.randn((out, cols), generator=gen, device=DEVICE) / math.sqrt(cols)
        w = w.view(out, padded // group, group)
        scale = (w.abs().amax(-1) * (1.0 / 7.0)).to(torch.bfloat16)
        sf = scale.float().unsqueeze(-1)
        codes = torch.where(sf > 0, (w / sf).round().clamp(-8, 7), torch.zeros_like(w)) + 8
        s["words"] = _to_blocks(_nibbles(codes.view(out, padded)))
        s["scales"] = scale
        s["x"] = _randn(gen, (case["rows"], cols), dtype)
        s["bias"] = _randn(gen, (out,), dtype, 0.1)
        s["out"] = torch.empty((case["rows"], out), dtype=dtype, device=DEVICE)
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------------------------------------------------------
# plain forms, in 32 bits


def _rotary_plain(s):
    c, pos, sec = s["case"], s["positions"], _sections(s["case"])
    which = torch.repeat_interleave(torch.arange(len(sec), device=DEVICE), torch.tensor(sec, device=DEVICE))
    angle = (pos.float()[which] * s["frequencies"][:, None, None]).permute(1, 2, 0)[:, None]  # [b, 1, t, pairs]
    cos, sin = angle.cos(), angle.sin()
    if c["inverse"]:
        sin = -sin
    p = sum(sec)

    def turn(x):
        x = x.float()
        rest = x[..., 2 * p:]
        if c["interleaved"]:
            a, b = x[..., 0:2 * p:2], x[..., 1:2 * p:2]
            y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        else:
            a, b = x[..., :p], x[..., p:2 * p]
            y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        return torch.cat([y, rest], -1).to(TYPES[c["dtype"]])

    return [turn(s["q"]), turn(s["k"])]


def _visible(position, keys, lengths, window, sinks, causal):
    """Which of the keys (0 .. keys) the queries at position [b, q] see: [b, 1, q, keys]."""
    p, j = position[:, None, :, None].long(), torch.arange(keys, device=DEVICE)
    see = (j > p - window) if window else torch.ones_like(p, dtype=torch.bool) & (j >= 0)
    if not causal and window:
        see = see & (j < p + window)
    see = see | (j < sinks)
    if causal:
        see = see & (j <= p)
    return see & (j < lengths[:, None, None, None])


def _attend_plain(q, k, v, see, dtype):
    b, heads, n, dim = q.shape
    kv = k.shape[1]
    q = q.float().reshape(b, kv, heads // kv * n, dim)
    scores = (q @ k.float().transpose(-1, -2)).view(b, heads, n, -1) * (1.0 / math.sqrt(dim))
    scores = scores.masked_fill(~see, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    out = (p.view(b, kv, heads // kv * n, -1) @ v.float()).view(b, heads, n, dim)
    return torch.where(total > 0, out / total, torch.zeros_like(out)).to(dtype)


def _window_plain(s):
    c = s["case"]
    b, n, keys = c["batch"], c["queries"], c["keys"]
    lengths = s["lengths"] if s["lengths"] is not None else torch.full((b,), keys, device=DEVICE)
    starts = s["starts"] if s["starts"] is not None else torch.full((b,), keys - n, device=DEVICE)
    position = starts[:, None] + torch.arange(n, device=DEVICE)
    see = _visible(position, keys, lengths, c["window"], c["sinks"], c["causal"])
    return _attend_plain(s["q"], s["k"], s["v"], see, TYPES[c["dtype"]])


def _append_plain(s):
    c = s["case"]
    at = s["starts"][:, None].long() + torch.arange(c["tokens"], device=DEVICE)
    page = torch.gather(s["table"].long(), 1, at // c["page"])
    slot = at % c["page"]
    got = []
    for n in ("k", "v"):
        words, scales = _quantise_cache(s[n].permute(0, 2, 1, 3))  # [b, t, heads, ...]
        s[n + "_words"][page, :, slot] = words
        s[n + "_scales"][page, :, slot] = scales
        back = _dequantise_cache(s[n + "_words"][page, :, slot], s[n + "_scales"][page, :, slot])
        got.append(back.permute(0, 2, 1, 3).to(TYPES[c["dtype"]]).contiguous())
    return got


def _cache4_plain(s):
    c = s["case"]
    b, per = s["table"].shape
    table = s["table"].long()

    def values(n):
        x = _dequantise_cache(s[n + "_words"][table], s[n + "_scales"][table])  # [b, pages, heads, page, dim]
        return x.transpose(1, 2).flatten(2, 3)

    position = s["lengths"][:, None] - c["queries"] + torch.arange(c["queries"], device=DEVICE)
    see = _visible(position, per * c["page"], s["lengths"], c["window"], c["sinks"], True)
    return _attend_plain(s["q"], values("k"), values("v"), see, TYPES[c["dtype"]])


def _linear4_plain(s):
    c = s["case"]
    words = s["words"].unflatten(-1, (-1, 4, 4)).transpose(-1, -2).flatten(-3)
    w = (_codes(words) - 8).unflatten(-1, (-1, c["group"])) * s["scales"].float().unsqueeze(-1)
    w = w.flatten(-2)[:, : c["cols"]]
    return (s["x"].float() @ w.t() + s["bias"].float()).to(TYPES[c["dtype"]])


# ---------------------------------------------------------------------------------------------------------------
# the package's operators


def _handles(s):
    """The package's tensors over the state's memory, which a program keeps beside its buffers."""
    import mtorch_b200 as mt

    names = {torch.bfloat16: mt.bfloat16, torch.float16: mt.float16, torch.float32: mt.float32, torch.int32: mt.int32}

    def wrap(t):
        return mt.from_device_memory(t.data_ptr(), t.shape, names[t.dtype], strides=t.stride(), owner=t)

    h = {"mt": mt}
    for name, t in s.items():
        if isinstance(t, torch.Tensor):
            h[name] = wrap(t)
        elif name == "out":
            h[name] = [wrap(x) for x in t]
        elif t is None:
            h[name] = None
    c = s["case"]
    if "k_words" in s:
        h["cache"] = mt.KVCache4(h["k_words"], h["k_scales"], h["v_words"], h["v_scales"])
    if "words" in s:
        h["weight"] = mt.Weight4(h["words"], h["scales"], c["cols"])
    if "sections" in c:
        h["sections"] = tuple(_sections(c))
    return h


def _run_own(s):
    if "handles" not in s:
        s["handles"] = _handles(s)
    h, c, op = s["handles"], s["case"], s["op"]
    mt = h["mt"]
    if op == "rotary":
        mt.rotary_embedding(h["q"], h["k"], h["positions"], h["frequencies"], h["sections"],
                            interleaved=c["interleaved"], inverse=c["inverse"], out=h["out"])
    elif op == "window":
        mt.window_attention(h["q"], h["k"], h["v"], c["window"], c["sinks"], causal=c["causal"], starts=h["starts"],
                            lengths=h["lengths"], out=h["out"])
    elif op == "append":
        mt.kv_cache_append(h["cache"], h["k"], h["v"], h["table"], h["starts"])
        mt.kv_cache_read(h["cache"], h["table"], h["starts"], c["tokens"], out=h["out"])
    elif op == "cache4":
        mt.kv_cache_attention(h["q"], h["cache"], h["table"], h["lengths"], window=c["window"] or None,
                              sinks=c["sinks"], out=h["out"])
    else:
        mt.linear_weight4(h["x"], h["weight"], h["bias"], out=h["out"])
    return s["out"]


def run(state):
    if own:
        return _run_own(state)
    return {"rotary": _rotary_plain, "window": _window_plain, "append": _append_plain, "cache4": _cache4_plain,
            "linear4": _linear4_plain}[state["op"]](state)


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without


def _pairs(queries, keys, start, window, sinks, causal):
    """Pairs of a query and a key that it sees, of queries at start, start + 1, ... against `keys` keys, and the keys
    that any of them sees."""
    p = torch.arange(queries, dtype=torch.int64) + start
    hi = torch.minimum(p if causal else (p + (window or keys) - 1), torch.tensor(keys - 1)) + 1
    lo = (p - window + 1).clamp(min=0) if window else torch.zeros_like(p)
    lo = torch.minimum(lo, hi.clamp(min=0))
    first = torch.minimum(torch.full_like(p, min(sinks, keys)), p + 1 if causal else torch.full_like(p, keys)).clamp(min=0)
    pairs = int(((hi - lo).clamp(min=0) + torch.minimum(first, lo).clamp(min=0)).sum())
    seen = int(min(keys, (hi.max() - lo.min()).clamp(min=0) + min(sinks, int(lo.min()))))
    return pairs, seen


def work(case):
    op, size = case["op"], torch.empty(0, dtype=TYPES[case["dtype"]]).element_size()
    if op == "rotary":
        n = case["batch"] * case["tokens"]
        values = n * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 2 * values * size + 4 * n * len(_sections(case)), "flops": 3 * values}
    if op == "append":
        values = 2 * case["batch"] * case["tokens"] * case["kv_heads"] * case["dim"]
        return {"bytes": 2 * values * size + values * (0.5 + 4 / GROUP), "flops": 6 * values}
    if op == "linear4":
        w = case["out"] * case["cols"]
        return {"bytes": w / 2 + 2 * w / case["group"] + size * (case["rows"] * (case["cols"] + case["out"]) + case["out"]),
                "flops": 2 * case["rows"] * w}
    # attention: mean length of the ragged sequences, as prepare() draws them
    b, n, dim, kv = case["batch"], case["queries"], case["dim"], case["kv_heads"]
    if op == "window":
        lo = max(1, case["keys"] // 3) if case["ragged"] else case["keys"]
        keys, each, causal = case["keys"], 2 * dim * size, case["causal"]
    else:
        keys, each, causal = case["capacity"], 2 * (dim // 2 + 4 * dim // GROUP), True
        lo = min(keys, max(n, keys // 4))
    pairs = seen = 0
    for i in range(b):
        length = keys if i == 0 else (lo + keys) // 2
        start = 0 if op == "window" and n == keys else length - n
        x, y = _pairs(n, length, start, case["window"], case["sinks"], causal)
        pairs, seen = pairs + x, seen + y
    return {"bytes": seen * kv * each + 2 * b * n * case["heads"] * dim * size, "flops": 4 * pairs * case["heads"] * dim}


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits


def _exact_attention(q, keys_of, values_of, see_of, dim):
    """softmax(q k / sqrt(dim)) v, a sequence and a head at a time; see_of gives 1 where a query sees a key."""
    b, heads, n, _ = q.shape
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for i in range(b):
        k, v, see = keys_of(i), values_of(i), see_of(i)
        for h in range(heads):
            at = h * k.shape[0] // heads
            z = torch.einsum("qd,kd->qk", q[i, h].double(), k[at]) / dim ** 0.5
            z[~see] = -1e300
            z -= z.max(1, keepdim=True).values
            e = torch.exp(z) * see
            norm = e.sum(1)
            norm[norm == 0] = 1.0
            out[i, h] = torch.einsum("qk,kd->qd", e, v[at]) / norm[:, None]
    return out


def _exact_see(start, n, keys, length, window, sinks, causal):
    rows = (torch.arange(n, device=DEVICE) + int(start)).unsqueeze(1)
    col = torch.arange(keys, device=DEVICE).unsqueeze(0)
    gap = rows - col
    near = (gap < window) & ((gap > -window) | causal) if window else torch.ones_like(gap, dtype=torch.bool)
    ok = near | (col < sinks)
    if causal:
        ok &= gap >= 0
    return ok & (col < int(length))


def _exact_unpack(words):
    """Codes of [..., words] by division, in 64 bits: [..., 8 words]."""
    w = words.to(torch.int64) % (1 << 32)
    return torch.stack([(w // 16 ** i) % 16 for i in range(8)], -1).reshape(words.shape[:-1] + (-1,)).double()


def _exact_cache(s, name, i):
    """The values of sequence i in order: [heads, capacity, dim]."""
    pages = s["table"][i].long()
    code = _exact_unpack(s[name + "_words"][pages])
    scale = s[name + "_scales"][pages].double()
    at = torch.arange(code.shape[-1], device=DEVICE) // GROUP
    x = code * scale[..., 0][..., at] + scale[..., 1][..., at]
    return x.permute(1, 0, 2, 3).reshape(x.shape[1], -1, x.shape[3])


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "rotary":
        sec, dim = _sections(case), case["dim"]
        got = []
        for x in (s["q"], s["k"]):
            y, at = x.double().clone(), 0
            for axis, n in enumerate(sec):
                for i in range(at, at + n):
                    turn = s["positions"][axis].double() * s["frequencies"][i].double()
                    if case["interleaved"]:
                        a, b = 2 * i, 2 * i + 1
                    else:
                        a, b = i, i + sum(sec)
                    z = torch.complex(x[..., a].double(), x[..., b].double())
                    z = z * torch.polar(torch.ones_like(turn), -turn if case["inverse"] else turn)[:, None]
                    y[..., a], y[..., b] = z.real, z.imag
                at += n
            got.append(y)
        return got
    if op == "window":
        n, keys = case["queries"], case["keys"]
        lengths = [keys] * case["batch"] if s["lengths"] is None else s["lengths"].tolist()
        starts = [keys - n] * case["batch"] if s["starts"] is None else s["starts"].tolist()
        return _exact_attention(s["q"], lambda i: s["k"][i].double(), lambda i: s["v"][i].double(),
                                lambda i: _exact_see(starts[i], n, keys, lengths[i], case["window"], case["sinks"],
                                                     case["causal"]), case["dim"])
    if op == "cache4":
        lengths = s["lengths"].tolist()
        return _exact_attention(s["q"], lambda i: _exact_cache(s, "k", i), lambda i: _exact_cache(s, "v", i),
                                lambda i: _exact_see(lengths[i] - case["queries"], case["queries"], case["capacity"],
                                                     lengths[i], case["window"], case["sinks"], True), case["dim"])
    if op == "append":
        got = []
        for n in ("k", "v"):
            x = s[n].double()
            y = torch.empty(x.shape, dtype=torch.float64, device=DEVICE)
            for at in range(0, case["dim"], GROUP):
                part = x[..., at:at + GROUP]
                low, high = part.min(-1, keepdim=True).values, part.max(-1, keepdim=True).values
                zero, step = low.half().double(), ((high - low) / 15).half().double()
                near = torch.where(step > 0, torch.clamp(torch.round((part - zero) / step), 0, 15), 0.0 * part)
                y[..., at:at + GROUP] = zero + near * step
            got.append(y)
        return got
    words = s["words"].view(case["out"], -1, 4, 4).permute(0, 1, 3, 2).reshape(case["out"], -1)
    y = torch.empty((case["rows"], case["out"]), dtype=torch.float64, device=DEVICE)
    for at in range(0, case["out"], 2048):
        code = _exact_unpack(words[at:at + 2048]) - 8
        group = torch.arange(case["cols"], device=DEVICE) // case["group"]
        w = code[:, : case["cols"]] * s["scales"][at:at + 2048].double()[:, group]
        y[:, at:at + 2048] = torch.einsum("mk,nk->mn", s["x"].double(), w)
    return y + s["bias"].double()
