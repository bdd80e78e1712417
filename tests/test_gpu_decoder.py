"""The decoder of images and text against a plain 64-bit forward pass of the same weights.

The forward pass below quantises the cache by its definition and computes everything else in 64 bits; the
device rounds activations to bf16 after every operation (2^-9 each, about ten in a layer, which LayerNorm
re-scales), and a code of the cache may differ by one where a rounded key stands near a tie.  Two layers of
such roundings stay below 40 * 2^-9 of the largest logit.
"""
import numpy as np
import pytest

import mtorch_b200 as mt
from mtorch_b200.decoder import Decoder
from test_gpu_decoding import attention_ref, quantised, rotary_ref

pytestmark = pytest.mark.gpu
TOL = 40 * 2.0 ** -9


def host(t):
    return t.float().numpy().astype(np.float64)


def norm(x, m):
    y = (x - x.mean(-1, keepdims=True)) / np.sqrt(x.var(-1, keepdims=True) + 1e-5)
    return y * host(m.weight) + host(m.bias)


def lin(x, m):
    return x @ host(m.weight4.unpack("float32")).T + host(m.bias)


def gelu(x):
    from scipy.special import erf

    return 0.5 * x * (1 + erf(x / np.sqrt(2)))


def forward(model, embed, positions, split):
    """Logits behind every token of [n, s, width]; tokens up to `split` attend to unrounded keys (the prompt's
    pass), the later ones to the cache."""
    h = embed
    n, s, width = h.shape
    for layer in model.layers:
        H, G, D = layer.heads, layer.kv_heads, layer.dim
        x = lin(norm(h, layer.norm1), layer.qkv).reshape(n, s, H + 2 * G, D).transpose(0, 2, 1, 3)
        pos = positions.astype(np.int32)[:, None].repeat(n, 1)
        f = model.frequencies.numpy()
        q = rotary_ref(x[:, :H], pos, f, model.sections, False, False)
        k = rotary_ref(x[:, H:H + G], pos, f, model.sections, False, False)
        v = x[:, H + G:]
        a = np.concatenate([
            attention_ref(q[:, :, :split], k[:, :, :split], v[:, :, :split], [0] * n, [split] * n, model.window, model.sinks, True),
            attention_ref(q[:, :, split:], quantised(k), quantised(v), [split] * n, [s] * n, model.window, model.sinks, True),
        ], axis=2)
        h = h + lin(a.transpose(0, 2, 1, 3).reshape(n, s, H * D), layer.out)
        h = h + lin(gelu(lin(norm(h, layer.norm2), layer.fc1)), layer.fc2)
    return norm(h, model.final_norm) @ host(model.token_embedding).T


def place(rows, cols, text):
    grid = np.indices((rows, cols)).reshape(2, -1)
    image = np.concatenate([np.zeros((1, rows * cols), int), grid])
    return np.concatenate([image, np.broadcast_to(max(rows, cols, 0) + np.arange(text), (3, text))], axis=1)


@pytest.mark.parametrize("heads,kv_heads,image", [(2, 2, None), (4, 2, (5, 7))])
def test_prompt_and_steps_match_the_plain_forward_pass(heads, kv_heads, image):
    mt.manual_seed(3)
    model = Decoder(vocab=300, width=64 * heads, layers=2, heads=heads, kv_heads=kv_heads, mlp=200, window=40, sinks=3,
                    page_size=16)
    rng = np.random.default_rng(0)
    n, s, steps = 2, 50, 6
    ids = rng.integers(0, 300, (n, s + steps))
    table = host(model.token_embedding)
    embed = table[ids]
    rows, cols = image or (0, 0)
    feats = None
    if image:
        feats = mt.tensor(rng.standard_normal((n, rows, cols, 64 * heads)).astype(np.float32) * 0.02).to("bfloat16").cuda()
        embed = np.concatenate([host(feats).reshape(n, rows * cols, -1), embed], axis=1)
    split = rows * cols + s
    want = forward(model, embed, place(rows, cols, s + steps), split)

    model.start(n, split + steps)
    logits = model.prefill(mt.tensor(ids[:, :s]), feats)
    got = [host(logits)]
    for i in range(steps):
        got.append(host(model.step(mt.tensor(ids[:, s + i]))))
    for i, g in enumerate(got):
        w = want[:, split - 1 + i]
        assert np.abs(g - w).max() <= TOL * np.abs(want).max(), (i, np.abs(g - w).max(), np.abs(want).max())


def test_generate_and_refusals():
    mt.manual_seed(4)
    model = Decoder(vocab=100, width=128, layers=1, heads=2, mlp=96, window=None, sinks=0, page_size=16)
    ids = mt.tensor(np.arange(20).reshape(2, 10))
    a = model.generate(ids, 5)
    b = model.generate(ids, 5)
    assert a.shape == (2, 5) and a.dtype == np.int64
    np.testing.assert_array_equal(a, b)
    model.start(2, 12)  # one page of 16 a sequence
    with pytest.raises(RuntimeError):
        model.step(mt.tensor(np.zeros(2, np.int64)))
    model.prefill(ids)
    for _ in range(6):
        model.step(mt.tensor(np.zeros(2, np.int64)))
    with pytest.raises(ValueError):
        model.step(mt.tensor(np.zeros(2, np.int64)))
    with pytest.raises(ValueError):
        Decoder(vocab=10, width=100, layers=1, heads=3, mlp=8)


def test_decode_step_in_a_graph():
    """Append and attention of a step replay from a captured graph, the split attention's joined launch included; the
    lengths are read from device memory."""
    rng = np.random.default_rng(1)
    B, H, G, D, page, per = 2, 4, 2, 64, 16, 64
    cache = mt.KVCache4.empty(B * per, page, G, D)
    table = mt.tensor(np.arange(B * per, dtype=np.int32).reshape(B, per), dtype="int32").cuda()

    def put(*shape):
        return mt.tensor(rng.standard_normal(shape).astype(np.float32)).to("bfloat16").cuda()

    fill = put(B, G, 1000, D)
    zeros = mt.zeros(B, dtype="int32", device="cuda")
    mt.kv_cache_append(cache, fill, fill, table, zeros)

    def step(q, k, v, starts, lengths):
        mt.kv_cache_append(cache, k, v, table, starts)
        return mt.kv_cache_attention(q, cache, table, lengths, window=700, sinks=4)

    from mtorch_b200.graphs import Graphed

    def index(x):
        return mt.tensor(np.full(B, x, np.int32), dtype="int32").cuda()

    g = Graphed(step, put(B, H, 1, D), put(B, G, 1, D), put(B, G, 1, D), index(1000), index(1001))
    for at in (1000, 1001, 1002):
        q, k, v = put(B, H, 1, D), put(B, G, 1, D), put(B, G, 1, D)
        got = host(g(q, k, v, index(at), index(at + 1)))
        np.testing.assert_array_equal(got, host(step(q, k, v, index(at), index(at + 1))))
