"""A decoder's weights are saved, loaded and moved as those of any module are."""
import numpy as np
import pytest

import mtorch_b200 as mt
from mtorch_b200 import nn
from mtorch_b200.decoder import Decoder, Linear4
from test_gpu_decoder import TOL, forward, host, place

pytestmark = pytest.mark.gpu


def make(seed, **kw):
    mt.manual_seed(seed)
    return Decoder(vocab=90, width=128, layers=2, heads=2, mlp=96, window=20, sinks=2, page_size=16, **kw)


def logits(model, steps=2):
    ids = np.arange(24).reshape(2, 12) % 90
    model.start(2, 12 + steps)
    out = [model.prefill(mt.tensor(ids)).float().numpy()]
    for i in range(steps):
        out.append(model.step(mt.tensor(np.array([3 + i, 40 + i]))).float().numpy())
    return np.stack(out)


def test_state_dict_holds_every_weight():
    a, b = make(1), make(2)
    want = logits(a)
    assert np.abs(want - logits(b)).max() > 0
    sd = {k: v.cpu() for k, v in a.state_dict().items()}
    for i in range(2):
        for name in ("qkv", "out", "fc1", "fc2"):
            assert {f"layers.{i}.{name}.words", f"layers.{i}.{name}.scales", f"layers.{i}.{name}.bias"} <= set(sd)
    assert sd["layers.0.qkv.words"].dtype is mt.int32 and sd["layers.0.qkv.scales"].dtype is mt.bfloat16
    b.load_state_dict(sd)
    np.testing.assert_array_equal(logits(b), want)
    with pytest.raises(KeyError):
        b.load_state_dict({"layers.0.qkv.weights": sd["layers.0.qkv.words"]})
    with pytest.raises(KeyError):
        b.load_state_dict({"layers.7.qkv.weight": sd["layers.0.qkv.words"]})


def test_there_and_back():
    a = make(3)
    want = logits(a)
    a.cpu()
    assert all(p.device.type == "cpu" for p in a.parameters()) and a.frequencies.device.type == "cpu"
    a.cuda()
    assert all(p.device.type == "cuda" for p in a.parameters()) and a.frequencies.device.type == "cuda"
    np.testing.assert_array_equal(logits(a), want)


def test_a_cast_leaves_the_packed_weights():
    a = make(4)
    words = a.layers[0].qkv.words.numpy().copy()
    scales = a.layers[0].qkv.scales.float().numpy().copy()
    want = logits(a)
    a.half()
    q = a.layers[0].qkv
    assert q.words.dtype is mt.int32 and q.scales.dtype is mt.bfloat16 and a.frequencies.dtype is mt.float32
    assert q.bias.dtype is mt.float16 and a.token_embedding.dtype is mt.float16
    np.testing.assert_array_equal(q.words.numpy(), words)
    np.testing.assert_array_equal(q.scales.float().numpy(), scales)
    got = logits(a)
    assert np.abs(got - want).max() <= 40 * 2.0 ** -9 * np.abs(want).max()  # bf16 activations against f16 ones


def test_a_floating_weight_is_packed_as_it_is_loaded():
    """The state dict of the `Linear` that the layer stands for."""
    rng = np.random.default_rng(5)
    floating = nn.Linear(100, 70, device="cuda", dtype="bfloat16")
    layer = Linear4(nn.Linear(100, 70, device="cuda", dtype="bfloat16"), 32)
    x = mt.tensor(rng.standard_normal((3, 100)).astype(np.float32)).to("bfloat16").cuda()
    for sd in (floating.state_dict(), {k: v.cpu() for k, v in floating.state_dict().items()}):
        layer.words.fill_(0)
        layer.load_state_dict(sd)
        np.testing.assert_array_equal(layer(x).float().numpy(), Linear4(floating, 32)(x).float().numpy())
    with pytest.raises(ValueError):
        layer.load_state_dict({"weight": mt.zeros(70, 99, dtype="bfloat16", device="cuda")})
    m = make(6)
    w = mt.tensor(rng.standard_normal((128, 96)).astype(np.float32) * 0.1)
    m.load_state_dict({"layers.1.fc2.weight": w})
    np.testing.assert_array_equal(m.layers[1].fc2.words.numpy(), mt.Weight4.pack(w.cuda(), 64).words.numpy())


def test_float32_prompt_and_steps():
    """Steps follow a prompt in float32 too."""
    mt.manual_seed(7)
    model = Decoder(vocab=90, width=128, layers=2, heads=2, kv_heads=1, mlp=96, window=20, sinks=2, page_size=16, dtype="float32")
    n, s, steps = 2, 30, 4
    ids = np.random.default_rng(0).integers(0, 90, (n, s + steps))
    want = forward(model, host(model.token_embedding)[ids], place(0, 0, s + steps), s)
    model.start(n, s + steps)
    got = [host(model.prefill(mt.tensor(ids[:, :s])))]
    for i in range(steps):
        got.append(host(model.step(mt.tensor(ids[:, s + i]))))
    for i, g in enumerate(got):
        assert np.abs(g - want[:, s - 1 + i]).max() <= TOL * np.abs(want).max(), i
    assert model.generate(mt.tensor(ids[:, :s]), 3).shape == (n, 3)
