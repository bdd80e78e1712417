"""Memory that a captured graph's launches refer to stays theirs for as long as the graph exists."""
import gc
import importlib
import weakref

import numpy as np
import pytest

import mtorch_b200 as mt
from mtorch_b200 import _lib, graphs, runtime

tensor = importlib.import_module("mtorch_b200.tensor")  # (the package's `tensor` is the function)


class _Buffer:
    def __init__(self, nbytes, idx):
        self.nbytes, self.ptr = nbytes, 4096

    def data_ptr(self):
        return self.ptr

    def numel(self):
        return self.nbytes


class _Lib:
    """The library calls of a capture, without a device."""

    def mt_cuda_launch_count(self):
        return 0

    def mt_cuda_graph_begin(self, stream):
        return 0

    def mt_cuda_graph_end(self, stream, out):
        return 0


class _Input:
    def _idx(self):
        return 5

    def clone(self):
        return self


@pytest.mark.parametrize("during", [[100], [100, 100000], [100, 100000, 10000000]])
def test_a_graph_keeps_the_workspaces_it_was_captured_with(monkeypatch, during):
    monkeypatch.setattr(tensor, "_alloc", _Buffer)
    monkeypatch.setattr(_lib, "lib", lambda: _Lib())
    monkeypatch.setattr(runtime, "synchronize", lambda: None)
    monkeypatch.setattr(runtime, "stream_ptr", lambda idx: 1)
    seen = []

    def fn(x):
        if 5 in runtime.capturing:  # the capture asks for more than the calls before it
            for n in during:
                tensor.workspace(n, 5)
                seen.append(weakref.ref(tensor._WS[5]))
        else:
            tensor.workspace(100, 5)
        return x

    try:
        g = graphs.Graphed(fn, _Input())
        assert 5 not in runtime.capturing
        tensor.workspace(10 ** 9, 5)  # a later call outgrows it
        gc.collect()
        assert len(seen) == len(during) and all(r() is not None for r in seen)
        del g
        gc.collect()
        assert all(r() is None for r in seen)
    finally:
        tensor._WS.pop(5, None)


@pytest.mark.gpu
def test_replay_after_the_workspace_grew():
    """A decoder's step whose split attention has partial results in the workspace, replayed after a call that needs a
    larger one: the old buffer is nobody else's."""
    rng = np.random.default_rng(1)
    B, H, G, D, page, per = 1, 4, 1, 64, 16, 600

    def put(*shape):
        return mt.tensor(rng.standard_normal(shape).astype(np.float32)).to("bfloat16").cuda()

    cache = mt.KVCache4.empty(B * per, page, G, D)
    table = mt.tensor(np.arange(B * per, dtype=np.int32).reshape(B, per), dtype="int32").cuda()
    fill = put(B, G, per * page, D)
    mt.kv_cache_append(cache, fill, fill, table, mt.zeros(B, dtype="int32", device="cuda"))
    lengths = mt.tensor(np.full(B, per * page, np.int32), dtype="int32").cuda()

    def step(q):
        return mt.kv_cache_attention(q, cache, table, lengths)

    q = put(B, H, 1, D)
    want = step(q).float().numpy()
    g = graphs.Graphed(step, q)
    ws = tensor._WS[0]
    lo, hi = ws.ptr, ws.ptr + ws.nbytes
    size = ws.nbytes
    del ws
    tensor.workspace(4 * size + (64 << 20), 0)
    gc.collect()
    others = [mt.zeros(size // 2, dtype="bfloat16", device="cuda") for _ in range(4)]
    assert all(t.data_ptr() + size <= lo or t.data_ptr() >= hi for t in others)
    np.testing.assert_array_equal(g(q).float().numpy(), want)
    assert all((t.float().numpy() == 0).all() for t in others)


@pytest.mark.gpu
def test_empty_cache_leaves_a_graphs_temporaries():
    """What a capture freed is written again by every replay: it stays until the graph is gone."""
    rng = np.random.default_rng(2)
    x = mt.tensor(rng.standard_normal((1024, 1024)).astype(np.float32)).to("bfloat16").cuda()

    def fn(t):
        return t * 2 + t * 3

    want = fn(x).float().numpy()
    g = graphs.Graphed(fn, x)
    mt.cuda.empty_cache()
    held = runtime.memory_stats(0)["cached_bytes"]
    assert held >= 2 * x.numel() * 2  # the two products
    others = [mt.zeros(1024, 1024, dtype="bfloat16", device="cuda") for _ in range(4)]
    np.testing.assert_array_equal(g(x).float().numpy(), want)
    assert all((t.float().numpy() == 0).all() for t in others)
    del g
    gc.collect()
    mt.cuda.empty_cache()
    assert runtime.memory_stats(0)["cached_bytes"] < held
