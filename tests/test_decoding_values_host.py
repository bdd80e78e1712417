"""Choices of the decoder's operators that are made on the host, by sizes and types alone."""
import ctypes as C

import pytest

from mtorch_b200 import _lib as L


def reads_packed_weight(M, N, K, group, dtype):
    d = L.LinearWeight4Desc(M, N, K, group, dtype, 16, K, 16, 16, None, 16, N)
    return L.lib().mt_cuda_linear_weight4_workspace_size(C.byref(d)) == 0


@pytest.mark.parametrize("group", [32, 64, 128])
def test_few_rows_of_a_wide_weight_need_no_copy(group):
    """One token of a projection from 28672 columns is read from the packed weight, not through a copy of four times its size."""
    for dtype in (L.MT_BF16, L.MT_F16):
        assert reads_packed_weight(1, 8192, 28672, group, dtype)
    assert reads_packed_weight(1, 8192, 28672 if group == 128 else 20480, group, L.MT_F32)  # (three operand rows)
    assert reads_packed_weight(4, 8192, 28672, group, L.MT_BF16)


def test_many_launches_give_way_to_the_copy():
    """fp32 rows of 8192 columns go three to a launch, of 16384 one: 64 of them would read the weight 22 or 64 times."""
    for K in (8192, 16384):
        assert not reads_packed_weight(64, 28672, K, 128, L.MT_F32)
        assert reads_packed_weight(3 if K == 8192 else 1, 28672, K, 128, L.MT_F32)
    assert not reads_packed_weight(64, 28672, 16384, 128, L.MT_BF16)
    assert reads_packed_weight(64, 2304, 768, 64, L.MT_BF16)
    assert not reads_packed_weight(65, 2304, 768, 64, L.MT_BF16)
    assert reads_packed_weight(100, 64, 0, 64, L.MT_BF16)  # (no columns: the bias alone)


def test_a_workspace_off_its_alignment_is_refused():
    """Partial results and copies are stored 16 bytes at a time: nothing is launched on a workspace that is not aligned."""
    lib = L.lib()
    st = (1 << 20, 1 << 14, 64, 1)
    w = L.WindowAttentionDesc(1, 4, 2, 1, 8192, 64, L.MT_BF16, 1, 0, 0, None, None, 16, st, 16, st, 16, st, 16, st, 0.125)
    need = lib.mt_cuda_window_attention_workspace_size(C.byref(w))
    assert need and lib.mt_cuda_window_attention(C.byref(w), 8, need, None) == L.MT_ERR_INVALID
    assert lib.mt_cuda_window_attention(C.byref(w), 16, need - 1, None) == L.MT_ERR_WORKSPACE
    cache = L.KvCache4Desc(1024, 16, 2, 64, 16, 16, 16, 16)
    c = L.KvCache4AttentionDesc(cache, 1, 4, 1, L.MT_BF16, 0, 0, 16, 1024, 1024, 16, 16, st, 16, st, 0.125)
    need = lib.mt_cuda_kv_cache4_attention_workspace_size(C.byref(c))
    assert need and lib.mt_cuda_kv_cache4_attention(C.byref(c), 8, need, None) == L.MT_ERR_INVALID
    d = L.LinearWeight4Desc(500, 80, 256, 64, L.MT_BF16, 16, 256, 16, 16, None, 16, 80)
    need = lib.mt_cuda_linear_weight4_workspace_size(C.byref(d))
    assert need and lib.mt_cuda_linear_weight4(C.byref(d), 8, need, None) == L.MT_ERR_INVALID
