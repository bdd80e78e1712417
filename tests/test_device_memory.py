"""Tensors over device memory of another library."""
import numpy as np
import pytest

import mtorch_b200 as mt


@pytest.mark.parametrize("device", ["cpu", "nothing"])
def test_other_devices_are_refused(device):
    with pytest.raises((ValueError, RuntimeError)):
        mt.from_device_memory(4096, (4,), mt.float32, device=device)


def test_bad_strides_and_addresses_are_refused():
    for kw in (dict(strides=(1, 1)), dict(strides=(-1,))):
        with pytest.raises(ValueError):
            mt.from_device_memory(4096, (4,), mt.float32, **kw)
    for ptr in (4098, 0):
        with pytest.raises(ValueError):
            mt.from_device_memory(ptr, (4,), mt.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("device", [0, "cuda", "cuda:0", mt.device("cuda"), mt.device("cuda", 0)])
def test_devices_by_number_name_and_object(device):
    a = mt.tensor(np.arange(12, dtype=np.float32).reshape(3, 4)).cuda()
    b = mt.from_device_memory(a.data_ptr(), (4, 3), mt.float32, strides=(1, 4), device=device, owner=a)
    assert b.device.type == "cuda" and (b.device.index or 0) == 0
    np.testing.assert_array_equal(b.numpy(), a.numpy().T)
    np.testing.assert_array_equal((b * 2).numpy(), a.numpy().T * 2)
