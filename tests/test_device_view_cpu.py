"""ffi.DeviceView.of refuses what is not GPU memory (a kernel given a host pointer would fault)."""
import pytest
import torch

from hodu_amd import ffi


def test_a_tensor_of_the_cpu_is_refused():
    for t in (torch.zeros(4), torch.zeros(4, 4)[:, 1]):
        with pytest.raises(ValueError, match="cpu"):
            ffi.DeviceView.of(t)
