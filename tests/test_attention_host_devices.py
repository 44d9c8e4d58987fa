"""Positions, lengths, masks, gains and 8-bit outputs on another device than the current one are refused by the binding; checked without a GPU, with stand-ins for
torch tensors and a library that must not be reached."""
import pytest
import torch

import darknet_b200 as dn
from darknet_b200 import api


class OnDevice:
    """What the binding asks of a CUDA tensor."""
    is_cuda = True

    def __init__(self, device, dtype, *shape):
        self.device, self.dtype, self.shape = device, dtype, torch.Size(shape)

    def is_contiguous(self):
        return True

    def get_device(self):
        return self.device

    def stride(self, i):
        return (self.shape[1] * self.shape[2], self.shape[2], 1)[i]

    def data_ptr(self):
        return 0x100000


@pytest.fixture
def reached(monkeypatch):
    """Device 1 is current; the names of the entry points that were called."""
    calls = []
    monkeypatch.setattr(api, "_device", lambda: 1, raising=False)
    monkeypatch.setattr(api, "_function", lambda name: lambda *a: calls.append(name) or 0)
    return calls


def tensor(n, h, w, c):
    return dn.Tensor(0x10000, dn.NHWC, dn.BF16, n, c, h, w, (c + 7) // 8 * 8)


def calls():
    q, k, x = tensor(2, 1, 5, 128), tensor(2, 3, 7, 64), tensor(2, 3, 3, 60)
    rope, attention = dn.RopePlan(64, 2, (8, 12, 12)), dn.CrossAttentionPlan(4, 2, 32)
    I, F = torch.int32, torch.float32
    return {
        "positions": lambda d: rope.forward(q, q, OnDevice(d, I, 10, 3), stream=0),
        "lengths": lambda d: attention.forward(q, k, k, q, lengths=OnDevice(d, I, 2), stream=0),
        "mask": lambda d: attention.forward(q, k, k, q, mask=OnDevice(d, torch.bool, 2, 5, 21), stream=0),
        "gain": lambda d: dn.rmsnorm(x, x, OnDevice(d, F, 60), stream=0),
        "e4m3": lambda d: dn.rmsnorm(x, x, e4m3=OnDevice(d, torch.uint8, 2, 3, 3, 64), scales=OnDevice(1, F, 2, 3, 3, 1), stream=0),
        "scales": lambda d: dn.rmsnorm(x, x, e4m3=OnDevice(1, torch.uint8, 2, 3, 3, 64), scales=OnDevice(d, F, 2, 3, 3, 1), stream=0)}


@pytest.mark.parametrize("what", ["positions", "lengths", "mask", "gain", "e4m3", "scales"])
def test_arrays_on_another_device(what, reached):
    call = calls()[what]
    with pytest.raises(ValueError, match=f"{what}.*device 0"):
        call(0)
    assert not reached
    call(1)
    assert len(reached) == 1


def test_values_in_8_bits_come_with_their_scales(reached):
    x = tensor(2, 3, 3, 60)
    with pytest.raises(ValueError, match="scales"):
        dn.rmsnorm(x, x, e4m3=OnDevice(1, torch.uint8, 2, 3, 3, 64), stream=0)
    with pytest.raises(ValueError, match="scales"):                         # they would stay as they are
        dn.rmsnorm(x, x, scales=OnDevice(1, torch.float32, 2, 3, 3, 1), stream=0)
    assert not reached
