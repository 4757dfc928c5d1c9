"""The differentiable forms look for a capture on the device of their operands, not on the current one (with stand-ins: no GPU is needed)."""
import pytest
import torch

from lightly_trian_quant_b200 import grad
from lightly_trian_quant_b200._lib import KfError


class _Leaf:
    """a tensor on a device as far as the look goes"""

    def __init__(self, index, requires_grad=True):
        self.device, self.requires_grad = torch.device("cuda", index), requires_grad


@pytest.fixture
def capturing(monkeypatch):
    """device 1 captures on its current stream, device 0 does not; device 0 is the current one"""
    current = [0]

    class Guard:
        def __init__(self, device):
            self.device = torch.device(device).index

        def __enter__(self):
            self.before, current[0] = current[0], self.device

        def __exit__(self, *exc):
            current[0] = self.before

    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: current[0] == 1)
    return current


def test_a_capture_on_the_operands_device_is_seen(capturing):
    with torch.enable_grad():
        grad._eager(_Leaf(0), None, _Leaf(0, False))
        with pytest.raises(KfError, match="capture"):
            grad._eager(_Leaf(1, False), None, _Leaf(1))
        grad._eager(_Leaf(1, False))                               # no gradient wanted: like the operator
    with torch.no_grad():
        grad._eager(_Leaf(1))
    with pytest.raises(KfError, match="capture"):
        grad._eager_backward(_Leaf(1))
    grad._eager_backward(_Leaf(0))
    assert capturing[0] == 0


def test_a_capture_on_another_device_is_none_of_theirs(capturing):
    capturing[0] = 1
    with torch.enable_grad():
        grad._eager(_Leaf(0))
        with pytest.raises(KfError, match="capture"):
            grad._eager(_Leaf(1))
    assert capturing[0] == 1
