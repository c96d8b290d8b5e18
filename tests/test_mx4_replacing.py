"""quantize_linears_ leaves alone what it cannot stand in for."""

import pytest
import torch
import torch.nn as nn

from sparseflow_amd import _lib
from sparseflow_amd.Ops import MX4Linear, SparseLinear, quantize_linears_


class Doubled(nn.Linear):
    def forward(self, x):
        return 2 * super().forward(x)


def test_subclasses_with_a_forward_or_an_owner_of_their_own():
    """A subclass may compute something else, and an nn.MultiheadAttention reads its projection's weight by itself."""
    net = nn.ModuleDict({"a": Doubled(32, 32), "b": nn.MultiheadAttention(32, 2, batch_first=True), "c": nn.Linear(32, 32),
                         "d": SparseLinear(32, 8)})
    x = torch.randn(2, 3, 32)
    with torch.no_grad():
        want = net["a"](x), net["b"](x, x, x)[0]
        assert quantize_linears_(net) == 2
        assert isinstance(net["c"], MX4Linear) and isinstance(net["d"], MX4Linear)
        assert torch.equal(net["a"](x), want[0]) and torch.equal(net["b"](x, x, x)[0], want[1])


def test_a_net_that_is_refused_is_left_as_it_was():
    net = nn.Sequential(nn.Linear(32, 32), nn.Linear(32, 8).double())
    with pytest.raises(_lib.UnsupportedError):
        quantize_linears_(net)
    assert [type(m) for m in net] == [nn.Linear, nn.Linear]
