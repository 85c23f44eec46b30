"""The GLRU decoder at the ends of what it takes: no snapshots, no nodes, one of each; bfloat16 modules;
unknown nodes."""
import pytest
import torch

from spiral_amd.dtdg.models.decoder.sequentialDecoders import GLRU
from spiral_amd.dtdg.models.decoder.simpleDecoders import MLP

pytestmark = pytest.mark.gpu


def make(n_nodes=9, in_d=12, hid=20, layers=2):
    torch.manual_seed(3)
    return GLRU(in_d, hid, n_nodes, layers, MLP(hid, [6, 5], dropout=0.0)).to("cuda")


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("t,n", [(0, 4), (0, 9), (3, 0), (0, 0), (1, 1), (1, 9)])
def test_empty_and_smallest_sequences(dev, t, n, masked):
    dec = make()
    dec.train(False)  # (batch statistics of no rows do not exist)
    state = dec.memory_h.memory.clone()
    active = torch.ones(t, n, dtype=torch.bool, device=dev) if masked else None
    x = torch.randn(t, n, 12, device=dev, requires_grad=True)
    out = dec.forward_sequence(x, None, active)
    assert out.shape == ((t * n, 1) if masked else (t, n, 1))
    out.sum().backward()
    assert x.grad.shape == x.shape
    if t == 0 or n == 0:
        assert torch.equal(dec.memory_h.memory, state)
        assert all(p.grad is None or not p.grad.any() for p in dec.base_model.parameters())
    else:
        assert not torch.equal(dec.memory_h.memory[:, :n], state[:, :n])
        assert torch.equal(dec.memory_h.memory[:, n:], state[:, n:])


def test_a_snapshot_without_nodes(dev):
    dec = make()
    dec.train(False)
    state = dec.memory_h.memory.clone()
    for ids in (None, torch.zeros(0, dtype=torch.int64, device=dev)):
        out = dec((torch.randn(0, 12, device=dev), ids))
        assert out.shape == (0, 1) and torch.equal(dec.memory_h.memory, state)
