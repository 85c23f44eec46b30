"""The gates of the recurrence, a = 1 / (1 + e^-z) and 1 - a, where one of them is small.

In u = 2^-24: e^-|z| is off by 2 (the exponential instruction, one unit in the last place) and 1 (its
correction), the reciprocal of 1 + e^-|z| by 1 and 2, their product by 1: 7 u of the value, for which 8
are allowed.  At |z| = 85 e^-|z| is 1.2e-37, still a normal number."""
import pytest
import torch

from spiral_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("low,high", [(0.0, 1.0), (1.0, 20.0), (20.0, 40.0), (40.0, 85.0)])
def test_small_gates_keep_their_digits(dev, low, high):
    h = 4096
    z = torch.linspace(low, high, h, device=dev)
    small = 1 / (1 + torch.exp(z.double().cpu()))
    one, zero = torch.ones(1, h, device=dev), torch.zeros(1, h, device=dev)
    # from nothing to a candidate of one: 1 - a; from a state of one to a candidate of nothing: a
    for gates, h0 in ((torch.cat([z[None], one], 1), zero), (torch.cat([-z[None], zero], 1), one)):
        states, last = ops.gated_scan(gates[None], h0)
        for got in (states[0, 0], last[0], ops.gated_step(gates, h0.clone())[0]):
            off = (got.double().cpu() - small).abs() / small
            assert float(off.max()) <= 8 * U, float(off.max()) / U
    leaf = torch.cat([z[None], one], 1)[None].requires_grad_()
    (dgates,) = torch.autograd.grad(ops.gated_scan(leaf, zero)[1], leaf, one)  # dc = 1 - a
    off = (dgates[0, 0, h:].double().cpu() - small).abs() / small
    assert float(off.max()) <= 8 * U, float(off.max()) / U
