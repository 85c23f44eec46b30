"""What autograd may and may not do with layer norm, the gated linear recurrence and the 8-bit
projection."""
import pytest
import torch

from spiral_amd import _native as nv
from spiral_amd import ops

pytestmark = pytest.mark.gpu


def rand(*shape, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda")


def cases():
    w, b = rand(12, seed=1), rand(12, seed=2)
    h0 = rand(3, 4, seed=3)
    yield "layer_norm", lambda x: ops.layer_norm(x, w, b), rand(5, 12)
    yield "layer_norm", lambda x: ops.layer_norm(rand(5, 12), x, b), w
    for dtype in (torch.float32, torch.bfloat16):
        gates = rand(6, 3, 8, seed=4).to(dtype)
        yield "gated_scan", lambda x: ops.gated_scan(x, h0)[0], gates
        yield "gated_scan", lambda x: ops.gated_scan(x, h0)[1], gates
    yield "gated_step", lambda x: ops.gated_step(x, h0.clone()), rand(3, 8, seed=5)


@pytest.mark.parametrize("which", range(7))
def test_second_derivatives_are_refused(dev, which):
    name, f, at = list(cases())[which]
    x = at.clone().requires_grad_()
    (want,) = torch.autograd.grad(f(x).sum(), x)
    (dx,) = torch.autograd.grad(f(x).sum(), x, create_graph=True)  # an incoming gradient of constants
    assert torch.equal(dx, want)
    with pytest.raises(nv.SpmiError, match=f"{name} has no second derivative"):
        (x.sum() + dx.float().square().sum()).backward()


def test_gradients_of_one_input_move_with_another(dev):
    """The weight's gradient depends on x, the gates' on h0: neither comes out as a constant."""
    x, w = rand(5, 12).requires_grad_(), rand(12, seed=1).requires_grad_()
    (dw,) = torch.autograd.grad(ops.layer_norm(x, w).sum(), w, create_graph=True)
    with pytest.raises(nv.SpmiError, match="second derivative"):
        torch.autograd.grad(dw.square().sum(), x)
    gates, h0 = rand(6, 3, 8).requires_grad_(), rand(3, 4, seed=1).requires_grad_()
    (dg,) = torch.autograd.grad(ops.gated_scan(gates, h0)[0].sum(), gates, create_graph=True)
    with pytest.raises(nv.SpmiError, match="second derivative"):
        torch.autograd.grad(dg.square().sum(), h0)


def test_a_recorded_backward_pass_is_an_ordinary_gradient(dev):
    x, w = rand(40, 12).requires_grad_(), rand(12, seed=1).requires_grad_()
    ops.layer_norm(x, w).sum().backward()
    want = x.grad, w.grad
    x.grad = w.grad = None
    ops.layer_norm(x, w).sum().backward(create_graph=True)
    assert torch.equal(x.grad, want[0]) and torch.equal(w.grad, want[1])
    x.grad = w.grad = None


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_under_activation_checkpointing(dev, dtype):
    """Forward runs again before the backward pass: the same gradients to the bit."""
    from torch.utils.checkpoint import checkpoint

    gates, h0 = rand(40, 3, 16).to(dtype).requires_grad_(), rand(3, 8, seed=1).requires_grad_()
    w = rand(8, seed=2).requires_grad_()

    def block(g, s, v):
        h, last = ops.gated_scan(g, s)
        return ops.layer_norm(h, v), last

    def grads(outs):
        return torch.autograd.grad(outs[0].float().sum() + outs[1].sum(), (gates, h0, w))

    want = grads(block(gates, h0, w))
    got = grads(checkpoint(block, gates, h0, w, use_reentrant=False))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_states_may_move_on_before_the_backward_pass(dev, dtype):
    """The start of a scan is a row of the node memory that later steps overwrite: what the backward pass needs
    of it was taken in the forward pass, or the change is noticed."""
    gates, memory = rand(30, 3, 16).to(dtype).requires_grad_(), rand(3, 8, seed=1)
    (want,) = torch.autograd.grad(ops.gated_scan(gates, memory)[1].sum(), gates)
    last = ops.gated_scan(gates, memory)[1]
    ops.gated_step(rand(3, 16, seed=2), memory)
    with pytest.raises(RuntimeError, match="modified"):
        torch.autograd.grad(last.sum(), gates)
    assert want.shape == gates.shape
