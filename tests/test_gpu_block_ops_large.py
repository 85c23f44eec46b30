"""Layer norm's gradient and the 8-bit projection of short rows on matrices of more than 2^31 values: rows past
that come out as they do alone."""
import pytest
import torch

from spiral_amd import ops

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def rand(*shape, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(BF16)


@pytest.mark.parametrize("d", [64, 1000, 4096])
def test_layer_norm_backward(dev, d):
    m = (1 << 31) // d + 5
    x, g = torch.zeros(m, d, dtype=BF16, device=dev), torch.zeros(m, d, dtype=BF16, device=dev)
    x[-3:], g[-3:] = rand(3, d), rand(3, d, seed=1)
    x, w = x.requires_grad_(), torch.ones(d, device=dev).requires_grad_()
    dx, dw = torch.autograd.grad(ops.layer_norm(x, w), (x, w), g)
    few, one = x[-3:].detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
    want, want_w = torch.autograd.grad(ops.layer_norm(few, one), (few, one), g[-3:].clone())
    assert torch.equal(dx[-3:], want) and not dx[:5].any()
    # three rows' terms in another order, each sum rounded twice, among zeros
    assert bool(((dw - want_w).abs() <= 4 * 2.0 ** -24 * 3 * 16).all())


@pytest.mark.parametrize("k", [128, 500])
def test_projection_in_one_pass(dev, k):
    m = (1 << 31) // k + 70
    x = torch.zeros(m, k, dtype=BF16, device=dev)
    x[-70:] = rand(70, k)
    w, s = torch.randint(-127, 128, (33, k), device=dev, dtype=torch.int8), torch.rand(33, device=dev)
    assert torch.equal(ops.linear_int8(x, w, s)[-70:], ops.linear_int8(x[-70:].clone(), w, s))
