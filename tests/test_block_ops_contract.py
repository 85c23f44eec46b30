"""What the C entry points and the wrappers of the gated-linear-recurrence block hold to, looked at without
a GPU: every call below returns or raises before any HIP call."""
import pytest
import torch

from spiral_amd import _native as nv
from spiral_amd import ops

P = 64  # stands for a pointer


def test_states_kept_for_the_backward_pass():
    lib = nv.lib()
    states = lib.spmi_gated_scan_states
    # a state between two groups of steps: of four where a thread walks them (up to 16, or many channels), of two
    assert [states(t, 3, 8) for t in (0, 1, 4, 5, 8, 9, 16)] == [0, 0, 0, 1, 1, 2, 3]
    assert [states(t, 3, 8) for t in (17, 18, 19, 700)] == [8, 8, 9, 349]
    assert states(32, 50_000, 128) == 7 and states(5, 0, 8) == 0 and states(5, 3, 0) == 0
    back = lib.spmi_gated_scan_bwd

    def call(dtype, t, h, states):
        return back(P, dtype, 16, 16, None, 0, None, 0, 0, t, 1, 8, h, 8, 8, states, None, 0, 0, None, 0, P, 16, 16, None,
                    None, 0, None)

    assert call(0, 5, None, None) == call(0, 5, None, P) == -1      # float32: the states are those in h
    assert call(1, 5, P, None) == call(1, 5, None, None) == -1      # bfloat16: those kept beside it
    assert lib.spmi_gated_scan_fwd_saved(P, 0, 8, 8, None, 0, None, 0, 0, 1, 1, 4, P, 4, 4, None, P, None, 0, None) == -1
    with pytest.raises(nv.SpmiError):
        ops.gated_scan(torch.zeros(3, 2, 8, dtype=torch.bfloat16))


def test_a_second_derivative_is_refused_whatever_the_incoming_gradient():
    """The base of the operators on the CPU, with x^2 in the place of a kernel: at x = 3 the derivative of
    x + (dx^2/dx)^2 is 1 + 8 x = 25; taking the backward pass' result for a constant would give 1."""
    from spiral_amd.block_ops import _Operator

    class Square(_Operator):
        @staticmethod
        def forward(ctx, x, y):
            ctx.save_for_backward(x)
            return x * x

        @staticmethod
        def gradients(ctx, g):
            return 2 * ctx.saved_tensors[0] * g, None

    Square._bind("square")
    x = torch.tensor(3.0, requires_grad=True)
    y = Square.apply(x, None)
    (dx,) = torch.autograd.grad(y, x, create_graph=True)
    assert float(dx.detach()) == 6.0 and dx.requires_grad
    with pytest.raises(nv.SpmiError, match="square has no second derivative"):
        torch.autograd.grad(x + dx.square(), x)
    g = torch.ones((), requires_grad=True)
    (dx,) = torch.autograd.grad(Square.apply(x, None), x, g, create_graph=True)
    with pytest.raises(nv.SpmiError, match="second derivative"):
        dx.backward()
