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
        def gradients(ctx, saved, g):
            return 2 * saved[0] * g, None

    Square._bind("square")
    x = torch.tensor(3.0, requires_grad=True)
    y = Square.apply(x, None)
    (dx,) = torch.autograd.grad(y, x, create_graph=True)
    assert float(dx.detach()) == 6.0 and dx.requires_grad
    with pytest.raises(nv.SpmiError, match="square has no second derivative"):
        torch.autograd.grad(x + dx.square(), x)
    from torch.utils.checkpoint import checkpoint  # (it hands out what was saved once)

    (dx,) = torch.autograd.grad(checkpoint(lambda v: Square.apply(v, None), x, use_reentrant=False), x, create_graph=True)
    with pytest.raises(nv.SpmiError, match="second derivative"):
        dx.backward()
    g = torch.ones((), requires_grad=True)
    (dx,) = torch.autograd.grad(Square.apply(x, None), x, g, create_graph=True)
    with pytest.raises(nv.SpmiError, match="second derivative"):
        dx.backward()


F = torch.zeros


@pytest.mark.parametrize("name,call", [
    ("layer_norm", lambda d: ops.layer_norm(d(F(3, 4)))),
    ("layer_norm", lambda d: ops.layer_norm(F(3, 4), d(F(4)))),
    ("layer_norm", lambda d: ops.layer_norm(F(3, 4), None, d(F(4)))),
    ("gated_scan", lambda d: ops.gated_scan(d(F(3, 2, 8)))),
    ("gated_scan", lambda d: ops.gated_scan(F(3, 2, 8), d(F(2, 4)))),
    ("gated_step", lambda d: ops.gated_step(d(F(3, 8)), F(5, 4))),
    ("gated_step", lambda d: ops.gated_step(F(3, 8), d(F(5, 4)))),
    ("quantize_rows_int8", lambda d: ops.quantize_rows_int8(d(F(3, 4)))),
    ("linear_int8", lambda d: ops.linear_int8(d(F(3, 4)), F(5, 4, dtype=torch.int8), F(5))),
    ("linear_int8", lambda d: ops.linear_int8(F(3, 4), F(5, 4, dtype=torch.int8), d(F(5)))),
    ("linear_int8", lambda d: ops.linear_int8(F(3, 4), F(5, 4, dtype=torch.int8), F(5), d(F(5)))),
])
def test_a_forward_mode_derivative_is_refused(name, call):
    """A dual tensor does not require a gradient; its tangent must not get lost all the same."""
    fwd = torch.autograd.forward_ad
    with fwd.dual_level(), pytest.raises(nv.SpmiError, match=f"{name} has no forward-mode derivative"):
        call(lambda t: fwd.make_dual(t, torch.ones_like(t)))
    with fwd.dual_level(), torch.no_grad(), pytest.raises(nv.SpmiError, match="forward-mode"):
        call(lambda t: fwd.make_dual(t, torch.ones_like(t)))
    with fwd.dual_level(), pytest.raises(nv.SpmiError, match="GPU"):  # no tangent: the usual answer to a CPU tensor
        call(lambda t: t)


def test_forward_mode_through_the_function_transforms_is_refused():
    x = torch.ones(3, 4)
    with pytest.raises(nv.SpmiError, match="forward-mode"):
        torch.func.jvp(ops.layer_norm, (x,), (x,))


def test_more_threads_than_a_grid_holds_are_refused():
    """A thread for each four units of a node, one at least; two for each row of the projection."""
    lib = nv.lib()
    scan = lib.spmi_gated_scan_fwd
    for n, h in ((1 << 32, 1), ((1 << 32) - 255, 2), ((1 << 31) - 127, 5)):
        assert scan(P, 0, 2 * h, 2 * h, None, 0, None, 0, 0, 1, n, h, P, h, h, P, None, 0, None) == -5
    lin, need = lib.spmi_linear_i8, lib.spmi_linear_i8_workspace_bytes
    for m in ((1 << 31) - 511, (1 << 31) - 1):
        assert lin(P, 1, 1, m, 1, P, 1, P, 1, None, 0, 0.0, P, 1, 1, P, need(m, 1, 1), None) == -5
        assert lib.spmi_quantize_rows_i8(P, 1, 1, m, 1, P, 1, P, None) == -5


@pytest.mark.parametrize("ids", [[0, 1, 5], [-1, 0, 1], torch.tensor([2, 3, 7])])
def test_sequences_of_unknown_nodes_are_refused(ids):
    """torch's indexing on the GPU would end the process."""
    from spiral_amd.dtdg.models.decoder.sequentialDecoders import GLRU
    from spiral_amd.dtdg.models.decoder.simpleDecoders import MLP

    dec = GLRU(6, 4, 5, 1, MLP(4, [3]))
    with pytest.raises(ValueError, match="nodes 0 to 4"):
        dec.forward_sequence(torch.zeros(2, 3, 6), ids)
