"""The gate's gradient of the gated linear recurrence, dz = d (h - c) a (1 - a), where the state h before a
step lies close to its candidate c: a state rounded on the way would leave little of the difference.

The tolerance is that of float32 arithmetic (16 u for each term of a step, u = 2^-24, carried on by the
recurrence itself) and of the one rounding of the stored result, half a step: 2^-8 of a value in bfloat16."""
import pytest
import torch

from spiral_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16
STORE = {F32: U, BF16: 2.0 ** -8}


def inputs(t, n, h, dtype, seed=0):
    """Candidates of 4 +- 0.25, logits around 1.5: states follow their candidates."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    gates = torch.cat([normal(t, n, h) + 1.5, 4 + 0.25 * normal(t, n, h)], 2).to(dtype)
    return gates, 4 + 0.25 * normal(n, h), normal(t, n, h).to(dtype), normal(n, h)


def gradients(gates, h0, on, g, g_last):
    """dgates and dh0 in float64 on the CPU, each with its tolerance."""
    kind, (t_end, n, h2) = gates.dtype, gates.shape
    hd = h2 // 2
    z, c = gates.double().cpu().split(hd, 2)
    a, rest = torch.sigmoid(z), torch.sigmoid(-z)
    state = h0.double().cpu()
    err = torch.zeros_like(state)
    states, errs = [], []
    for t in range(t_end):
        states.append(state)
        errs.append(err)
        there = on[t][:, None]
        err = torch.where(there, a[t] * err + 16 * U * (a[t] * state.abs() + rest[t] * c[t].abs()), err)
        state = torch.where(there, a[t] * state + rest[t] * c[t], state)
    e, err = g_last.double().cpu(), torch.zeros_like(state)
    value, tol = torch.zeros(t_end, n, h2, dtype=torch.float64), torch.zeros(t_end, n, h2, dtype=torch.float64)
    for t in reversed(range(t_end)):
        there = on[t][:, None]
        gt = g[t].double().cpu()
        d, e_d = e + gt, err + 2 * U * (e.abs() + gt.abs())
        gap = states[t] - c[t]
        dz, dc = d * gap * a[t] * rest[t], d * rest[t]
        e_gap = errs[t] + 4 * U * (states[t].abs() + c[t].abs())
        e_z = (e_d * gap.abs() + d.abs() * e_gap) * a[t] * rest[t] + (16 * U + STORE[kind]) * dz.abs()
        e_c = e_d * rest[t] + (8 * U + STORE[kind]) * dc.abs()
        value[t] = torch.where(there, torch.cat([dz, dc], 1), 0.0)
        tol[t] = torch.where(there, torch.cat([e_z, e_c], 1), 0.0)
        err = torch.where(there, a[t] * e_d + 16 * U * a[t] * d.abs(), e_d + 4 * U * d.abs())
        e = torch.where(there, a[t] * d, d)
    return value, tol + 1e-37, e, err + 1e-37


def check(gates, h0, on, g, g_last, batch_first=False):
    turn = (lambda v: v.transpose(0, 1).contiguous()) if batch_first else (lambda v: v)
    value, tol, e, e_tol = gradients(gates, h0, on.cpu(), g, g_last)
    leaf, start = turn(gates).clone().requires_grad_(), h0.clone().requires_grad_()
    h, last = ops.gated_scan(leaf, start, turn(on), batch_first)
    dgates, dh0 = torch.autograd.grad((h, last), (leaf, start), (turn(g), g_last))
    for name, got, want, allowed in (("dgates", turn(dgates), value, tol), ("dh0", dh0, e, e_tol)):
        off = (got.double().cpu() - want).abs() / allowed
        assert bool((off <= 1).all()), f"{name}: {int((off > 1).sum())} values off, {float(off.max()):.3g} of the tolerance"


# walked (few steps; 65536 lanes of four units and more), strands of a workgroup, steps split over workgroups; rows
# of fewer than four units and of no whole number of fours
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("t,n,h", [(12, 6, 20), (16, 3, 3), (19, 2100, 126), (22, 66000, 2), (40, 5, 3), (200, 3, 40),
                                   (65, 700, 12), (3001, 1, 24), (517, 9, 66), (1200, 1, 1)])
def test_states_that_follow_their_candidates(dev, t, n, h, dtype):
    gates, h0, g, g_last = inputs(t, n, h, dtype, seed=t + n + h)
    check(gates, h0, torch.ones(t, n, dtype=torch.bool, device=dev), g, g_last)
    on = torch.rand(t, n, generator=torch.Generator().manual_seed(1)) < 0.7
    on[:, ::5] = False
    check(gates, h0, on.to(dev), g, g_last, batch_first=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("t", range(1, 10))
@pytest.mark.parametrize("more", [0, 16])
def test_every_remainder_of_a_group(dev, t, more, dtype):
    """Sequences whose last group is not whole, walked and in strands."""
    gates, h0, g, g_last = inputs(t + more, 4, 6, dtype, seed=t)
    on = torch.ones(t + more, 4, dtype=torch.bool, device=dev)
    on[-1, 1] = on[0, 2] = on[-2:, 3] = False
    check(gates, h0, on, g, g_last)


def test_step_and_scan_train_alike(dev):
    """The recurrence as steps on a memory, the gradient of each step's own gates: what a scan of one
    step gives, to the bit of the stored type's rounding."""
    gates, h0, g, _ = inputs(1, 9, 20, BF16)
    one, two = gates[0].clone().requires_grad_(), gates.clone().requires_grad_()
    out = ops.gated_step(one, h0.clone())
    (a,) = torch.autograd.grad(out, one, g[0].float())
    (b,) = torch.autograd.grad(ops.gated_scan(two, h0)[0], two, g)
    assert torch.equal(a, b[0])


@pytest.mark.parametrize("t,n,h", [(11, 40, 20), (300, 2, 64), (3000, 1, 24)])
def test_captured_and_replayed(dev, t, n, h):
    """Forward and backward of bfloat16 sequences in one graph, in each layout: every replay on new inputs
    against the eager result, with eager work between the replays."""
    gates, h0, g, g_last = inputs(t, n, h, BF16)
    on = torch.rand(t, n, generator=torch.Generator().manual_seed(1)).to(dev) < 0.8
    leaf, start = gates.clone().requires_grad_(), h0.clone().requires_grad_()

    def work(leaf, start):
        h, last = ops.gated_scan(leaf, start, on)
        return [h.detach(), last.detach(), *torch.autograd.grad((h, last), (leaf, start), (g, g_last))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(leaf, start)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work(leaf, start)
    for k in range(3):
        new, new0 = inputs(t, n, h, BF16, seed=50 + k)[:2]
        with torch.no_grad():
            leaf.copy_(new)
            start.copy_(new0)
        graph.replay()
        torch.cuda.synchronize()
        want = work(new.requires_grad_(), new0.requires_grad_())
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_offsets_past_32_bits_of_many_nodes(dev, dtype):
    """Gates of more than 2^31 values: the last nodes come out as they do alone."""
    t, n, h = 5, (1 << 31) // (5 * 128) + 9, 64
    tail = inputs(t, 8, h, dtype)
    gates = torch.zeros(t, n, 2 * h, dtype=dtype, device=dev)
    gates[:, -8:] = tail[0]
    leaf, short = gates.requires_grad_(), tail[0].clone().requires_grad_()
    last = ops.gated_scan(leaf)[1]
    g_last = torch.zeros_like(last)
    g_last[-8:] = tail[3]
    (dgates,) = torch.autograd.grad(last, leaf, g_last)
    (want,) = torch.autograd.grad(ops.gated_scan(short)[1], short, tail[3])
    assert torch.equal(dgates[:, -8:], want) and not dgates[:, :8].any()


def test_offsets_past_32_bits_of_many_steps(dev):
    """A sequence of more than 2^31 values, split over workgroups: the gradient of its last steps is that of
    a short one from their first state on, up to the roundings of joined maps (16 u a step, 40 steps)."""
    t, h = (1 << 31) // 128 + 40, 64
    gates = torch.zeros(t, 1, 2 * h, device=dev)
    gates[-200:] = inputs(200, 1, h, F32)[0]
    leaf = gates.requires_grad_()
    hs, last = ops.gated_scan(leaf)
    g_last = torch.ones(1, h, device=dev)
    start, short = hs[-41].detach().clone(), gates[-40:].detach().clone().requires_grad_()
    (dgates,) = torch.autograd.grad(last, leaf, g_last)
    del hs
    (want,) = torch.autograd.grad(ops.gated_scan(short, start)[1], short, g_last)
    got = dgates[-40:]
    # dz cancels: the states (of about 4) are off by 16 u a step, carried on
    allowed = 40 * 16 * U * (want.abs() + (want[..., h:].abs() * 8).repeat(1, 1, 2)) + 1e-30
    assert bool(((got - want).abs() <= allowed).all())
