"""The GLRU decoder at the ends of what it takes: no snapshots, no nodes, one of each; bfloat16 modules."""
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


def restated(dec, xs):
    """The decoder's states over the snapshots `xs` [T, N, D] of every node in float64, and by how much the last
    layer's may be off where every layer rounds its normalised rows, its gates and its states to
    bfloat16 (half a step: 2^-8 of the largest value)."""
    u8 = 2.0 ** -8
    p = {k: v.detach().double().cpu() for k, v in dec.base_model.named_parameters()}
    states = dec.memory_h.memory.double().cpu()
    off = [0.0] * dec.n_layers
    out = []
    for x in xs.double().cpu():
        e_x = u8 * float(x.abs().max())
        for k in range(dec.n_layers):
            w, b = p[f"norms.{k}.weight"], p[f"norms.{k}.bias"]
            u = torch.nn.functional.layer_norm(x, (x.shape[1],), w, b)
            # mean and deviation of a row move by at most e_x each: (1 + 1 + |xh|) e_x / deviation
            xh = ((u - b) / w).abs().max()
            e_u = float((2 + xh) * w.abs().max() / x.std(1, correction=0).min()) * e_x + u8 * float(u.abs().max())
            wk = p[f"projections.{k}.weight"]
            g = u @ wk.t() + p[f"projections.{k}.bias"]
            e_g = float(wk.abs().sum(1).max()) * e_u + u8 * float(g.abs().max())
            z, c = g.chunk(2, 1)
            reach = float((states[k] - c).abs().max())
            x = torch.sigmoid(z) * states[k] + torch.sigmoid(-z) * c
            off[k] = max(off[k], e_g) + e_g * reach / 4  # a convex combination of the two, and its weight's change
            states[k] = x
            e_x = off[k] + u8 * float(x.abs().max())
        out.append(x)
    return torch.stack(out), e_x


@pytest.mark.parametrize("head", [torch.bfloat16, torch.float32])
def test_bfloat16_modules_step_and_scan(dev, head):
    x = torch.randn(3, 9, 12, device=dev)
    got = []
    for sequence in (False, True):
        dec = make()
        dec.base_model.bfloat16()
        dec.simple_decoder.to(head)
        want, allowed = restated(dec, x)
        seen = []
        dec.simple_decoder.register_forward_pre_hook(lambda m, a: seen.append(a[0][0]))
        out = [dec.forward_sequence(x.bfloat16())] if sequence else [dec((x[t].bfloat16(), torch.arange(9))) for t in range(3)]
        rows = torch.cat(seen).reshape(3, 9, 20)
        assert rows.dtype == head and all(o.dtype == head for o in out)
        assert float((rows.detach().double().cpu() - want).abs().max()) <= allowed
        assert dec.memory_h.memory.dtype == torch.float32
        sum(o.float().sum() for o in out).backward()
        for p in dec.parameters():
            assert p.grad is not None and p.grad.dtype == p.dtype and bool(p.grad.isfinite().all())
        assert all(bool(p.grad.any()) for p in dec.base_model.parameters())
        got.append(rows.detach().double())
    assert float((got[0] - got[1]).abs().max()) <= 2 * allowed


def test_bfloat16_serving_in_8_bits(dev):
    dec = make().bfloat16()
    dec.train(False)
    x = torch.randn(2, 9, 12, device=dev, dtype=torch.bfloat16)
    with torch.no_grad():
        dec.to_int8()
        out = dec((x[0], torch.arange(9)))
        assert out.shape == (9, 1) and out.dtype == torch.bfloat16 and bool(out.isfinite().all())
        assert dec.forward_sequence(x).shape == (2, 9, 1)


@pytest.mark.parametrize("n", [9, 5])
def test_a_sequence_that_leaves_the_memory_alone(dev, n):
    """In eval mode the memory stays as it is; steps that move it on before the sequence's backward pass do not
    reach what that pass uses."""
    dec = make()
    dec.train(False)
    dec.eval_mode()
    x = torch.randn(4, n, 12, device=dev)
    state = dec.memory_h.memory.clone()
    leaf = next(dec.base_model.parameters())
    (want,) = torch.autograd.grad(dec.forward_sequence(x).sum(), leaf)
    out = dec.forward_sequence(x)
    assert torch.equal(dec.memory_h.memory, state)
    dec.train_mode()
    with torch.no_grad():
        dec((x[0], torch.arange(n)))
    assert not torch.equal(dec.memory_h.memory, state)
    (got,) = torch.autograd.grad(out.sum(), leaf)
    assert torch.equal(got, want)
