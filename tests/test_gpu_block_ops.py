"""Layer norm, the gated linear recurrence (scan and step) and the 8-bit projection on the GPU against
their definitions in 64 bits.

Tolerances count roundings.  u = 2^-24 is half a step of float32, and a result stored in bfloat16
carries half a step of its own, 2^-8 of its value.  Sums over a row are pairwise over lanes (about
log2 D + D / 256 additions deep), so a row sum is off by at most ~(8 + D / 256) u of the sum of its
magnitudes; errors of the recurrence are carried by the recurrence itself."""
import pytest
import torch

from spiral_amd import _native as nv
from spiral_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16
STORE = {F32: U, BF16: 2.0 ** -8}


def within(got, want, tol):
    """Every value of `got` is within `tol` (a tensor or a number) of the float64 `want`."""
    got, want = got.detach().double().cpu(), want.double().cpu()
    tol = torch.as_tensor(tol, dtype=torch.float64).cpu()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= tol)
    worst = ((got - want).abs() / tol.clamp_min(1e-300)).max() if got.numel() else 0
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, {float(worst):.3g} of the tolerance at most"


def rand(*shape, dtype=F32, seed=0, device="cuda"):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device=device).to(dtype)


# ------------------------------------------------------------------------------- layer norm
def norm_ref(x, w, b, eps, g=None):
    """Definition in float64 with, for each output, the tolerance that its roundings add up to."""
    kind, xd = x.dtype, x.detach().double().cpu()
    d = xd.shape[-1]
    xd = xd.reshape(-1, d)
    w = torch.ones(d, dtype=torch.float64) if w is None else w.detach().double().cpu()
    b = torch.zeros(d, dtype=torch.float64) if b is None else b.detach().double().cpu()
    depth = (8 + d / 256) * U
    mu = xd.mean(1, keepdim=True)
    c = xd - mu
    r = 1 / (c.square().mean(1, keepdim=True) + eps).sqrt()
    xh = c * r
    # the mean is off by depth * mean|x|, which moves every xh by that times r; r by depth of itself
    e_xh = depth * (xd.abs().mean(1, keepdim=True) * r + xh.abs()) + 4 * U * (xd.abs() * r + xh.abs())
    y = xh * w + b
    out = {"y": (y, e_xh * w.abs() + 2 * U * (y.abs() + b.abs()) + STORE[kind] * y.abs())}
    if g is not None:
        gd = g.detach().double().cpu().reshape(-1, d)
        gw = gd * w
        m1, m2 = gw.mean(1, keepdim=True), (gw * xh).mean(1, keepdim=True)
        dx = r * (gw - m1 - xh * m2)
        e_m1 = depth * gw.abs().mean(1, keepdim=True) + U * gw.abs().mean(1, keepdim=True)
        e_m2 = (2 * depth * (gw * xh).abs() + gw.abs() * e_xh).mean(1, keepdim=True)
        e = e_m1 + e_m2 * xh.abs() + m2.abs() * e_xh + 6 * U * (gw.abs() + m1.abs() + (xh * m2).abs())
        out["dx"] = (dx, r * e + (depth + 4 * U) * dx.abs() + STORE[kind] * dx.abs())
        # rows one after the other in a lane (at most rows / 1024 / 1), then lanes, groups, partial sums
        chain = (xd.shape[0] / 1024 + 96) * U
        out["dw"] = ((gd * xh).sum(0), chain * (gd * xh).abs().sum(0) + (gd.abs() * e_xh).sum(0))
        out["db"] = (gd.sum(0), chain * gd.abs().sum(0))
    return out


def check_norm(x, w, b, g, eps=1e-5):
    ref = norm_ref(x, w, b, eps, g)
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    it = iter(leaves)
    xl = next(it)
    wl = next(it) if w is not None else None
    bl = next(it) if b is not None else None
    with torch.no_grad():
        free = ops.layer_norm(xl, wl, bl, eps)
    y = ops.layer_norm(xl, wl, bl, eps)
    assert torch.equal(free, y) and y.dtype == x.dtype and y.shape == x.shape
    within(y.reshape(-1, x.shape[-1]), *ref["y"])
    grads = list(torch.autograd.grad(y, leaves, g))
    dx = grads.pop(0)
    assert dx.dtype == x.dtype and dx.shape == x.shape
    within(dx.reshape(-1, x.shape[-1]), *ref["dx"])
    if w is not None:
        dw = grads.pop(0)
        assert dw.dtype == w.dtype
        value, tol = ref["dw"]
        within(dw, value, tol + STORE[w.dtype] * value.abs())
    if b is not None:
        value, tol = ref["db"]
        within(grads.pop(0), value, tol + STORE[b.dtype] * value.abs())


WIDTHS = [1, 2, 3, 4, 10, 31, 32, 33, 64, 65, 128, 129, 255, 256, 511, 513, 1000, 1031, 2048, 2049, 4095, 4100, 8192,
          8193, 16383, 16384]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", WIDTHS)
def test_layer_norm_widths(dev, d, dtype):
    rows = 37 if d < 4096 else 5
    x = (rand(rows, d, seed=d) * 3 + 1.5).to(dtype)
    check_norm(x, 1 + 0.2 * rand(d, seed=1), rand(d, seed=2), rand(rows, d, dtype=dtype, seed=3))


@pytest.mark.parametrize("rows", [0, 1, 2, 7, 255, 8191, 20_001])
def test_layer_norm_row_counts(dev, rows):
    x = rand(rows, 96, seed=rows) + 0.5
    check_norm(x, 1 + 0.2 * rand(96, seed=1), rand(96, seed=2), rand(rows, 96, seed=3))


@pytest.mark.parametrize("w,b", [(None, None), (F32, None), (None, F32), (BF16, BF16)])
def test_layer_norm_optional_and_bf16_parameters(dev, w, b):
    x = rand(33, 5, 72, dtype=BF16)
    check_norm(x, None if w is None else rand(72, dtype=w, seed=1), None if b is None else rand(72, dtype=b, seed=2),
               rand(33, 5, 72, dtype=BF16, seed=3))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layer_norm_strides(dev, dtype):
    base = rand(50, 3, 260, dtype=dtype)
    g = rand(50, 100, dtype=dtype, seed=3)
    w, b = rand(100, seed=1), rand(100, seed=2)
    for x in (base[:, 1, 3:103], base[:, 0, 1:201:2], base.transpose(0, 2)[3:53, 1, :50].repeat(1, 2),
              base[0, 0, 7:107].expand(50, 100), base[:, 2, :200].reshape(100, 100)[:50]):
        check_norm(x, w, b, g)
    check_norm(base[:, 0, :100], w, b, g[:1].expand(50, 100))        # one gradient row for all
    check_norm(base[:, 0, :100], w, b, torch.ones((), device=dev, dtype=dtype).expand(50, 100))
    x = rand(40, 64, dtype=dtype).t()                               # values are the strided dimension
    check_norm(x, rand(40, seed=1), rand(40, seed=2), rand(40, 64, dtype=dtype, seed=3).t())


def test_layer_norm_offset_and_flat_rows(dev):
    # a mean of 1000 deviations: E[x^2] - E[x]^2 in float32 would leave nothing of the variance
    check_norm(rand(64, 128) + 1000.0, rand(128, seed=1), rand(128, seed=2), rand(64, 128, seed=3))
    flat = torch.full((4, 128), 3.25, device=dev)
    y = ops.layer_norm(flat, None, rand(128, seed=2))
    assert torch.equal(y, rand(128, seed=2).expand(4, 128))


def test_layer_norm_rows_that_are_not_finite_stay_alone(dev):
    x = rand(9, 130)
    want = ops.layer_norm(x)
    x[2, 5], x[6, 129] = float("nan"), float("inf")
    y = ops.layer_norm(x)
    ok = torch.tensor([i not in (2, 6) for i in range(9)], device=dev)
    assert torch.equal(y[ok], want[ok]) and bool(y[~ok].isnan().any(1).all())


def test_layer_norm_partial_gradients_and_repeats(dev):
    x, w, b = rand(3000, 128).requires_grad_(), rand(128, seed=1).requires_grad_(), rand(128, seed=2).requires_grad_()
    g = rand(3000, 128, seed=3)
    full = torch.autograd.grad(ops.layer_norm(x, w, b), (x, w, b), g)
    for pick in ([0], [1], [2], [0, 2], [1, 2]):
        leaves = [(x, w, b)[i] for i in pick]
        args = [t if i in pick else t.detach() for i, t in enumerate((x, w, b))]
        got = torch.autograd.grad(ops.layer_norm(*args), leaves, g)
        assert all(torch.equal(a, full[i]) for a, i in zip(got, pick))
    with pytest.raises(RuntimeError):  # no second derivative
        (dx,) = torch.autograd.grad(ops.layer_norm(x, w, b), x, g, create_graph=True)
        dx.sum().backward()


# -------------------------------------------------------------------- gated linear recurrence
def scan_ref(gates, h0, active, g=None, g_last=None):
    """Time-major definition in float64 on the CPU, with tolerances.  A step rounds a, 1 - a (4 u
    each: exponential, reciprocal, product) and two products and a sum; joined maps round as often
    again: 16 u of each term, and what came in is carried on by a."""
    kind = gates.dtype
    t_end, n, h2 = gates.shape
    hd = h2 // 2
    gates = gates.detach().double().cpu()
    state = torch.zeros(n, hd, dtype=torch.float64) if h0 is None else h0.detach().double().cpu()
    active = torch.ones(t_end, n, dtype=torch.bool) if active is None else active.cpu()
    err = torch.zeros_like(state)
    hs, errs = [state], [err]
    for t in range(t_end):
        z, c = gates[t, :, :hd], gates[t, :, hd:]
        on = active[t][:, None]
        a, rest = torch.sigmoid(z), torch.sigmoid(-z)
        err = torch.where(on, a * err + 16 * U * (a * state.abs() + rest * c.abs()), err + 4 * U * state.abs())
        state = torch.where(on, a * state + rest * torch.where(on, c, 0.0), state)
        hs.append(state)
        errs.append(err)
    h = torch.stack(hs[1:]) if t_end else torch.zeros(0, n, hd, dtype=torch.float64)
    e_h = torch.stack(errs[1:]) if t_end else h
    out = {"h": (h, e_h + STORE[kind] * h.abs() + 1e-37), "last": (state, err + 1e-37)}
    if g is not None or g_last is not None:
        e = torch.zeros(n, hd, dtype=torch.float64) if g_last is None else g_last.detach().double().cpu()
        err = torch.zeros_like(e)
        dgates, tol = torch.zeros_like(gates), torch.zeros_like(gates)
        for t in reversed(range(t_end)):
            z, c = gates[t, :, :hd], gates[t, :, hd:]
            on = active[t][:, None]
            a, rest = torch.sigmoid(z), torch.sigmoid(-z)
            gt = 0.0 if g is None else g[t].detach().double().cpu()
            d = e + gt
            e_d = err + 2 * U * (e.abs() + (0.0 if g is None else gt.abs()))
            # the state before the step is read back as it was stored
            e_p = errs[t] + (STORE[kind] if t else 0.0) * hs[t].abs()
            gap = hs[t] - torch.where(on, c, 0.0)
            dz, dc = d * gap * a * rest, d * rest
            e_z = (e_d * gap.abs() + d.abs() * (e_p + 4 * U * (hs[t].abs() + c.abs()))) * a * rest
            dgates[t, :, :hd] = torch.where(on, dz, 0.0)
            dgates[t, :, hd:] = torch.where(on, dc, 0.0)
            tol[t, :, :hd] = torch.where(on, e_z + 16 * U * dz.abs() + STORE[kind] * dz.abs(), 0.0)
            tol[t, :, hd:] = torch.where(on, e_d * rest + 8 * U * dc.abs() + STORE[kind] * dc.abs(), 0.0)
            err = torch.where(on, a * e_d + 16 * U * a * d.abs(), e_d + 4 * U * d.abs())
            e = torch.where(on, a * d, d)
        out["dgates"], out["dh0"] = (dgates, tol + 1e-37), (e, err + 1e-37)
    return out


def check_scan(gates, h0=None, active=None, batch_first=False, with_g=True, with_last=True):
    turn = (lambda t: None if t is None else t.transpose(0, 1)) if batch_first else (lambda t: t)
    hd = gates.shape[2] // 2
    g = rand(*gates.shape[:2], hd, dtype=gates.dtype, seed=11) if with_g else None
    g_last = rand(gates.shape[0 if batch_first else 1], hd, seed=12) if with_last else None
    ref = scan_ref(turn(gates), h0, turn(active), turn(g), g_last)
    gl = gates.detach().requires_grad_()
    hl = None if h0 is None else h0.detach().requires_grad_()
    with torch.no_grad():
        free = ops.gated_scan(gl, hl, active, batch_first)
    h, last = ops.gated_scan(gl, hl, active, batch_first)
    assert torch.equal(free[0], h) and torch.equal(free[1], last)
    assert h.dtype == gates.dtype and last.dtype == F32 and h.shape == (*gates.shape[:2], hd)
    within(turn(h), *ref["h"])
    within(last, *ref["last"])
    outs, grads = zip(*[(o, d) for o, d in ((h, g), (last, g_last)) if d is not None])
    leaves = [gl] + ([] if hl is None else [hl])
    got = torch.autograd.grad(outs, leaves, grads)
    assert got[0].dtype == gates.dtype
    within(turn(got[0]), *ref["dgates"])
    if hl is not None:
        within(got[1], *ref["dh0"])


def make_active(t, n, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    on = torch.rand(t, n, generator=g, device="cuda") < 0.7
    on[:, ::5] = False                                     # never there
    start = torch.randint(0, max(t, 1), (n,), generator=g, device="cuda")
    on[:, 1::3] = torch.arange(t, device="cuda")[:, None] >= start[None, 1::3]
    return on


# one step to long sequences, odd sizes, every layout of the work: one thread walking the steps
# (few steps, or 65536 lanes of four units and more), strands of one workgroup, split sequences
SIZES = [(0, 3, 8), (1, 1, 1), (1, 5, 33), (2, 3, 7), (7, 4, 10), (16, 2, 128), (17, 2, 128), (40, 3, 5), (64, 1, 32),
         (65, 700, 12), (100, 2, 128), (129, 1, 3), (513, 9, 66), (1500, 1, 128), (5000, 1, 4), (33, 600, 40),
         (6, 4096, 64)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("t,n,h", SIZES)
def test_scan_sizes(dev, t, n, h, dtype):
    gates = rand(t, n, 2 * h, dtype=dtype, seed=t + n + h)
    gates[..., :h] += 1.0
    check_scan(gates, rand(n, h, seed=1))
    check_scan(gates, None, make_active(t, n), with_last=False)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scan_many_lanes(dev, dtype):
    t, n, h = 19, 2100, 126   # 67200 lanes of four units: the walking layout past 16 steps
    check_scan(rand(t, n, 2 * h, dtype=dtype), rand(n, h, seed=1), make_active(t, n))


# rows of fewer than four units, and of a few more, in each layout: walked (few steps; many lanes), strands of
# enough workgroups to leave the steps whole, and split steps
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("t,n,h", [(3, 50, 1), (5, 7, 2), (19, 70000, 3), (21, 66000, 2), (23, 33000, 5), (40, 17000, 3),
                                   (37, 4200, 14), (700, 3, 2), (901, 2, 3), (1200, 1, 1), (333, 5, 7)])
def test_scan_short_rows_in_every_layout(dev, t, n, h, dtype):
    gates = rand(t, n, 2 * h, dtype=dtype, seed=t + n + h)
    on = make_active(t, n)
    check_scan(gates, rand(n, h, seed=1), on)
    check_scan(gates.masked_fill(~on[..., None], float("nan")), None, on, with_g=False)
    check_scan(gates.transpose(0, 1).contiguous(), rand(n, h, seed=2), on.t(), batch_first=True)


@pytest.mark.parametrize("t,n,h", [(33, 5, 12), (300, 2, 128), (9, 70, 30)])
def test_scan_batch_first_and_strides(dev, t, n, h):
    on = make_active(t, n)
    check_scan(rand(n, t, 2 * h), rand(n, h, seed=1), on.t(), batch_first=True)
    check_scan(rand(n, t, 2 * h), rand(n, h, seed=1), on.t().contiguous(), batch_first=True, with_g=False)
    wide = rand(t, n, 2 * h + 5)
    check_scan(wide[..., 3:3 + 2 * h], rand(n, h + 1, seed=1)[:, 1:], on)
    check_scan(rand(t, 2 * h, n).transpose(1, 2), rand(h, n, seed=1).t())
    check_scan(rand(1, n, 2 * h).expand(t, n, 2 * h), rand(1, h, seed=1).expand(n, h))
    check_scan(rand(2 * t, 2 * n, 2 * h)[::2, 1::2], None, on)


def test_scan_extreme_gates(dev):
    t, n, h = 70, 2, 6
    gates = rand(t, n, 2 * h)
    levels = torch.tensor([-3.0e38, -200.0, -30.0, 30.0, 200.0, 3.0e38], device=dev)
    gates[..., :h] = levels
    check_scan(gates, rand(n, h, seed=1))
    gates[..., :h] = torch.tensor([float("-inf"), float("inf")] * 3, device=dev)
    h0 = rand(n, h, seed=1)
    hs, last = ops.gated_scan(gates, h0)
    assert torch.equal(hs[..., ::2], gates[..., h::2])          # forgets everything
    assert torch.equal(last[:, 1::2], h0[:, 1::2])              # keeps everything


@pytest.mark.parametrize("t,n,h", [(12, 6, 20), (200, 3, 40), (3000, 1, 24)])
def test_scan_ignores_what_stands_in_inactive_steps(dev, t, n, h):
    on = make_active(t, n)
    gates = rand(t, n, 2 * h)
    dirty = gates.clone()
    dirty[~on] = torch.tensor([float("nan"), float("inf")], device=dev).repeat(h)
    h0 = rand(n, h, seed=1).requires_grad_()
    a, b = gates.requires_grad_(), dirty.requires_grad_()
    ha, la = ops.gated_scan(a, h0, on)
    hb, lb = ops.gated_scan(b, h0, on)
    assert torch.equal(ha, hb) and torch.equal(la, lb)
    g, gl = rand(t, n, h, seed=4), rand(n, h, seed=5)
    ga, ea = torch.autograd.grad((ha, la), (a, h0), (g, gl))
    gb, eb = torch.autograd.grad((hb, lb), (b, h0), (g, gl))
    assert torch.equal(ga, gb) and torch.equal(ea, eb)
    assert bool((ga[~on] == 0).all())
    none = torch.zeros(t, n, dtype=torch.bool, device=dev)
    hn, ln = ops.gated_scan(dirty, h0, none)
    assert torch.equal(hn, h0.expand(t, n, h)) and torch.equal(ln, h0)


def test_scan_gradient_against_differences(dev):
    """Directional derivative of <h, g> + <last, g_last>, central differences of the definition in
    float64 (step 1e-4: off by ~1e-8 of the third derivative), against the kernel's gradient, whose
    terms are off by ~100 u each over 90 steps: 1e-5 of the sum of their magnitudes."""
    t, n, h = 90, 3, 10
    on = make_active(t, n)
    gates, h0 = rand(t, n, 2 * h), rand(n, h, seed=1)
    g, gl = rand(t, n, h, seed=2), rand(n, h, seed=3)
    dg, dh = rand(t, n, 2 * h, seed=4), rand(n, h, seed=5)

    def f(step):
        ref = scan_ref_values(gates.double().cpu() + step * dg.double().cpu(), h0.double().cpu() + step * dh.double().cpu(),
                              on.cpu())
        return float((ref[0] * g.double().cpu()).sum() + (ref[1] * gl.double().cpu()).sum())

    a, b = gates.requires_grad_(), h0.requires_grad_()
    ga, gb = torch.autograd.grad(ops.gated_scan(a, b, on), (a, b), (g, gl))
    got = float((ga.double() * dg.double()).sum() + (gb.double() * dh.double()).sum())
    size = float((ga.double() * dg.double()).abs().sum() + (gb.double() * dh.double()).abs().sum())
    assert abs(got - (f(1e-4) - f(-1e-4)) / 2e-4) <= 1e-5 * size


def scan_ref_values(gates, h0, on):
    hd, state, hs = gates.shape[2] // 2, h0, []
    for t in range(gates.shape[0]):
        a = torch.sigmoid(gates[t, :, :hd])
        state = torch.where(on[t][:, None], a * state + (1 - a) * gates[t, :, hd:], state)
        hs.append(state)
    return torch.stack(hs), state


def test_norm_gradient_against_differences(dev):
    x, w, b, g = rand(7, 33), rand(33, seed=1), rand(33, seed=2), rand(7, 33, seed=3)
    dirs = [rand(7, 33, seed=4), rand(33, seed=5), rand(33, seed=6)]

    def f(step):
        xs, ws, bs = (v.double().cpu() + step * d.double().cpu() for v, d in zip((x, w, b), dirs))
        c = xs - xs.mean(1, keepdim=True)
        return float(((c / (c.square().mean(1, keepdim=True) + 1e-5).sqrt() * ws + bs) * g.double().cpu()).sum())

    leaves = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(ops.layer_norm(*leaves), leaves, g)
    terms = [(gr.double() * d.double()) for gr, d in zip(grads, dirs)]
    got, size = sum(float(t.sum()) for t in terms), sum(float(t.abs().sum()) for t in terms)
    assert abs(got - (f(1e-4) - f(-1e-4)) / 2e-4) <= 1e-5 * size


def test_scan_joined_pieces_equal_the_whole(dev):
    """A sequence cut in two, the second piece started from the first one's last state: the same
    states up to the roundings of scan_ref."""
    gates, h0 = rand(700, 2, 128), rand(2, 64, seed=1)
    whole, last = ops.gated_scan(gates, h0)
    first, mid = ops.gated_scan(gates[:311], h0)
    second, end = ops.gated_scan(gates[311:], mid)
    ref = scan_ref(gates, h0, None)
    within(torch.cat([first, second]), ref["h"][0], 2 * ref["h"][1])
    within(end, ref["last"][0], 2 * ref["last"][1])


# --------------------------------------------------------------------------- the single step
def step_ref(gates, mem, ids):
    hd = gates.shape[1] // 2
    z, c = gates.detach().double().cpu()[:, :hd], gates.detach().double().cpu()[:, hd:]
    old = mem.double().cpu()[ids.cpu()]
    a, rest = torch.sigmoid(z), torch.sigmoid(-z)
    new = a * old + rest * c
    return new, 16 * U * (a * old.abs() + rest * c.abs()) + 1e-37, old, a, rest, c


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,nodes,h", [(0, 4, 8), (1, 1, 1), (1, 900, 128), (64, 900, 127), (900, 900, 10),
                                       (1024, 2000, 6), (1025, 2000, 6), (3000, 5000, 64), (1500, 1500, 3)])
def test_step(dev, m, nodes, h, dtype):
    gates, mem = rand(m, 2 * h, dtype=dtype), rand(nodes, h, seed=1)
    ids = torch.randperm(nodes, generator=torch.Generator().manual_seed(2))[:m].to(dev)
    for listed in (ids, None):
        use = ids if listed is not None else torch.arange(m, device=dev)
        new, tol, old, a, rest, c = step_ref(gates, mem, use)
        state = mem.clone()
        kept = ops.gated_step(gates, state, listed, mem_write=False)
        assert torch.equal(state, mem)
        gl = gates.detach().requires_grad_()
        got = ops.gated_step(gl, state, listed)
        assert got.dtype == F32 and torch.equal(kept, got)
        within(got, new, tol)
        want = mem.clone()
        want[use] = got.detach()
        assert torch.equal(state, want)
        g = rand(m, h, seed=3)
        (dg,) = torch.autograd.grad(got, gl, g)
        gd = g.double().cpu()
        dz, dc = gd * (old - c) * a * rest, gd * rest
        within(dg, torch.cat([dz, dc], 1), torch.cat(
            [(16 * U + STORE[dtype]) * dz.abs() + 16 * U * gd.abs() * (old.abs() + c.abs()) * a * rest,
             (8 * U + STORE[dtype]) * dc.abs()], 1) + 1e-37)


@pytest.mark.parametrize("m", [50, 1024, 4000])
def test_step_names_a_node_twice(dev, m):
    """Every row starts from the old state; the memory keeps the last row of a node."""
    nodes, h = m // 3, 20
    gates, mem = rand(m, 2 * h), rand(nodes, h, seed=1)
    ids = torch.randint(0, nodes, (m,), generator=torch.Generator().manual_seed(2)).to(dev)
    new, tol, *_ = step_ref(gates, mem, ids)
    for _ in range(3):
        state = mem.clone()
        got = ops.gated_step(gates, state, ids)
        within(got, new, tol)
        want = mem.cpu().clone()
        for i, node in enumerate(ids.tolist()):
            want[node] = got[i].cpu()
        assert torch.equal(state.cpu(), want)


@pytest.mark.parametrize("m", [6, 2000])
def test_step_leaves_unknown_nodes_alone(dev, m):
    nodes, h = m, 9
    gates, mem = rand(m, 2 * h), rand(nodes, h, seed=1)
    ids = torch.arange(m, device=dev)
    ids[1], ids[4] = nodes, -1
    state = mem.clone()
    got = ops.gated_step(gates, state, ids)
    bad = torch.zeros(m, dtype=torch.bool, device=dev)
    bad[1] = bad[4] = True
    assert bool(got[bad].isnan().all()) and bool(got[~bad].isfinite().all())
    assert torch.equal(state[bad], mem[bad]) and torch.equal(state[~bad], got[~bad])


def test_step_and_scan_agree_and_the_version_counts(dev):
    gates, mem = rand(40, 25, 64), rand(25, 32, seed=1)
    hs, last = ops.gated_scan(gates, mem.clone())
    state = mem.clone()
    before = state._version
    for t in range(40):
        out = ops.gated_step(gates[t], state)
    assert state._version == before + 40
    ref = scan_ref(gates, mem, None)
    within(state, ref["last"][0], 2 * ref["last"][1])
    assert torch.equal(out, state)
    within(hs, *ref["h"])
    kept = state.clone().requires_grad_()
    with torch.no_grad():  # a state an autograd graph saved is not changed unnoticed
        leaf = rand(5, 64).requires_grad_()
    y = (kept * 1.0)
    z = y.square().sum()
    with torch.no_grad():
        ops.gated_step(rand(25, 64), y)
    with pytest.raises(RuntimeError, match="modified"):
        z.backward()
    del leaf


# -------------------------------------------------------------------------- 8-bit projection
def quantized(x):
    """The whole numbers and scales by the definition: float32 quotient and product, each the float64
    one rounded once."""
    xd = x.detach().double().cpu()
    top = xd.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -120)
    q = torch.round((xd * (127.0 / top).float().double()).float()).double()
    return q, (top / 127.0).squeeze(-1)


def check_int8(x, wq, ws, bias=None, act=None, slope=0.01, out_dtype=None):
    k, n = x.shape[-1], wq.shape[0]
    q, s = quantized(x.reshape(-1, k))
    terms = (q @ wq.double().cpu().t()) * s[:, None] * ws.double().cpu()
    b = torch.zeros(n, dtype=torch.float64) if bias is None else bias.double().cpu()
    y = terms + b
    tol = 6 * U * terms.abs() + 2 * U * (terms.abs() + b.abs())
    if act is not None:
        low = 0.0 if act == "relu" else slope
        y, tol = torch.where(y < 0, y * low, y), tol * max(1.0, abs(low)) + U * y.abs()
    kind = x.dtype if out_dtype is None else out_dtype
    got = ops.linear_int8(x, wq, ws, bias, act, slope, out_dtype)
    assert got.dtype == kind and got.shape == (*x.shape[:-1], n)
    within(got.reshape(-1, n), y, tol + STORE[kind] * y.abs() + 1e-37)
    return got


def weight8(n, k, seed=5):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8),
            torch.rand(n, generator=g, device="cuda") * 0.01 + 1e-4)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,k", [(0, 5), (1, 1), (3, 2), (5, 63), (64, 64), (130, 129), (7, 1000), (2, 5001),
                                 (1, 131072), (2000, 128)])
def test_quantize_rows(dev, m, k, dtype):
    x = rand(m, k, dtype=dtype, seed=m + k) * 3
    q, scale = ops.quantize_rows_int8(x)
    want_q, want_s = quantized(x)
    assert q.dtype == torch.int8 and q.shape == x.shape and scale.shape == (m,)
    assert torch.equal(q.double().cpu(), want_q)
    within(scale, want_s, U * want_s)
    back = q.double().cpu() * scale.double().cpu()[:, None]
    # half a scale, and the roundings of quotient, product and scale: 127 (3 u) scales
    within(back, x.double().cpu(), (0.5 + 127 * 4 * U) * want_s[:, None].expand(m, k))


def test_quantize_ranges_and_rows_that_are_not_finite(dev):
    x = rand(10, 40)
    x[1] = 0.0
    x[2] *= 1e38 / x[2].abs().max()
    x[3] *= 1e-36
    x[4] *= 1e-44
    x[5, 7], x[6, 0], x[7, 39] = float("nan"), float("inf"), float("-inf")
    q, scale = ops.quantize_rows_int8(x)
    bad = torch.zeros(10, dtype=torch.bool, device=dev)
    bad[5:8] = True
    assert bool(scale[bad].isnan().all()) and bool((q[bad] == 0).all())
    want_q, want_s = quantized(x[~bad])
    assert torch.equal(q[~bad].double().cpu(), want_q)
    within(scale[~bad], want_s, U * want_s + 2.0 ** -149)
    assert bool((q[1] == 0).all()) and bool((q[4] == 0).all())
    wq, ws = weight8(20, 40)
    y = ops.linear_int8(x, wq, ws, rand(20, seed=3), "relu")
    assert bool(y[bad].isnan().all()) and bool(y[~bad].isfinite().all())
    assert torch.equal(y[~bad], ops.linear_int8(x[~bad], wq, ws, rand(20, seed=3), "relu"))


INT8_SIZES = [(0, 8, 8), (1, 1, 1), (1, 128, 256), (1, 4096, 100), (2, 17, 3), (3, 100, 33), (16, 2048, 300),
              (17, 64, 64), (31, 65, 31), (32, 513, 129), (33, 32, 1000), (64, 128, 64), (65, 63, 65), (127, 130, 255),
              (128, 512, 128), (129, 1000, 257), (255, 96, 384), (257, 129, 1025), (512, 256, 512), (1000, 384, 33),
              (1023, 1, 70), (2049, 40, 7), (4100, 128, 256), (300, 4096, 300)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,k,n", INT8_SIZES)
def test_linear_int8_sizes(dev, m, k, n, dtype):
    wq, ws = weight8(n, k)
    x = rand(m, k, dtype=dtype, seed=m + k + n)
    check_int8(x, wq, ws, rand(n, seed=1))
    check_int8(x, wq, ws, None, "leaky_relu", 0.2, BF16 if dtype == F32 else F32)


# rows on both sides of what a workgroup holds of them (16 pieces of 2048 values), of the pieces a wave
# or four waves hold, and of rows that are read twice
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,k,n", [(8, 4096, 40), (8, 4097, 40), (5, 4098, 17), (1, 32768, 20), (1, 32769, 5), (3, 9000, 33),
                                   (2, 16384, 16), (2, 16390, 16), (16, 1, 3), (16, 3, 20), (15, 2047, 50), (65, 8193, 20),
                                   (70, 16385, 9), (20, 1025, 30), (18, 2049, 31), (100, 5000, 70)])
def test_linear_int8_long_rows(dev, m, k, n, dtype):
    wq, ws = weight8(n, k)
    check_int8(rand(m, k, dtype=dtype, seed=m + k + n), wq, ws, rand(n, seed=1))


# few rows by so many columns that they are brought to whole numbers in a launch of their own, and just below
@pytest.mark.parametrize("m,k,n", [(16, 100, 8192), (16, 100, 8193), (3, 65, 43690), (3, 65, 43691), (1, 40, 140000),
                                   (2, 40, 65537)])
def test_linear_int8_few_rows_many_columns(dev, m, k, n):
    wq, ws = weight8(n, k)
    check_int8(rand(m, k, dtype=BF16, seed=m + k + n), wq, ws, rand(n, seed=1))
    check_int8(rand(m, k, seed=m + k + n), wq, ws, None, "relu")


def test_linear_int8_activations_bias_types_and_shapes(dev):
    wq, ws = weight8(40, 72)
    x = rand(4, 9, 72)
    for act in (None, "none", "relu", "leaky_relu"):
        check_int8(x, wq, ws, rand(40, dtype=BF16, seed=1), None if act == "none" else act)
    check_int8(x[0, 0], wq, ws)
    assert ops.linear_int8(x, wq[:0], ws[:0]).shape == (4, 9, 0)


@pytest.mark.parametrize("m,k,n", [(1, 200, 70), (40, 200, 70), (700, 130, 260)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_linear_int8_strides(dev, m, k, n, dtype):
    wq, ws = weight8(n + 3, 2 * k + 5)
    x = rand(m + 1, 2 * k + 7, dtype=dtype)
    for xv in (x[1:, 3:3 + k], x[1:, 1:2 * k:2], x[1, :k].expand(m, k), rand(k, m, dtype=dtype).t()):
        for wv in (wq[3:, 1:1 + k], wq[:n, ::2][:, :k], wq[0, :k].expand(n, k)):
            check_int8(xv, wv, ws[3:], rand(n, seed=1))
    check_int8(x[1:, :k], wq[:n, :k], torch.rand(2 * n, device=dev)[::2], rand(2 * n, seed=1)[::2])


def test_linear_int8_sums_are_exact(dev):
    """All products at their largest and of one sign: the sum is past 2^24, and past 2^30 at the
    largest K."""
    for k in (4096, 131072):
        x = torch.ones(5, k, device=dev)
        wq = torch.full((6, k), 127, dtype=torch.int8, device=dev)
        wq[1] = -127
        wq[2, 0] = 126
        y = check_int8(x, wq, torch.ones(6, device=dev))
        assert float(y[0, 0]) == float(torch.tensor(127 * 127 * k / 127.0))


# ------------------------------------------------------------------- streams, graphs, sizes
def block_forward(x, p):
    """The operators together, as a block of the decoder runs them."""
    t, n, d = x.shape
    y = ops.layer_norm(x, p["g"], p["b"])
    gates = y @ p["w"]
    h, last = ops.gated_scan(gates, p["h0"], p["on"])
    return ops.layer_norm(h), last


def block_params(t, n, d, dev):
    p = {"g": 1 + 0.1 * rand(d, seed=1), "b": rand(d, seed=2), "w": rand(d, 2 * d, seed=3) / d ** 0.5,
         "h0": rand(n, d, seed=4)}
    for v in p.values():
        v.requires_grad_()
    p["on"] = make_active(t, n)
    return p


def test_other_streams_give_the_same_bits(dev):
    t, n, d = 500, 3, 64
    x, p = rand(t, n, d).requires_grad_(), block_params(t, n, d, dev)
    leaves = [x, p["g"], p["b"], p["w"], p["h0"]]
    y, last = block_forward(x, p)
    want = [y, last, *torch.autograd.grad((y, last), leaves, (rand(t, n, d, seed=8), rand(n, d, seed=9)))]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            y, last = block_forward(x, p)
            got.append([y, last, *torch.autograd.grad((y, last), leaves, (rand(t, n, d, seed=8), rand(n, d, seed=9)))])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


def test_captured_and_replayed(dev):
    """Forward, backward, the step on the memory and the 8-bit projection in one graph; every replay
    on new inputs against the eager result, with eager work between the replays."""
    t, n, d = 260, 2, 64
    x = rand(t, n, d)
    p = block_params(t, n, d, dev)
    leaves = [p["g"], p["b"], p["w"], p["h0"]]
    grads = (rand(t, n, d, seed=8), rand(n, d, seed=9))
    wq, ws = weight8(2 * d, d)
    ids = torch.tensor([5, 3, 5, 0] * 300, device=dev)
    mem = rand(7, d, seed=7)

    def work(mem):
        y, last = block_forward(x, p)
        g = torch.autograd.grad((y, last), leaves, grads)
        with torch.no_grad():
            rows = ops.linear_int8(y.detach().reshape(-1, d)[:1], wq, ws).expand(len(ids), 2 * d)
            few = ops.linear_int8(y.detach().reshape(-1, d), wq, ws)
            h = ops.gated_step(rows, mem, ids)
        return [y.detach(), last.detach(), *g, few, h]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        work(mem.clone())
    torch.cuda.current_stream().wait_stream(s)
    held = mem.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work(held)
    for k in range(4):
        with torch.no_grad():
            x.copy_(rand(t, n, d, seed=20 + k))
        held.copy_(mem)
        graph.replay()
        torch.cuda.synchronize()
        fresh = mem.clone()
        want = work(fresh)
        assert all(torch.equal(a, b) for a, b in zip(outs, want)) and torch.equal(held, fresh)


def test_offsets_past_32_bits(dev):
    """Matrices of more than 2^31 values: the last rows come out as they do alone."""
    d = 4096
    m = 2 ** 31 // d + 3
    x = torch.zeros(m, d, dtype=BF16, device=dev)
    x[-4:] = rand(4, d, dtype=BF16)
    y = ops.layer_norm(x)
    assert torch.equal(y[-4:], ops.layer_norm(x[-4:].clone()))
    del y
    wq, ws = weight8(8, d)
    assert torch.equal(ops.linear_int8(x, wq, ws)[-4:], ops.linear_int8(x[-4:].clone(), wq, ws))
    gates = x.view(-1, 1, 2 * 64)[: 2 ** 31 // 128 + 2]
    h, last = ops.gated_scan(gates)
    short, last2 = ops.gated_scan(x.view(-1, 1, 128)[-40:])
    del h
    h, last = ops.gated_scan(x.view(-1, 1, 128)[-(2 ** 31 // 128 + 1):])
    assert torch.allclose(last, last2, rtol=1e-6, atol=1e-7)
    del h, x
    mem = torch.zeros(2 ** 31 // 64 + 5, 64, device=dev)
    ids = torch.tensor([mem.shape[0] - 1, 2 ** 25, 3], device=dev)
    step = rand(3, 128)
    out = ops.gated_step(step, mem, ids)
    assert torch.equal(mem[ids], out) and int((mem != 0).any(1).sum()) == 3


def test_library_was_used(dev):
    assert nv.lib().spmi_version() >= 100


def test_more_rows_than_a_grid_has_waves(dev):
    """2^24 rows and some: the launches are bounded, the kernels go on."""
    m = (1 << 24) + 77
    x = torch.zeros(m, 4, dtype=BF16, device=dev)
    x[-100:] = rand(100, 4, dtype=BF16)
    q, scale = ops.quantize_rows_int8(x)
    want_q, want_s = quantized(x[-100:])
    assert torch.equal(q[-100:].double().cpu(), want_q) and int(q[:-100].count_nonzero()) == 0
    within(scale[-100:], want_s, U * want_s)
    y = ops.layer_norm(x)
    assert torch.equal(y[-100:], ops.layer_norm(x[-100:].clone())) and int(y[:-100].count_nonzero()) == 0


def test_empty_problems(dev):
    h, last = ops.gated_scan(torch.zeros(5, 0, 8, device=dev))
    assert h.shape == (5, 0, 4) and last.shape == (0, 4)
    gates = torch.zeros(0, 3, 8, device=dev, requires_grad=True)
    h0 = rand(3, 4).requires_grad_()
    h, last = ops.gated_scan(gates, h0)
    (g,) = torch.autograd.grad(last, h0, rand(3, 4, seed=1))
    assert torch.equal(last, h0) and torch.equal(g, rand(3, 4, seed=1))
    x, w = torch.zeros(0, 8, device=dev, requires_grad=True), torch.ones(8, device=dev, requires_grad=True)
    gx, gw = torch.autograd.grad(ops.layer_norm(x, w).sum(), (x, w))
    assert gx.shape == (0, 8) and bool((gw == 0).all())
    mem = torch.zeros(0, 4, device=dev)
    assert bool(ops.gated_step(torch.zeros(2, 8, device=dev), mem, torch.zeros(2, dtype=torch.int64, device=dev)).isnan().all())
    assert ops.quantize_rows_int8(torch.zeros(0, 8, device=dev))[0].shape == (0, 8)


def test_inference_mode(dev):
    mem = rand(6, 8)
    want = ops.gated_step(rand(6, 16), mem.clone())
    with torch.inference_mode():
        inside = mem.clone()
        assert torch.equal(ops.gated_step(rand(6, 16), inside), want) and torch.equal(inside, want)
        assert torch.equal(ops.gated_step(rand(6, 16), mem), want) and torch.equal(mem, want)
        wq, ws = weight8(5, 8)
        assert ops.linear_int8(ops.layer_norm(mem), wq, ws).shape == (6, 5)


def test_a_backward_pass_runs_twice_and_sees_changed_inputs(dev):
    gates, h0 = rand(40, 3, 16).requires_grad_(), rand(3, 8, seed=1).requires_grad_()
    h, last = ops.gated_scan(gates, h0)
    g = rand(40, 3, 8, seed=2)
    first = torch.autograd.grad(h, (gates, h0), g, retain_graph=True)
    second = torch.autograd.grad(h, (gates, h0), g, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    with torch.no_grad():
        h.add_(1.0)
    with pytest.raises(RuntimeError, match="modified"):
        torch.autograd.grad(h, (gates, h0), g)
