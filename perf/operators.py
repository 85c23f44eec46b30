"""What the operators of a gated-linear-recurrence decoder block are measured on: layer norm
(forward, and with the gradients of its input, weight and bias), the gated linear recurrence (a
scan over a sequence of snapshots, with its gradients, and the one-snapshot step on the node
memory) and the 8-bit integer projection with a scale per row and per output channel.

`run` computes an operator in plain torch operations, or, where `own` is true, through
spiral_amd.ops.  `exact` evaluates the definitions in 64 bits."""
import math

import torch

own = False

F32, BF16 = "float32", "bfloat16"
_TYPES = {F32: torch.float32, BF16: torch.bfloat16}
EPS = 1e-5
TINY = 2.0 ** -120  # smallest row maximum of the 8-bit rows: 127 / 2^-120 is still finite


def listed():
    return [
        # one node's embedding normalised on its way to the head: latency
        {"name": "norm_one_row", "op": "norm", "rows": 1, "width": 128, "dtype": F32, "train": False},
        # every node of the headline snapshot in a training step
        {"name": "norm_train_nodes", "op": "norm", "rows": 1_000_000, "width": 128, "dtype": F32, "train": True},
        # wide bfloat16 rows of an odd width and count in a training step
        {"name": "norm_train_odd_bf16", "op": "norm", "rows": 12_289, "width": 1031, "dtype": BF16, "train": True},
        # one snapshot served for a short list of nodes out of a large memory: latency
        {"name": "step_few_nodes", "op": "step", "rows": 64, "nodes": 100_000, "hidden": 128, "dtype": F32},
        # a long history of one entity replayed into its state: only 128 channels to work on
        {"name": "scan_long_single", "op": "scan", "steps": 65_536, "nodes": 1, "hidden": 128, "dtype": F32,
         "train": False, "ragged": False, "batch_first": False},
        # 32 snapshots of a growing node set trained through time
        {"name": "scan_train_snapshots", "op": "scan", "steps": 32, "nodes": 50_000, "hidden": 128, "dtype": F32,
         "train": True, "ragged": True, "batch_first": False},
        # a padded batch of sequences of different lengths, batch first, bfloat16 storage
        {"name": "scan_train_padded_bf16", "op": "scan", "steps": 1021, "nodes": 24, "hidden": 384, "dtype": BF16,
         "train": True, "ragged": True, "batch_first": True},
        # one row through the projection of a block of 128 units: latency
        {"name": "int8_one_row", "op": "int8", "rows": 1, "inner": 128, "outer": 256, "dtype": F32,
         "bias": True, "act": "none"},
        # a handful of rows against a wide weight: reading the weight is the work
        {"name": "int8_few_rows", "op": "int8", "rows": 16, "inner": 2048, "outer": 4096, "dtype": BF16,
         "bias": True, "act": "none"},
        # every node of the headline snapshot through the projection of a block of 128 units
        {"name": "int8_nodes", "op": "int8", "rows": 1_000_000, "inner": 128, "outer": 256, "dtype": F32,
         "bias": True, "act": "none"},
        # rows of the wide stress model with an odd row count
        {"name": "int8_wide_rows", "op": "int8", "rows": 100_003, "inner": 512, "outer": 1024, "dtype": F32,
         "bias": True, "act": "leaky_relu"},
        # a product whose arithmetic is the work
        {"name": "int8_large_bf16", "op": "int8", "rows": 8200, "inner": 2048, "outer": 4096, "dtype": BF16,
         "bias": False, "act": "relu"},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["norm", "scan", "step", "int8"])
    dtype = rng.choice([F32, BF16])
    if op == "norm":
        width = _spread(rng, 8, 8192)
        rows = _spread(rng, 1, min(1_000_000, 128_000_000 // width))
        return {"op": op, "rows": rows, "width": width, "dtype": dtype, "train": rng.random() < 0.6}
    if op == "scan":
        hidden = _spread(rng, 8, 1024)
        steps = _spread(rng, 1, 65_536)
        nodes = _spread(rng, 1, max(1, min(200_000, 100_000_000 // (hidden * steps))))
        return {"op": op, "steps": steps, "nodes": nodes, "hidden": hidden, "dtype": dtype,
                "train": rng.random() < 0.6, "ragged": rng.random() < 0.5, "batch_first": rng.random() < 0.5}
    if op == "step":
        hidden = _spread(rng, 8, 1024)
        nodes = _spread(rng, 1, 200_000_000 // (4 * hidden))
        return {"op": op, "rows": _spread(rng, 1, nodes), "nodes": nodes, "hidden": hidden, "dtype": dtype}
    inner, outer = _spread(rng, 16, 4096), _spread(rng, 16, 4096)
    rows = _spread(rng, 1, min(1_000_000, 256_000_000 // max(inner, outer), 60_000_000_000 // (inner * outer)))
    return {"op": op, "rows": rows, "inner": inner, "outer": outer, "dtype": dtype, "bias": rng.random() < 0.5,
            "act": rng.choice(["none", "relu", "leaky_relu"])}


def _eight_bits(x):
    """Rows of x as whole numbers of -127..127 (held in float32) and the float32 scale of each:
    q = rint(x * (127 / m)), scale = m / 127 with m the row's largest magnitude."""
    x = x.float()
    top = x.abs().amax(1).clamp_min(TINY)
    most = torch.full((), 127.0, device=x.device)
    return torch.round(x * torch.div(most, top)[:, None]), torch.div(top, most)


def _active(case, g, dev):
    """[steps, nodes] truth values: a node joins at its own step and stays (snapshots), or a
    sequence ends at its own length (a padded batch, batch first: [nodes, steps]); one in twenty is
    never there."""
    t, n = case["steps"], case["nodes"]
    at = torch.randint(0, t, (n,), generator=g, device=dev)
    at[torch.rand(n, generator=g, device=dev) < 0.5] = 0
    absent = torch.rand(n, generator=g, device=dev) < 0.05
    step = torch.arange(t, device=dev)[:, None]
    if case["batch_first"]:
        return ((step < t - at) & ~absent).t().contiguous()
    return (step >= at) & ~absent


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dt = _TYPES[case["dtype"]]

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=dev, dtype=dtype)

    s = {"case": case}
    if case["op"] == "norm":
        m, d = case["rows"], case["width"]
        s["x"] = (normal(m, d) * 1.5 + 0.25).to(dt)
        s["weight"], s["bias"] = 1 + 0.1 * normal(d), 0.1 * normal(d)
        if case["train"]:
            s["grad"] = normal(m, d, dtype=dt)
            for name in ("x", "weight", "bias"):
                s[name].requires_grad_()
    elif case["op"] == "scan":
        t, n, h = case["steps"], case["nodes"], case["hidden"]
        lead = (n, t) if case["batch_first"] else (t, n)
        s["gates"] = normal(*lead, 2 * h, dtype=dt)
        s["gates"][..., :h] += 1.5  # states that remember a few steps up to some hundreds
        s["h0"] = normal(n, h)
        s["active"] = _active(case, g, dev) if case["ragged"] else None
        if case["train"]:
            s["grad"], s["grad_last"] = normal(*lead, h, dtype=dt), normal(n, h)
            s["gates"].requires_grad_()
            s["h0"].requires_grad_()
    elif case["op"] == "step":
        m, n, h = case["rows"], case["nodes"], case["hidden"]
        s["gates"] = normal(m, 2 * h, dtype=dt)
        s["gates"][:, :h] += 1.5
        s["memory"] = normal(n, h)
        s["ids"] = torch.randperm(n, generator=g, device=dev)[:m]
    else:
        m, k, n = case["rows"], case["inner"], case["outer"]
        s["x"] = normal(m, k, dtype=dt)
        q, s["weight_scale"] = _eight_bits(normal(n, k) / math.sqrt(k))
        s["weight"] = q.to(torch.int8)
        s["bias"] = 0.1 * normal(n) if case["bias"] else None
    return s


# ------------------------------------------------------------------------------ plain forms
def _norm(s):
    x, w, b = s["x"].detach(), s["weight"].detach(), s["bias"].detach()
    x32 = x.float()
    d = x32 - x32.mean(1, keepdim=True)
    r = torch.rsqrt((d * d).mean(1, keepdim=True) + EPS)
    xh = d * r
    y = (xh * w + b).to(x.dtype)
    if not s["case"]["train"]:
        return {"y": y}
    g = s["grad"].float()
    gw = g * w
    dx = r * (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True))
    return {"y": y, "dx": dx.to(x.dtype), "dweight": (g * xh).sum(0), "dbias": g.sum(0)}


def _recur(a, b):
    """r[t] = a[t] r[t-1] + b[t] along the first axis, r[-1] = 0: pairs of (factor, sum) joined over
    distances 1, 2, 4, ..."""
    k = 1
    while k < a.shape[0]:
        b = torch.cat([b[:k], torch.addcmul(b[k:], a[k:], b[:-k])])
        a = torch.cat([a[:k], a[k:] * a[:-k]])
        k *= 2
    return b


def _scan(s):
    case, h = s["case"], s["case"]["hidden"]
    gates, h0, active = s["gates"].detach(), s["h0"].detach(), s["active"]
    turn = (lambda v: v.transpose(0, 1)) if case["batch_first"] else (lambda v: v)
    gate, cand = turn(gates[..., :h]).float(), turn(gates[..., h:]).float()
    keep, take = torch.sigmoid(gate), torch.sigmoid(-gate)
    if active is not None:
        there = turn(active)[..., None]
        keep = torch.where(there, keep, torch.ones_like(keep))
        take = torch.where(there, take, torch.zeros_like(take))
        cand = torch.where(there, cand, torch.zeros_like(cand))
    b = take * cand
    b[0] += keep[0] * h0
    state = _recur(keep, b)
    out = {"h": turn(state).to(gates.dtype), "last": state[-1]}
    if not case["train"]:
        return out
    # gradient with respect to each state: d[t] = g[t] + keep[t+1] d[t+1]
    g = turn(s["grad"]).float().clone()
    g[-1] += s["grad_last"]
    after = torch.cat([keep[1:], torch.zeros_like(keep[:1])])
    d = _recur(after.flip(0), g.flip(0)).flip(0)
    before = torch.cat([h0[None], state[:-1]])
    dgate = d * (before - cand) * keep * take
    dgates = torch.cat([turn(dgate), turn(d * take)], -1).to(gates.dtype)
    return {**out, "dgates": dgates, "dh0": keep[0] * d[0]}


def _step(s):
    h, mem, ids = s["case"]["hidden"], s["memory"], s["ids"]
    gate, cand = s["gates"][:, :h].float(), s["gates"][:, h:].float()
    new = torch.sigmoid(gate) * mem[ids] + torch.sigmoid(-gate) * cand
    mem[ids] = new
    return {"h": new, "memory": mem}


def _int8(s):
    q, scale = _eight_bits(s["x"])
    y = (q @ s["weight"].float().t()) * scale[:, None] * s["weight_scale"]
    if s["bias"] is not None:
        y = y + s["bias"]
    act = s["case"]["act"]
    if act != "none":
        y = torch.where(y > 0, y, y * (0.01 if act == "leaky_relu" else 0.0))
    return {"y": y.to(s["x"].dtype)}


# ----------------------------------------------------------------------- the framework's calls
def _own(s):
    from spiral_amd import ops

    case = s["case"]
    if case["op"] == "norm":
        y = ops.layer_norm(s["x"], s["weight"], s["bias"], EPS)
        if not case["train"]:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["grad"])
        return {"y": y, "dx": dx, "dweight": dw, "dbias": db}
    if case["op"] == "scan":
        h, last = ops.gated_scan(s["gates"], s["h0"], s["active"], batch_first=case["batch_first"])
        if not case["train"]:
            return {"h": h, "last": last}
        dgates, dh0 = torch.autograd.grad((h, last), (s["gates"], s["h0"]), (s["grad"], s["grad_last"]))
        return {"h": h, "last": last, "dgates": dgates, "dh0": dh0}
    if case["op"] == "step":
        return {"h": ops.gated_step(s["gates"], s["memory"], s["ids"]), "memory": s["memory"]}
    return {"y": ops.linear_int8(s["x"], s["weight"], s["weight_scale"], s["bias"], case["act"])}


def run(state):
    if own:
        return _own(state)
    return {"norm": _norm, "scan": _scan, "step": _step, "int8": _int8}[state["case"]["op"]](state)


def work(case):
    """Every input read once and every output written once."""
    size = 4 if case["dtype"] == F32 else 2
    if case["op"] == "norm":
        cells = case["rows"] * case["width"]
        ends = 2 * 4 * case["width"]
        if case["train"]:
            return {"bytes": 4 * size * cells + 2 * ends, "flops": 20 * cells}
        return {"bytes": 2 * size * cells + ends, "flops": 8 * cells}
    if case["op"] == "scan":
        cells, rim = case["steps"] * case["nodes"] * case["hidden"], 4 * case["nodes"] * case["hidden"]
        mask = case["steps"] * case["nodes"] if case["ragged"] else 0
        if case["train"]:
            return {"bytes": 6 * size * cells + 4 * rim + mask, "flops": 20 * cells}
        return {"bytes": 3 * size * cells + 2 * rim + mask, "flops": 8 * cells}
    if case["op"] == "step":
        cells = case["rows"] * case["hidden"]
        return {"bytes": (2 * size + 3 * 4) * cells + 8 * case["rows"], "flops": 8 * cells}
    m, k, n = case["rows"], case["inner"], case["outer"]
    return {"bytes": size * m * (k + n) + n * k + (8 if case["bias"] else 4) * n, "flops": 2 * m * n * k}


# -------------------------------------------------------------------------- the definitions
def _exact_norm(s):
    x, w, b = s["x"].detach().double(), s["weight"].detach().double(), s["bias"].detach().double()
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    xh = (x - mean) / (var + EPS).sqrt()
    out = {"y": xh * w + b}
    if s["case"]["train"]:
        g, d = s["grad"].double(), x.shape[1]
        out["dbias"] = g.sum(0)
        out["dweight"] = torch.einsum("md,md->d", g, xh)
        v = g * w
        # the projection of v onto what is orthogonal to 1 and to xh, over the deviation
        along = (v * xh).sum(1, keepdim=True) / d
        out["dx"] = (v - v.sum(1, keepdim=True) / d - along * xh) / (var + EPS).sqrt()
    return out


def _exact_scan(s):
    case, h = s["case"], s["case"]["hidden"]
    gates, active = s["gates"].detach(), s["active"]
    if case["batch_first"]:
        gates, active = gates.transpose(0, 1), None if active is None else active.t()
    t_end = case["steps"]

    def at(t):
        z, c = gates[t, :, :h].double(), gates[t, :, h:].double()
        on = torch.ones(case["nodes"], 1, dtype=torch.bool, device=z.device) if active is None else active[t][:, None]
        return 1 / (1 + torch.exp(-z)), 1 / (1 + torch.exp(z)), c, on

    state = s["h0"].detach().double()
    states = torch.empty(t_end + 1, *state.shape, dtype=torch.float64, device=state.device)
    states[0] = state
    for t in range(t_end):
        a, rest, c, on = at(t)
        state = torch.where(on, a * state + rest * c, state)
        states[t + 1] = state
    turn = (lambda v: v.transpose(0, 1).contiguous()) if case["batch_first"] else (lambda v: v)
    out = {"h": turn(states[1:]), "last": states[-1]}
    if case["train"]:
        grad = s["grad"].transpose(0, 1) if case["batch_first"] else s["grad"]
        dgates = torch.empty(t_end, case["nodes"], 2 * h, dtype=torch.float64, device=state.device)
        coming = s["grad_last"].double()
        for t in reversed(range(t_end)):
            a, rest, c, on = at(t)
            d = coming + grad[t].double()
            zero = torch.zeros_like(d)
            dgates[t, :, :h] = torch.where(on, d * (states[t] - c) * a * rest, zero)
            dgates[t, :, h:] = torch.where(on, d * rest, zero)
            coming = torch.where(on, a * d, d)
        out["dgates"], out["dh0"] = turn(dgates), coming
    return out


def _exact_step(s):
    h, mem, ids = s["case"]["hidden"], s["memory"].double(), s["ids"]
    z, c = s["gates"][:, :h].double(), s["gates"][:, h:].double()
    new = c + (mem[ids] - c) / (1 + torch.exp(-z))
    mem[ids] = new
    return {"h": new, "memory": mem}


def _exact_int8(s):
    # the whole numbers are defined by float32 arithmetic (quotient and product rounded once
    # each, which double precision followed by one rounding gives); everything after is not rounded
    x = s["x"].double()
    top = x.abs().amax(1, keepdim=True).clamp_min(TINY)
    q = torch.round((x * (127.0 / top).float().double()).float()).double()
    y = (q @ s["weight"].double().t()) * (top / 127.0) * s["weight_scale"].double()
    if s["bias"] is not None:
        y = y + s["bias"].double()
    act = s["case"]["act"]
    if act == "relu":
        y = y.clamp_min(0)
    elif act == "leaky_relu":
        y = torch.maximum(y, 0.01 * y)
    return {"y": y}


def exact(case, seed):
    form = {"norm": _exact_norm, "scan": _exact_scan, "step": _exact_step, "int8": _exact_int8}[case["op"]]
    return form(prepare(case, seed))
