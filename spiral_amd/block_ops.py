"""The operators of a gated-linear-recurrence decoder block: layer norm, the recurrence as a scan
over a sequence and as one step on the node memory, and the projection in 8-bit integers.  They are
part of `spiral_amd.ops`, which offers them under the same names.

Each call queues its kernels on torch's current stream of the device its tensors live on, takes its
workspace from torch's allocator for that stream, and waits for nothing, so it can be captured into
a graph and run on any stream.  (torch's own rule holds for capturing a backward pass: no eager graph
of the same leaves may be alive on another stream meanwhile.)

A small call is bound by the host: a launch costs ~3 us there and torch.empty ~1 us, so the wrappers
look at each argument once, ask for the raw stream, and switch the device only where it differs."""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _native as nv
from .graph import _ACT_CODES

_F32 = torch.float32
_DTYPE_CODES = {torch.float32: 0, torch.bfloat16: 1}
LAYER_NORM_MAX_WIDTH = 16384  # spmi_layer_norm_max_width()
INT8_MAX_INNER = 131072       # 127^2 times this still fits the 32-bit sums

_INT8_MAX_STRIDE = 1 << 24     # values from one row to the next, in x and in the result

_tracking = torch.is_grad_enabled
_empty = torch.empty


def _refuse(what: str) -> None:
    raise nv.SpmiError(what)


def _code(t: torch.Tensor, what: str) -> int:
    code = _DTYPE_CODES.get(t.dtype)
    if code is None:
        _refuse(f"{what} must be float32 or bfloat16, got {t.dtype}")
    return code


def _device_of(t: torch.Tensor, *others: Optional[torch.Tensor]) -> int:
    """The device all of these live on."""
    at = t.get_device()
    for o in others:
        if o is not None and o.get_device() != at:
            at = -1
            break
    if at < 0:
        nv.require_cuda(t, *others)
        _refuse(f"tensors on different devices: {[str(o.device) for o in (t, *others) if o is not None]}")
    return at


def _no_tangent(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """Refuse inputs of forward-mode differentiation: the kernels know nothing of a tangent and would
    drop it.  Outside a dual level, which is nearly always, this is one comparison."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                _refuse(f"{what} has no forward-mode derivative")


def _rows_of(t: torch.Tensor) -> torch.Tensor:
    """[..., D] as a matrix of rows with neighbouring values (a view where the strides allow it)."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _units_last(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _float_vector(v: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """A vector of parameters as the kernels read it: float32, contiguous."""
    if v is None or (v.dtype == _F32 and v.is_contiguous()):
        return v
    return v.detach().to(_F32).contiguous()


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _workspace(nbytes: int, device: torch.device) -> Optional[torch.Tensor]:
    return _empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _launch(name: str, at: int, *args) -> None:
    """Queue entry point `name` on the current stream of device `at`."""
    fn = getattr(nv.lib(), name)
    if nv.current_device() == at:
        rc = fn(*args, nv.raw_stream(at))
    else:
        with torch.cuda.device(at):
            rc = fn(*args, nv.raw_stream(at))
    if rc:
        nv.check(rc, name)


class _OnceOnly(torch.autograd.Function):
    """Gradients as they are, in a graph that leads back to `anchors` and cannot be walked."""

    @staticmethod
    def forward(ctx, name, anchors, *values):
        ctx.name = name
        return tuple(v.detach() for v in values[anchors:])

    @staticmethod
    def backward(ctx, *g):
        _refuse(f"{ctx.name} has no second derivative")


class _Operator(torch.autograd.Function):
    """Base of the operators below: `gradients(ctx, saved, *g)` is the backward pass.  It runs kernels
    autograd does not see, so a second derivative through it raises instead of being wrong: where a
    graph of the backward pass is recorded, its results depend on whatever they were computed
    from, the saved inputs as well as the incoming gradients, through a node that raises.  (The saved
    tensors are asked for once: activation checkpointing hands them out once.)"""

    @staticmethod
    def gradients(ctx, saved, *g):
        raise NotImplementedError

    @classmethod
    def _bind(cls, name):
        plain = cls.gradients

        def backward(ctx, *g):
            saved = ctx.saved_tensors
            if not _tracking():
                return plain(ctx, saved, *g)
            with torch.no_grad():
                found = list(plain(ctx, saved, *g))
            anchors = [t for t in (*saved, *g) if t is not None and t.requires_grad]
            at = [i for i, t in enumerate(found) if t is not None]
            if anchors and at:
                for i, t in zip(at, _OnceOnly.apply(name, len(anchors), *anchors, *(found[i] for i in at))):
                    found[i] = t
            return tuple(found)

        cls.backward = staticmethod(backward)
        return cls


# --------------------------------------------------------------------------- layer norm
def _layer_norm_fwd(xr, shape, weight, bias, eps, code, at, keep):
    m, d = xr.shape
    w, b = _float_vector(weight), _float_vector(bias)
    y = _empty(shape, dtype=xr.dtype, device=xr.device)
    stats = _empty(m, 2, dtype=_F32, device=xr.device) if keep else None
    _launch("spmi_layer_norm_fwd", at, xr.data_ptr(), code, xr.stride(0), m, d, _ptr(w), _ptr(b), eps, y.data_ptr(),
            d, _ptr(stats))
    return y, stats


class _LayerNorm(_Operator):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, code, at):
        xr = _rows_of(x)
        y, stats = _layer_norm_fwd(xr, x.shape, weight, bias, eps, code, at, True)
        ctx.save_for_backward(x, weight, stats)
        m, d = xr.shape
        # what the backward pass would otherwise ask for again, in a thread that is slow at asking
        ctx.plain = (code, at, m, d, xr.stride(0) if xr.data_ptr() == x.data_ptr() else None,
                     nv.lib().spmi_layer_norm_bwd_workspace_bytes(m, d), None if bias is None else bias.dtype)
        return y

    @staticmethod
    def gradients(ctx, saved, g):
        x, weight, stats = saved
        code, at, m, d, ld, ws_bytes, bias_dtype = ctx.plain
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dev = x.device
        if ld is None:
            x = _rows_of(x)
            ld = x.stride(0)
        ldg = d
        shape = g.shape
        if not g.is_contiguous():
            g = _rows_of(g)
            ldg = g.stride(0)
        w = _float_vector(weight)
        dx = _empty(shape, dtype=x.dtype, device=dev) if need_x else None
        dw = _empty(d, dtype=_F32, device=dev) if need_w else None
        db = _empty(d, dtype=_F32, device=dev) if need_b else None
        if not (need_w or need_b):
            ws_bytes = 0
        ws = _workspace(ws_bytes, dev)
        _launch("spmi_layer_norm_bwd", at, x.data_ptr(), g.data_ptr(), code, ld, ldg, m, d, _ptr(w), stats.data_ptr(),
                _ptr(dx), d, _ptr(dw), _ptr(db), _ptr(ws), ws_bytes)
        if need_w and weight.dtype != _F32:
            dw = dw.to(weight.dtype)
        if need_b and bias_dtype != _F32:
            db = db.to(bias_dtype)
        return dx, dw, db, None, None, None


_LayerNorm._bind("layer_norm")


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last dimension of x [..., D],
    differentiable in x, weight and bias.  x: float32 or bfloat16 of any strides, D from 1 to 16384;
    weight and bias: [D] in either type, or None.  Statistics and gradient sums are float32; the
    gradients of weight and bias are added up in a fixed order (the same bits every time).  There is
    no second derivative and no forward mode; a call that would need one is refused."""
    code = _code(x, "layer_norm: x")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= LAYER_NORM_MAX_WIDTH:
        _refuse(f"layer_norm: the last dimension of x must be 1 to {LAYER_NORM_MAX_WIDTH}, got {tuple(x.shape)}")
    grad = x.requires_grad
    for v in (weight, bias):
        if v is not None:
            _code(v, "layer_norm: weight and bias")
            if v.shape != x.shape[-1:]:
                _refuse(f"layer_norm: weight and bias must have shape ({x.shape[-1]},), got {tuple(v.shape)}")
            grad = grad or v.requires_grad
    eps = float(eps)
    if not 0.0 <= eps < float("inf"):
        _refuse(f"layer_norm: eps must be finite and not negative, got {eps}")
    _no_tangent("layer_norm", x, weight, bias)
    at = _device_of(x, weight, bias)
    if grad and _tracking():
        return _LayerNorm.apply(x, weight, bias, eps, code, at)
    return _layer_norm_fwd(_rows_of(x), x.shape, weight, bias, eps, code, at, False)[0]


# --------------------------------------------------------------------------- gated linear recurrence
def _step_strides(t: Optional[torch.Tensor], batch_first: bool) -> Tuple[int, int]:
    """Strides along steps and along nodes."""
    if t is None:
        return 0, 0
    return (t.stride(1), t.stride(0)) if batch_first else (t.stride(0), t.stride(1))


def _scan_sizes(gates, h0, active, batch_first, h):
    """The numbers both directions take: strides of gates, h0, active and h, and T, N, H."""
    n, t = gates.shape[:2] if batch_first else (gates.shape[1], gates.shape[0])
    return (_step_strides(gates, batch_first), 0 if h0 is None else h0.stride(0), _step_strides(active, batch_first),
            (t, n, gates.shape[2] // 2), _step_strides(h, batch_first))


def _scan_bwd(gates, h0, active, batch_first, code, at, h, states, g, g_last, dgates, dh0, sizes, ws_bytes):
    of_gates, of_h0, of_active, tnh, of_h = sizes
    ws = _workspace(ws_bytes, gates.device)
    _launch("spmi_gated_scan_bwd", at, gates.data_ptr(), code, *of_gates, _ptr(h0), of_h0, _ptr(active), *of_active,
            *tnh, _ptr(h), *of_h, _ptr(states), _ptr(g), *_step_strides(g, batch_first), _ptr(g_last),
            0 if g_last is None else g_last.stride(0), _ptr(dgates), *_step_strides(dgates, batch_first), _ptr(dh0),
            _ptr(ws), ws_bytes)


def _scan_fwd(gates, h0, active, batch_first, code, at, keep):
    gates = _units_last(gates)
    if h0 is not None:
        h0 = _units_last(h0)
    dev = gates.device
    h = _empty(*gates.shape[:2], gates.shape[2] // 2, dtype=gates.dtype, device=dev)
    sizes = _scan_sizes(gates, h0, active, batch_first, h)
    of_gates, of_h0, of_active, tnh, of_h = sizes
    last = _empty(tnh[1:], dtype=_F32, device=dev)
    ws_bytes = nv.lib().spmi_gated_scan_fwd_workspace_bytes(*tnh)
    ws = _workspace(ws_bytes, dev)
    # float32 states are whole in h; of those stored in bfloat16 the backward pass gets some in float32 as well
    states = None
    if keep and gates.dtype != _F32:
        states = _empty(nv.lib().spmi_gated_scan_states(*tnh), *tnh[1:], dtype=_F32, device=dev)
    _launch("spmi_gated_scan_fwd_saved", at, gates.data_ptr(), code, *of_gates, _ptr(h0), of_h0, _ptr(active),
            *of_active, *tnh, h.data_ptr(), *of_h, last.data_ptr(), _ptr(states), _ptr(ws), ws_bytes)
    return h, last, states, sizes


class _GatedScan(_Operator):
    @staticmethod
    def forward(ctx, gates, h0, active, batch_first, code, at):
        h, last, states, sizes = _scan_fwd(gates, h0, active, batch_first, code, at, True)
        ctx.save_for_backward(gates, h0, active, h if states is None else None, states)
        ctx.plain = (batch_first, code, at, sizes, nv.lib().spmi_gated_scan_bwd_workspace_bytes(*sizes[3]))
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    def gradients(ctx, saved, g, g_last):
        gates, h0, active, h, states = saved
        batch_first, code, at, sizes, ws_bytes = ctx.plain
        need_gates, need_h0 = ctx.needs_input_grad[:2]
        if g is None and g_last is None:
            return None, None, None, None, None, None
        gates = _units_last(gates)  # the same copy as in forward, if it was one: sizes fit
        if h0 is not None:
            h0 = _units_last(h0)
        dgates = _empty(gates.shape, dtype=gates.dtype, device=gates.device) if need_gates else None
        dh0 = _empty(h0.shape, dtype=_F32, device=gates.device) if need_h0 else None
        _scan_bwd(gates, h0, active, batch_first, code, at, h, states, None if g is None else _units_last(g),
                  None if g_last is None else _units_last(g_last), dgates, dh0, sizes, ws_bytes)
        return dgates, dh0, None, None, None, None


_GatedScan._bind("gated_scan")


def gated_scan(gates: torch.Tensor, h0: Optional[torch.Tensor] = None, active: Optional[torch.Tensor] = None,
               batch_first: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """The gated linear recurrence over a sequence, differentiable in `gates` and `h0`:

        h_t = a_t h_{t-1} + (1 - a_t) c_t,   a_t = sigmoid(z_t)

    gates: [T, N, 2H] ([N, T, 2H] with `batch_first`), the logits z and then the candidates c of each
    row (one projection's output), float32 or bfloat16.  h0: float32 [N, H], None for zeros.  active:
    bool [T, N] ([N, T]); where it is False the node's state passes the step unchanged, its gates
    are not used (they may hold anything) and receive a zero gradient.  A node that joins late or a
    sequence that ends early is described by it.  Returns the states [T, N, H] ([N, T, H]) in the
    type of `gates` and the last state [N, H] in float32 (h0 where no step is active).

    The gradient is that of float32 states whatever the type of `gates`: with bfloat16, a tracked call keeps
    a float32 state for every 4 steps (2 where the channels are few) besides."""
    code = _code(gates, "gated_scan: gates")
    if gates.dim() != 3 or gates.shape[2] < 2 or gates.shape[2] % 2:
        _refuse(f"gated_scan: gates must be [T, N, 2H], got {tuple(gates.shape)}")
    batch_first = bool(batch_first)
    n, hd = gates.shape[0 if batch_first else 1], gates.shape[2] // 2
    grad = gates.requires_grad
    if h0 is not None:
        if h0.shape != (n, hd) or h0.dtype != _F32:
            _refuse(f"gated_scan: h0 must be float32 [{n}, {hd}], got {h0.dtype} {tuple(h0.shape)}")
        grad = grad or h0.requires_grad
    if active is not None and (active.dtype != torch.bool or active.shape != gates.shape[:2]):
        _refuse(f"gated_scan: active must be bool {tuple(gates.shape[:2])}, got {active.dtype} {tuple(active.shape)}")
    _no_tangent("gated_scan", gates, h0)
    at = _device_of(gates, h0, active)
    if grad and _tracking():
        return _GatedScan.apply(gates, h0, active, batch_first, code, at)
    return _scan_fwd(gates, h0, active, batch_first, code, at, False)[:2]


def _step_fwd(gates, h_mem, ids, mem_write, code, at, keep):
    gates = _units_last(gates)
    m, hd = gates.shape[0], gates.shape[1] // 2
    nodes = h_mem.shape[0]
    h = _empty(m, hd, dtype=_F32, device=gates.device)
    before = _empty(m, hd, dtype=_F32, device=gates.device) if keep else None
    ws_bytes = nv.lib().spmi_gated_step_workspace_bytes(m, nodes) if mem_write and ids is not None else 0
    ws = _workspace(ws_bytes, gates.device)
    _launch("spmi_gated_step", at, gates.data_ptr(), code, gates.stride(0), h_mem.data_ptr(), nodes, _ptr(ids), m, hd,
            h.data_ptr(), _ptr(before), mem_write, _ptr(ws), ws_bytes)
    if mem_write:
        torch.autograd.graph.increment_version(h_mem)
    return h, before


class _GatedStep(_Operator):
    @staticmethod
    def forward(ctx, gates, h_mem, ids, mem_write, code, at):
        h, before = _step_fwd(gates, h_mem, ids, mem_write, code, at, True)
        ctx.save_for_backward(gates, before)
        ctx.plain = (code, at)
        return h

    @staticmethod
    def gradients(ctx, saved, g):
        # the scan's backward pass over one step, with the rows' old states as its start
        gates, before = saved
        gates = _units_last(gates)
        dgates = _empty(gates.shape, dtype=gates.dtype, device=gates.device)
        m, h2 = gates.shape
        sizes = ((0, gates.stride(0)), h2 // 2, (0, 0), (1, m, h2 // 2), (0, 0))
        _scan_bwd(gates, before, None, False, *ctx.plain, None, None, None, _units_last(g), dgates[None], None, sizes, 0)
        return dgates, None, None, None, None, None


_GatedStep._bind("gated_step")


def gated_step(gates: torch.Tensor, h_mem: torch.Tensor, ids: Optional[torch.Tensor] = None,
               mem_write: bool = True) -> torch.Tensor:
    """One step of the gated linear recurrence on rows of the node memory: `gates` [M, 2H] (logits and
    candidates, float32 or bfloat16), `h_mem` [nodes, H] float32 and contiguous, `ids` int64 [M] the
    node of each row (None: row i is node i, M <= nodes).  Returns the new states, float32 [M, H],
    and with `mem_write` puts them into the memory in place.  Differentiable in `gates`; the memory
    is a state, no gradient goes through it.

    Every row starts from the memory as it was before the call.  Where `ids` names a node several
    times the memory keeps the last of its rows.  A row whose id is outside [0, nodes) comes out as
    NaN and is written nowhere else."""
    code = _code(gates, "gated_step: gates")
    if gates.dim() != 2 or gates.shape[1] < 2 or gates.shape[1] % 2:
        _refuse(f"gated_step: gates must be [M, 2H], got {tuple(gates.shape)}")
    m, hd = gates.shape[0], gates.shape[1] // 2
    if h_mem.dim() != 2 or h_mem.shape[1] != hd or h_mem.dtype != _F32 or not h_mem.is_contiguous():
        _refuse(f"gated_step: the node memory must be contiguous float32 [nodes, {hd}], got {h_mem.dtype} "
                f"{tuple(h_mem.shape)}")
    if h_mem.requires_grad and _tracking():
        _refuse("gated_step: the node memory is a state and takes no gradient")
    if ids is None:
        if m > h_mem.shape[0]:
            _refuse("gated_step: more rows than nodes in the memory")
    elif ids.dtype != torch.int64 or ids.shape != (m,):
        _refuse(f"gated_step: ids must be int64 [{m}], got {ids.dtype} {tuple(ids.shape)}")
    elif not ids.is_contiguous():
        ids = ids.contiguous()
    _no_tangent("gated_step", gates, h_mem)
    at = _device_of(gates, h_mem, ids)
    mem_write = bool(mem_write)
    if gates.requires_grad and _tracking():
        return _GatedStep.apply(gates, h_mem, ids, mem_write, code, at)
    return _step_fwd(gates, h_mem, ids, mem_write, code, at, False)[0]


# --------------------------------------------------------------------------- 8-bit integers
def quantize_rows_int8(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows of x [..., K] (float32 or bfloat16) in 8-bit integers: `q` int8 of x's shape and `scale`
    float32 of its leading shape, x = q * scale to within half a scale.  With m the row's largest
    magnitude (at least 2^-120), scale = m / 127 and q = rint(x * (127 / m)), each operation rounded
    to float32.  A row with a value that is not finite gets q = 0 and scale = NaN.  Applied to a
    weight [N, K] this gives the arguments of `linear_int8`.  Both results are constants to autograd."""
    code = _code(x, "quantize_rows_int8: x")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= INT8_MAX_INNER:
        _refuse(f"quantize_rows_int8: the last dimension of x must be 1 to {INT8_MAX_INNER}, got {tuple(x.shape)}")
    _no_tangent("quantize_rows_int8", x)
    at = _device_of(x)
    xr = _rows_of(x)
    m, k = xr.shape
    q = _empty(x.shape, dtype=torch.int8, device=x.device)
    scale = _empty(x.shape[:-1], dtype=_F32, device=x.device)
    _launch("spmi_quantize_rows_i8", at, xr.data_ptr(), code, xr.stride(0), m, k, q.data_ptr(), k, scale.data_ptr())
    return q, scale


def linear_int8(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                bias: Optional[torch.Tensor] = None, act: Optional[str] = None, slope: float = 0.01,
                out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """act(x @ (weight * weight_scale[:, None]).T + bias) with the products in 8-bit integers: the
    rows of x [..., K] (float32 or bfloat16) are brought to whole numbers with a scale each
    (`quantize_rows_int8`), the sums over K are exact, scales, bias and activation (None, "relu" or
    "leaky_relu" with `slope`) follow in float32, and the result [..., N] is rounded once to
    `out_dtype` (default: x's type).  weight: int8 [N, K], weight_scale: float32 [N]; K up to 131072.
    A result depends on its own row of x and its own channel alone, to the bit.  For serving: there is no backward pass, and a call that would need one is refused."""
    code = _code(x, "linear_int8: x")
    if weight.dim() != 2 or weight.dtype != torch.int8:
        _refuse(f"linear_int8: weight must be int8 [N, K], got {weight.dtype} {tuple(weight.shape)}")
    n, k = weight.shape
    if n >= _INT8_MAX_STRIDE:
        _refuse(f"linear_int8: {n} output channels are too many (below {_INT8_MAX_STRIDE})")
    if x.dim() < 1 or x.shape[-1] != k or not 1 <= k <= INT8_MAX_INNER:
        _refuse(f"linear_int8: x {tuple(x.shape)} does not fit a weight {tuple(weight.shape)}")
    if weight_scale.shape != (n,) or weight_scale.dtype != _F32:
        _refuse(f"linear_int8: weight_scale must be float32 [{n}]")
    grad = x.requires_grad or weight_scale.requires_grad
    if bias is not None:
        if bias.shape != (n,):
            _refuse(f"linear_int8: bias must have shape ({n},), got {tuple(bias.shape)}")
        _code(bias, "linear_int8: bias")
        grad = grad or bias.requires_grad
    act_code = _ACT_CODES.get(act)
    if act_code is None:
        _refuse(f"linear_int8: unknown activation {act!r}")
    if out_dtype is None:
        out_dtype = x.dtype
    out_code = _DTYPE_CODES.get(out_dtype)
    if out_code is None:
        _refuse("linear_int8: out_dtype must be float32 or bfloat16")
    if grad and _tracking():
        _refuse("linear_int8 has no backward pass: call it under torch.no_grad()")
    _no_tangent("linear_int8", x, weight_scale, bias)
    at = _device_of(x, weight, weight_scale, bias)
    bias = _float_vector(bias)
    xr, w, s = _rows_of(x), _units_last(weight), _float_vector(weight_scale)
    m, ld = xr.shape[0], xr.stride(0)
    if ld >= _INT8_MAX_STRIDE:  # a single row's stride says nothing, and torch calls such a view contiguous
        xr, ld = xr.contiguous(), k
    out = _empty(*x.shape[:-1], n, dtype=out_dtype, device=x.device)
    ws_bytes = nv.lib().spmi_linear_i8_workspace_bytes(m, k, n)
    ws = _workspace(ws_bytes, x.device)
    _launch("spmi_linear_i8", at, xr.data_ptr(), code, ld, m, k, w.data_ptr(), w.stride(0), s.data_ptr(), n,
            _ptr(bias), act_code, slope, out.data_ptr(), out_code, n, _ptr(ws), ws_bytes)
    return out
