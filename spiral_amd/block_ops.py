"""The operators of a gated-linear-recurrence decoder block: layer norm, the recurrence as a scan
over a sequence and as one step on the node memory, and the projection in 8-bit integers.  They are
part of `spiral_amd.ops`, which offers them under the same names.

Each call queues its kernels on torch's current stream of the device its tensors live on, takes its
workspace from torch's allocator for that stream, and waits for nothing, so it can be captured into
a graph and run on any stream."""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _native as nv
from .graph import _ACT_CODES

_DTYPE_CODES = {torch.float32: 0, torch.bfloat16: 1}


def _rows_dtype(t: torch.Tensor, what: str) -> int:
    code = _DTYPE_CODES.get(t.dtype)
    if code is None:
        raise nv.SpmiError(f"{what} must be float32 or bfloat16, got {t.dtype}")
    return code


def _same_device(t: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
    nv.require_cuda(t, *others)
    for o in others:
        if o is not None and o.device != t.device:
            raise nv.SpmiError(f"tensors on different devices: {t.device} and {o.device}")


def _rows_of(t: torch.Tensor) -> torch.Tensor:
    """[..., D] as a matrix of rows with neighbouring values (a view where the strides allow it)."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _workspace(nbytes: int, device: torch.device) -> Optional[torch.Tensor]:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _tracked(*tensors: Optional[torch.Tensor]) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# --------------------------------------------------------------------------- layer norm
LAYER_NORM_MAX_WIDTH = 16384  # spmi_layer_norm_max_width()


def _float_vector(v: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if v is None else v.detach().to(torch.float32).contiguous()


def _layer_norm_fwd(x, weight, bias, eps, keep):
    xd = _rows_of(x.detach())
    m, d = xd.shape
    w, b = _float_vector(weight), _float_vector(bias)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty(m, 2, dtype=torch.float32, device=x.device) if keep else None
    with torch.cuda.device(x.device):
        nv.check(nv.lib().spmi_layer_norm_fwd(nv.ptr(xd), _DTYPE_CODES[x.dtype], xd.stride(0), m, d, nv.ptr(w),
                                              nv.ptr(b), eps, nv.ptr(y), d, nv.ptr(stats), nv.stream()),
                 "spmi_layer_norm_fwd")
    return y, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _layer_norm_fwd(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, stats)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        x, weight, stats = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        xd, gd = _rows_of(x.detach()), _rows_of(g)
        m, d = xd.shape
        dev = x.device
        w = _float_vector(weight)
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
        dw = torch.empty(d, dtype=torch.float32, device=dev) if need_w else None
        db = torch.empty(d, dtype=torch.float32, device=dev) if need_b else None
        lib = nv.lib()
        ws_bytes = lib.spmi_layer_norm_bwd_workspace_bytes(m, d) if need_w or need_b else 0
        with torch.cuda.device(dev):
            ws = _workspace(ws_bytes, dev)
            nv.check(lib.spmi_layer_norm_bwd(nv.ptr(xd), nv.ptr(gd), _DTYPE_CODES[x.dtype], xd.stride(0),
                                             gd.stride(0), m, d, nv.ptr(w), nv.ptr(stats), nv.ptr(dx), d, nv.ptr(dw),
                                             nv.ptr(db), nv.ptr(ws), ws_bytes, nv.stream()), "spmi_layer_norm_bwd")
        return (dx, dw.to(weight.dtype) if need_w else None, db.to(ctx.bias_dtype) if need_b else None, None)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last dimension of x [..., D],
    differentiable in x, weight and bias.  x: float32 or bfloat16 of any strides, D from 1 to 16384;
    weight and bias: [D] in either type, or None.  Statistics and gradient sums are float32; the
    gradients of weight and bias are added up in a fixed order (the same bits every time)."""
    _rows_dtype(x, "layer_norm: x")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= LAYER_NORM_MAX_WIDTH:
        raise nv.SpmiError(f"layer_norm: the last dimension of x must be 1 to {LAYER_NORM_MAX_WIDTH}, got "
                           f"{tuple(x.shape)}")
    for name, v in (("weight", weight), ("bias", bias)):
        if v is not None:
            _rows_dtype(v, f"layer_norm: {name}")
            if v.shape != x.shape[-1:]:
                raise nv.SpmiError(f"layer_norm: {name} must have shape ({x.shape[-1]},), got {tuple(v.shape)}")
    eps = float(eps)
    if not 0.0 <= eps < float("inf"):
        raise nv.SpmiError(f"layer_norm: eps must be finite and not negative, got {eps}")
    _same_device(x, weight, bias)
    if _tracked(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps)
    return _layer_norm_fwd(x, weight, bias, eps, False)[0]


# --------------------------------------------------------------------------- gated linear recurrence
def _units_last(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _step_strides(t: torch.Tensor, batch_first: bool) -> Tuple[int, int]:
    """Strides along steps and along nodes."""
    return (t.stride(1), t.stride(0)) if batch_first else (t.stride(0), t.stride(1))


def _scan_call(direction, gates, h0, active, batch_first, h, last, g=None, g_last=None, dgates=None, dh0=None):
    n, t = gates.shape[:2] if batch_first else (gates.shape[1], gates.shape[0])
    hd = gates.shape[2] // 2
    lib = nv.lib()
    a_t, a_n = (0, 0) if active is None else _step_strides(active, batch_first)
    head = (nv.ptr(gates), _DTYPE_CODES[gates.dtype], *_step_strides(gates, batch_first), nv.ptr(h0),
            0 if h0 is None else h0.stride(0), nv.ptr(active), a_t, a_n, t, n, hd, nv.ptr(h),
            *_step_strides(h, batch_first))
    with torch.cuda.device(gates.device):
        if direction == "fwd":
            ws_bytes = lib.spmi_gated_scan_fwd_workspace_bytes(t, n, hd)
            ws = _workspace(ws_bytes, gates.device)
            nv.check(lib.spmi_gated_scan_fwd(*head, nv.ptr(last), nv.ptr(ws), ws_bytes, nv.stream()),
                     "spmi_gated_scan_fwd")
        else:
            ws_bytes = lib.spmi_gated_scan_bwd_workspace_bytes(t, n, hd)
            ws = _workspace(ws_bytes, gates.device)
            g_t, g_n = (0, 0) if g is None else _step_strides(g, batch_first)
            d_t, d_n = (0, 0) if dgates is None else _step_strides(dgates, batch_first)
            nv.check(lib.spmi_gated_scan_bwd(*head, nv.ptr(g), g_t, g_n, nv.ptr(g_last),
                                             0 if g_last is None else g_last.stride(0), nv.ptr(dgates), d_t, d_n,
                                             nv.ptr(dh0), nv.ptr(ws), ws_bytes, nv.stream()), "spmi_gated_scan_bwd")


def _scan_fwd(gates, h0, active, batch_first):
    gd = _units_last(gates.detach())
    hd = gd.shape[2] // 2
    h0d = None if h0 is None else _units_last(h0.detach())
    h = torch.empty(*gd.shape[:2], hd, dtype=gd.dtype, device=gd.device)
    last = torch.empty(gd.shape[0 if batch_first else 1], hd, dtype=torch.float32, device=gd.device)
    _scan_call("fwd", gd, h0d, active, batch_first, h, last)
    return h, last


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gates, h0, active, batch_first):
        h, last = _scan_fwd(gates, h0, active, batch_first)
        ctx.save_for_backward(gates, h0, active, h)
        ctx.batch_first = batch_first
        ctx.set_materialize_grads(False)
        return h, last

    @staticmethod
    @once_differentiable
    def backward(ctx, g, g_last):
        gates, h0, active, h = ctx.saved_tensors
        need_gates, need_h0 = ctx.needs_input_grad[:2]
        if g is None and g_last is None:
            return None, None, None, None
        gd = _units_last(gates.detach())
        h0d = None if h0 is None else _units_last(h0.detach())
        dgates = torch.empty(gd.shape, dtype=gd.dtype, device=gd.device) if need_gates else None
        dh0 = torch.empty(h0.shape, dtype=torch.float32, device=gd.device) if need_h0 else None
        _scan_call("bwd", gd, h0d, active, ctx.batch_first, h, None,
                   None if g is None else _units_last(g), None if g_last is None else _units_last(g_last),
                   dgates, dh0)
        return dgates, dh0, None, None


def gated_scan(gates: torch.Tensor, h0: Optional[torch.Tensor] = None, active: Optional[torch.Tensor] = None,
               batch_first: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """The gated linear recurrence over a sequence, differentiable in `gates` and `h0`:

        h_t = a_t h_{t-1} + (1 - a_t) c_t,   a_t = sigmoid(z_t)

    gates: [T, N, 2H] ([N, T, 2H] with `batch_first`), the logits z and then the candidates c of each
    row (one projection's output), float32 or bfloat16.  h0: float32 [N, H], None for zeros.  active:
    bool [T, N] ([N, T]); where it is False the node's state passes the step unchanged, its gates
    are not used (they may hold anything) and receive a zero gradient.  A node that joins late or a
    sequence that ends early is described by it.  Returns the states [T, N, H] ([N, T, H]) in the
    type of `gates` and the last state [N, H] in float32 (h0 where no step is active)."""
    _rows_dtype(gates, "gated_scan: gates")
    if gates.dim() != 3 or gates.shape[2] < 2 or gates.shape[2] % 2:
        raise nv.SpmiError(f"gated_scan: gates must be [T, N, 2H], got {tuple(gates.shape)}")
    n, hd = gates.shape[0 if batch_first else 1], gates.shape[2] // 2
    if h0 is not None and (h0.shape != (n, hd) or h0.dtype != torch.float32):
        raise nv.SpmiError(f"gated_scan: h0 must be float32 [{n}, {hd}], got {h0.dtype} {tuple(h0.shape)}")
    if active is not None:
        if active.dtype != torch.bool or active.shape != gates.shape[:2]:
            raise nv.SpmiError(f"gated_scan: active must be bool {tuple(gates.shape[:2])}, got {active.dtype} "
                               f"{tuple(active.shape)}")
    _same_device(gates, h0, active)
    if _tracked(gates, h0):
        return _GatedScan.apply(gates, h0, active, bool(batch_first))
    return _scan_fwd(gates, h0, active, bool(batch_first))


def _step_fwd(gates, h_mem, ids, mem_write, keep):
    gd = gates.detach()
    gd = gd if gd.stride(1) == 1 else gd.contiguous()
    m, hd = gd.shape[0], gd.shape[1] // 2
    dev = gd.device
    h = torch.empty(m, hd, dtype=torch.float32, device=dev)
    before = torch.empty(m, hd, dtype=torch.float32, device=dev) if keep else None
    lib = nv.lib()
    nodes = h_mem.shape[0]
    ws_bytes = lib.spmi_gated_step_workspace_bytes(m, nodes) if mem_write and ids is not None else 0
    with torch.cuda.device(dev):
        ws = _workspace(ws_bytes, dev)
        nv.check(lib.spmi_gated_step(nv.ptr(gd), _DTYPE_CODES[gd.dtype], gd.stride(0), nv.ptr(h_mem), nodes,
                                     nv.ptr(ids), m, hd, nv.ptr(h), nv.ptr(before), int(mem_write), nv.ptr(ws),
                                     ws_bytes, nv.stream()), "spmi_gated_step")
    if mem_write:
        torch.autograd.graph.increment_version(h_mem)
    return h, before


class _GatedStep(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gates, h_mem, ids, mem_write):
        h, before = _step_fwd(gates, h_mem, ids, mem_write, True)
        ctx.save_for_backward(gates, before)
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        # the scan's backward over one step, with the rows' old states as its start
        gates, before = ctx.saved_tensors
        gd = gates.detach()
        gd = gd if gd.stride(1) == 1 else gd.contiguous()
        dgates = torch.empty(gd.shape, dtype=gd.dtype, device=gd.device)
        _scan_call("bwd", gd[None], before, None, False, before[None], None, None, _units_last(g), dgates[None])
        return dgates, None, None, None


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
    _rows_dtype(gates, "gated_step: gates")
    if gates.dim() != 2 or gates.shape[1] < 2 or gates.shape[1] % 2:
        raise nv.SpmiError(f"gated_step: gates must be [M, 2H], got {tuple(gates.shape)}")
    m, hd = gates.shape[0], gates.shape[1] // 2
    if h_mem.dim() != 2 or h_mem.shape[1] != hd or h_mem.dtype != torch.float32 or not h_mem.is_contiguous():
        raise nv.SpmiError(f"gated_step: the node memory must be contiguous float32 [nodes, {hd}], got "
                           f"{h_mem.dtype} {tuple(h_mem.shape)}")
    if h_mem.requires_grad and torch.is_grad_enabled():
        raise nv.SpmiError("gated_step: the node memory is a state and takes no gradient")
    if ids is None:
        if m > h_mem.shape[0]:
            raise nv.SpmiError("gated_step: more rows than nodes in the memory")
    elif ids.dtype != torch.int64 or ids.shape != (m,):
        raise nv.SpmiError(f"gated_step: ids must be int64 [{m}], got {ids.dtype} {tuple(ids.shape)}")
    else:
        ids = ids.contiguous()
    _same_device(gates, h_mem, ids)
    if _tracked(gates):
        return _GatedStep.apply(gates, h_mem, ids, bool(mem_write))
    return _step_fwd(gates, h_mem, ids, bool(mem_write), False)[0]


# --------------------------------------------------------------------------- 8-bit integers
INT8_MAX_INNER = 131072  # 127^2 times this still fits the 32-bit sums


def quantize_rows_int8(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows of x [..., K] (float32 or bfloat16) in 8-bit integers: `q` int8 of x's shape and `scale`
    float32 of its leading shape, x = q * scale to within half a scale.  With m the row's largest
    magnitude (at least 2^-120), scale = m / 127 and q = rint(x * (127 / m)), each operation rounded
    to float32.  A row with a value that is not finite gets q = 0 and scale = NaN.  Applied to a
    weight [N, K] this gives the arguments of `linear_int8`."""
    code = _rows_dtype(x, "quantize_rows_int8: x")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= INT8_MAX_INNER:
        raise nv.SpmiError(f"quantize_rows_int8: the last dimension of x must be 1 to {INT8_MAX_INNER}, got "
                           f"{tuple(x.shape)}")
    nv.require_cuda(x)
    xd = _rows_of(x.detach())
    m, k = xd.shape
    q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        nv.check(nv.lib().spmi_quantize_rows_i8(nv.ptr(xd), code, xd.stride(0), m, k, nv.ptr(q), k, nv.ptr(scale),
                                                nv.stream()), "spmi_quantize_rows_i8")
    return q, scale


def linear_int8(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                bias: Optional[torch.Tensor] = None, act: Optional[str] = None, slope: float = 0.01,
                out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """act(x @ (weight * weight_scale[:, None]).T + bias) with the products in 8-bit integers: the
    rows of x [..., K] (float32 or bfloat16) are brought to whole numbers with a scale each
    (`quantize_rows_int8`), the sums over K are exact, scales, bias and activation (None, "relu" or
    "leaky_relu" with `slope`) follow in float32, and the result [..., N] is rounded once to
    `out_dtype` (default: x's type).  weight: int8 [N, K], weight_scale: float32 [N]; K up to 131072.
    For serving: there is no backward pass, and a call that would need one is refused."""
    code = _rows_dtype(x, "linear_int8: x")
    if weight.dim() != 2 or weight.dtype != torch.int8:
        raise nv.SpmiError(f"linear_int8: weight must be int8 [N, K], got {weight.dtype} {tuple(weight.shape)}")
    n, k = weight.shape
    if x.dim() < 1 or x.shape[-1] != k or not 1 <= k <= INT8_MAX_INNER:
        raise nv.SpmiError(f"linear_int8: x {tuple(x.shape)} does not fit a weight {tuple(weight.shape)}")
    if weight_scale.shape != (n,) or weight_scale.dtype != torch.float32:
        raise nv.SpmiError(f"linear_int8: weight_scale must be float32 [{n}]")
    if bias is not None:
        if bias.shape != (n,):
            raise nv.SpmiError(f"linear_int8: bias must have shape ({n},), got {tuple(bias.shape)}")
        _rows_dtype(bias, "linear_int8: bias")
    if act not in _ACT_CODES:
        raise nv.SpmiError(f"linear_int8: unknown activation {act!r}")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in _DTYPE_CODES:
        raise nv.SpmiError("linear_int8: out_dtype must be float32 or bfloat16")
    if _tracked(x, weight_scale, bias):
        raise nv.SpmiError("linear_int8 has no backward pass: call it under torch.no_grad()")
    _same_device(x, weight, weight_scale, bias)
    bias = _float_vector(bias)
    xd = _rows_of(x.detach())
    w = weight if weight.stride(1) == 1 or k == 1 else weight.contiguous()
    s = weight_scale.detach().contiguous()
    m = xd.shape[0]
    lib = nv.lib()
    out = torch.empty(*x.shape[:-1], n, dtype=out_dtype, device=x.device)
    ws_bytes = lib.spmi_linear_i8_workspace_bytes(m, k, n)
    with torch.cuda.device(x.device):
        ws = _workspace(ws_bytes, x.device)
        nv.check(lib.spmi_linear_i8(nv.ptr(xd), code, xd.stride(0), m, k, nv.ptr(w), w.stride(0), nv.ptr(s), n,
                                    nv.ptr(bias), _ACT_CODES[act], float(slope), nv.ptr(out),
                                    _DTYPE_CODES[out_dtype], n, nv.ptr(ws), ws_bytes, nv.stream()), "spmi_linear_i8")
    return out
