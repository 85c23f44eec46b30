"""What layer norm, the gated linear recurrence and the 8-bit projection refuse, checked without a GPU:
the arguments of spiral_amd.ops, and the sizes and pointers of the C entry points (which are looked
at before any HIP call)."""
import pytest
import torch

from spiral_amd import _native as nv
from spiral_amd import ops

F = torch.zeros


@pytest.mark.parametrize("call", [
    lambda: ops.layer_norm(F(3, 4, dtype=torch.float64)),
    lambda: ops.layer_norm(F(3, 4, dtype=torch.float16)),
    lambda: ops.layer_norm(F(())),
    lambda: ops.layer_norm(F(3, 0)),
    lambda: ops.layer_norm(F(1, 16385)),
    lambda: ops.layer_norm(F(3, 4), F(3)),
    lambda: ops.layer_norm(F(3, 4), F(1, 4)),
    lambda: ops.layer_norm(F(3, 4), None, F(5)),
    lambda: ops.layer_norm(F(3, 4), F(4, dtype=torch.float64)),
    lambda: ops.layer_norm(F(3, 4), eps=-1.0),
    lambda: ops.layer_norm(F(3, 4), eps=float("nan")),
    lambda: ops.gated_scan(F(3, 8)),
    lambda: ops.gated_scan(F(3, 2, 7)),
    lambda: ops.gated_scan(F(3, 2, 0)),
    lambda: ops.gated_scan(F(3, 2, 8, dtype=torch.float16)),
    lambda: ops.gated_scan(F(3, 2, 8), F(3, 4)),
    lambda: ops.gated_scan(F(3, 2, 8), F(2, 8)),
    lambda: ops.gated_scan(F(3, 2, 8), F(2, 4, dtype=torch.bfloat16)),
    lambda: ops.gated_scan(F(3, 2, 8), F(2, 4), batch_first=True),
    lambda: ops.gated_scan(F(3, 2, 8), None, F(3, 2)),
    lambda: ops.gated_scan(F(3, 2, 8), None, F(2, 3, dtype=torch.bool)),
    lambda: ops.gated_step(F(3, 2, 8), F(5, 4)),
    lambda: ops.gated_step(F(3, 7), F(5, 4)),
    lambda: ops.gated_step(F(3, 8), F(5, 8)),
    lambda: ops.gated_step(F(3, 8), F(4, 5).t()),
    lambda: ops.gated_step(F(3, 8), F(5, 4, dtype=torch.bfloat16)),
    lambda: ops.gated_step(F(6, 8), F(5, 4)),
    lambda: ops.gated_step(F(3, 8), F(5, 4), F(3, dtype=torch.int32)),
    lambda: ops.gated_step(F(3, 8), F(5, 4), F(2, dtype=torch.int64)),
    lambda: ops.gated_step(F(3, 8), F(5, 4).requires_grad_()),
    lambda: ops.quantize_rows_int8(F(3, 4, dtype=torch.int32)),
    lambda: ops.quantize_rows_int8(F(3, 0)),
    lambda: ops.quantize_rows_int8(F(1, 131073)),
    lambda: ops.linear_int8(F(3, 4), F(5, 4), F(5)),
    lambda: ops.linear_int8(F(3, 4), F(5, 3, dtype=torch.int8), F(5)),
    lambda: ops.linear_int8(F(3, 4), F(5, 4, dtype=torch.int8), F(4)),
    lambda: ops.linear_int8(F(3, 4), F(5, 4, dtype=torch.int8), F(5, dtype=torch.bfloat16)),
    lambda: ops.linear_int8(F(3, 4), F(5, 4, dtype=torch.int8), F(5), F(4)),
    lambda: ops.linear_int8(F(3, 4), F(5, 4, dtype=torch.int8), F(5), act="gelu"),
    lambda: ops.linear_int8(F(3, 4), F(5, 4, dtype=torch.int8), F(5), out_dtype=torch.float16),
    lambda: ops.linear_int8(F(3, 4).requires_grad_(), F(5, 4, dtype=torch.int8), F(5)),
    lambda: ops.linear_int8(F(3, 4), F(5, 4, dtype=torch.int8), F(5), F(5).requires_grad_()),
])
def test_refused_arguments(call):
    with pytest.raises(nv.SpmiError):
        call()


@pytest.mark.parametrize("call", [
    lambda: ops.layer_norm(F(3, 4), F(4), F(4)),
    lambda: ops.gated_scan(F(3, 2, 8), F(2, 4), F(3, 2, dtype=torch.bool)),
    lambda: ops.gated_step(F(3, 8), F(5, 4), F(3, dtype=torch.int64)),
    lambda: ops.quantize_rows_int8(F(3, 4)),
    lambda: ops.linear_int8(F(3, 4), F(5, 4, dtype=torch.int8), F(5), F(5)),
])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(nv.SpmiError, match="GPU"):
        call()


def test_c_entry_points_refuse_bad_sizes_and_pointers():
    lib = nv.lib()
    P = 64  # stands for a pointer; every call below returns before it is used
    assert lib.spmi_layer_norm_max_width() == ops.LAYER_NORM_MAX_WIDTH
    norm = lib.spmi_layer_norm_fwd
    assert norm(P, 7, 4, 3, 4, P, P, 1e-5, P, 4, None, None) == -1
    assert norm(P, 0, 4, -1, 4, P, P, 1e-5, P, 4, None, None) == -1
    assert norm(P, 0, 4, 3, 0, P, P, 1e-5, P, 4, None, None) == -1
    assert norm(P, 0, 4, 3, 16385, P, P, 1e-5, P, 16385, None, None) == -5
    assert norm(None, 0, 4, 3, 4, P, P, 1e-5, P, 4, None, None) == -1
    assert norm(P, 0, 4, 3, 4, P, P, 1e-5, P, 3, None, None) == -1
    assert norm(P, 0, -4, 3, 4, P, P, 1e-5, P, 4, None, None) == -1
    assert norm(None, 0, 4, 0, 4, None, None, 1e-5, None, 4, None, None) == 0
    back = lib.spmi_layer_norm_bwd
    need = lib.spmi_layer_norm_bwd_workspace_bytes(100, 64)
    assert need > 0 and lib.spmi_layer_norm_bwd_workspace_bytes(0, 64) == 0
    assert back(P, P, 0, 64, 64, 100, 64, P, P, P, 64, P, P, P, need - 1, None) == -3
    assert back(P, P, 0, 64, 64, 100, 64, P, P, P, 64, P, None, None, 0, None) == -3
    assert back(P, P, 0, 64, 64, 100, 64, P, None, P, 64, None, None, None, 0, None) == -1
    assert back(P, P, 0, 64, 64, 100, 64, P, P, P, 63, None, None, None, 0, None) == -1

    scan = lib.spmi_gated_scan_fwd
    assert scan(P, 9, 8, 8, None, 0, None, 0, 0, 1, 1, 4, P, 4, 4, P, None, 0, None) == -1
    assert scan(P, 0, 8, 8, None, 0, None, 0, 0, -1, 1, 4, P, 4, 4, P, None, 0, None) == -1
    assert scan(P, 0, 8, 8, None, 0, None, 0, 0, 1, 1, 0, P, 4, 4, P, None, 0, None) == -1
    assert scan(P, 0, 8, 8, None, 0, None, 0, 0, 1, 1 << 40, 4, P, 4, 4, P, None, 0, None) == -5
    assert scan(P, 0, 8, 8, None, 0, None, 0, 0, 1, 1, 4, P, 4, 4, None, None, 0, None) == -1
    assert scan(None, 0, 8, 8, None, 0, None, 0, 0, 5, 0, 4, None, 4, 4, None, None, 0, None) == 0
    need = lib.spmi_gated_scan_fwd_workspace_bytes(65536, 1, 128)
    assert need > 0 and lib.spmi_gated_scan_fwd_workspace_bytes(8, 1, 128) == 0
    assert scan(P, 0, 256, 256, None, 0, None, 0, 0, 65536, 1, 128, P, 128, 128, P, P, need - 1, None) == -3
    assert scan(P, 0, 256, 256, None, 0, None, 0, 0, 65536, 1, 128, P, 128, 128, P, P + 4, need, None) == -1
    step = lib.spmi_gated_step
    assert step(P, 0, 8, P, 5, None, 6, 4, P, None, 1, None, 0, None) == -1
    assert step(P, 0, 8, P, -5, None, 3, 4, P, None, 1, None, 0, None) == -1
    assert step(P, 0, 8, None, 5, None, 3, 4, P, None, 1, None, 0, None) == -1
    need = lib.spmi_gated_step_workspace_bytes(5000, 9000)
    assert need >= 9000 * 4
    assert step(P, 0, 8, P, 9000, P, 5000, 4, P, None, 1, P, need - 1, None) == -3

    lin = lib.spmi_linear_i8
    need = lib.spmi_linear_i8_workspace_bytes(100, 70, 30)
    assert lin(P, 0, 70, 100, 131073, P, 131073, P, 30, None, 0, 0.0, P, 0, 30, P, 1 << 40, None) == -5
    assert lin(P, 0, 70, 100, 70, P, 70, P, 30, None, 5, 0.0, P, 0, 30, P, need, None) == -1
    assert lin(P, 0, 70, 100, 70, P, 70, P, 30, None, 0, 0.0, P, 3, 30, P, need, None) == -1
    assert lin(P, 0, 70, 100, 70, P, 70, P, 30, None, 0, 0.0, P, 0, 29, P, need, None) == -1
    assert lin(P, 0, 70, 100, 70, None, 70, P, 30, None, 0, 0.0, P, 0, 30, P, need, None) == -1
    assert lin(None, 0, 70, 0, 70, None, 70, None, 30, None, 0, 0.0, None, 0, 30, None, 0, None) == 0
    assert lib.spmi_quantize_rows_i8(P, 0, 70, 3, 70, P, 69, P, None) == -1
    assert lib.spmi_quantize_rows_i8(None, 0, 70, 3, 70, P, 70, P, None) == -1
