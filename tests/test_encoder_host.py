"""Host checks of the token-encoder operators that need no GPU: refusals come before
any launch, at the C entry points and in Python."""
import ctypes as C

import pytest
import torch


def test_entry_points_reject_before_launching(fms):
    L = fms.load_library()
    one = C.c_void_p(16)
    # gated_ffn: float32 features, unknown activation, negative size, missing pointers, no workspace
    assert L.fms_gated_ffn_fwd(0, one, one, one, 4, 8, 8, 0, one, None, 0, None) == -2
    assert L.fms_gated_ffn_fwd(1, one, one, one, 4, 8, 8, 4, one, None, 0, None) == -1
    assert L.fms_gated_ffn_fwd(1, one, one, one, -1, 8, 8, 0, one, None, 0, None) == -1
    assert L.fms_gated_ffn_fwd(1, None, one, one, 4, 8, 8, 0, one, None, 0, None) == -1
    assert L.fms_gated_ffn_fwd(1, None, None, None, 0, 8, 8, 0, None, None, 0, None) == 0
    assert L.fms_gated_ffn_bwd(1, one, one, one, one, 4, 8, 8, 0, one, one, one, None, 0, None) == -4
    assert L.fms_gated_ffn_workspace_size(100, 64, 32, 1) >= 100 * 32 * 2 * 2
    # norm_residual: types, kind, groups that do not divide the rows, an empty row
    fwd = lambda dt, vt, kind, groups, rows, dim: L.fms_norm_residual_fwd(  # noqa: E731
        dt, vt, kind, one, one, one, None, one, None, None, groups, rows, dim, 1e-6, 1.0, one, one, None, None)
    assert fwd(3, 3, 0, 1, 4, 8) == -2 and fwd(1, 2, 0, 1, 4, 8) == -2
    assert fwd(1, 1, 2, 1, 4, 8) == -1 and fwd(1, 1, 0, 3, 4, 8) == -1 and fwd(1, 1, 0, 1, 4, 0) == -1
    assert fwd(1, 1, 0, 1, 0, 8) == 0
    # int8_linear
    assert L.fms_int8_linear_fwd(3, one, None, one, one, None, 1, 8, 8, 0, one, None, 0, None) == -2
    assert L.fms_int8_linear_fwd(4, one, None, one, one, None, 1, 8, 8, 0, one, None, 0, None) == -1
    assert L.fms_int8_linear_fwd(0, one, None, one, one, None, 1, 0, 8, 0, one, None, 0, None) == -1
    assert L.fms_int8_linear_fwd(0, one, None, one, one, None, 99, 8, 8, 0, one, None, 0, None) == -4
    # adamw: width, step, betas, a tensor without a pointer, none at all
    assert L.fms_adamw_step(16, 0, None, 1, 1e-3, 0.9, 0.99, 1e-8, 0.0, 0, None, None) == -2
    assert L.fms_adamw_step(32, 0, None, 0, 1e-3, 0.9, 0.99, 1e-8, 0.0, 0, None, None) == -1
    assert L.fms_adamw_step(32, 0, None, 1, 1e-3, 1.0, 0.99, 1e-8, 0.0, 0, None, None) == -1
    assert L.fms_adamw_step(32, 1, None, 1, 1e-3, 0.9, 0.99, 1e-8, 0.0, 0, None, None) == -1
    empty = (C.c_int64 * 10)(0, 0, 0, 0, 0, 0, 0, 5, 0, 0)  # one tensor of five values, no pointers
    assert L.fms_adamw_step(32, 1, empty, 1, 1e-3, 0.9, 0.99, 1e-8, 0.0, 0, None, None) == -1
    assert L.fms_adamw_step(32, 0, None, 1, 1e-3, 0.9, 0.99, 1e-8, 0.0, 0, None, None) == 0


def test_host_tensors_are_refused(fms):
    h = torch.zeros(4, 8, dtype=torch.bfloat16)
    w = torch.zeros(6, 8, dtype=torch.bfloat16)
    with pytest.raises(fms.ArgumentError):
        fms.gated_ffn(h, w, w)
    with pytest.raises(fms.ArgumentError):
        fms.norm_residual(h, h, h[0], h[0])
    with pytest.raises(fms.ArgumentError):
        fms.int8_linear(h, fms.Int8Index(torch.zeros(6, 8, dtype=torch.int8), torch.zeros(6)))
    z = torch.zeros(8)
    with pytest.raises(fms.ArgumentError):
        fms.adamw_step([z], [z], [z], [z], step=1)


def test_shapes_are_checked_first(fms):
    h = torch.zeros(4, 8, dtype=torch.bfloat16)
    with pytest.raises(fms.DimensionMismatch):
        fms.gated_ffn(h, torch.zeros(6, 7, dtype=torch.bfloat16), torch.zeros(6, 7, dtype=torch.bfloat16))
    with pytest.raises(fms.DimensionMismatch):
        fms.norm_residual(h, h[:2], h[0], h[0])
    with pytest.raises(fms.DimensionMismatch):
        fms.int8_linear(h, fms.Int8Index(torch.zeros(6, 7, dtype=torch.int8), torch.zeros(6)))
    codes, scales = fms.moments8(torch.zeros(3, 100))
    assert codes.shape == (3, 100) and codes.dtype == torch.float8_e4m3fn and scales.shape == (2,)
