"""Refusals of the fused block seam (no GPU: the argument checks come before any device call)."""
import ctypes

import pytest
import torch

from trinity_lowering import kernels as k


def arguments(**changes):
    args = k.RmsnormResidualArgs()
    base = 1 << 20
    args.x, args.residual, args.residual_out, args.out = base, 2 * base, 3 * base, 4 * base
    args.rows, args.cols = 4, 64
    args.ld_x = args.ld_residual = args.ld_residual_out = args.ld_out = 64
    args.x_dtype = args.residual_dtype = k.DT_BF16
    for name, value in changes.items():
        setattr(args, name, value)
    return args


@pytest.mark.parametrize("changes,code,text", [
    ({"x": None}, -1, "null"), ({"residual": None}, -1, "null"), ({"out": None}, -1, "null"),
    ({"residual_out": None}, -1, "null"), ({"rows": 0}, -1, "empty"), ({"cols": 0}, -1, "empty"),
    ({"rows": -3}, -1, "empty"), ({"rows": 1 << 31}, -2, "rows"),
    ({"cols": 16385, "ld_x": 16385, "ld_residual": 16385, "ld_residual_out": 16385, "ld_out": 16385}, -2, "16385"),
    ({"ld_x": 63}, -1, "leading"), ({"ld_out": 0}, -1, "leading"), ({"x_dtype": 7}, -1, "dtype"),
    ({"residual_dtype": -1}, -1, "dtype"), ({"x": (1 << 20) + 1}, -1, "aligned"),
    ({"residual": (1 << 21) + 2, "residual_dtype": 1}, -1, "aligned"),
    ({"gate": 5 << 20, "gate_row_stride": 8, "gate_col_stride": 1}, -1, "gate"),
    ({"gate": 5 << 20, "gate_row_stride": 64, "gate_col_stride": 2}, -1, "gate"),
    ({"out": 3 << 20}, -1, "share"),
    ({"residual_out": 2 << 20, "ld_residual_out": 128}, -1, "overlaps"),
    ({"out": 1 << 20, "x_dtype": 1}, -1, "overlaps"),
    ({"out": 2 << 20, "residual_dtype": 1}, -1, "overlaps"),
])
def test_entry_point_refuses(changes, code, text):
    lib = k.library()
    assert lib.trinity_sm100_rmsnorm_residual(ctypes.byref(arguments(**changes)), None) == code
    assert text in lib.trinity_sm100_last_error().decode()


def test_null_argument_block():
    assert k.library().trinity_sm100_rmsnorm_residual(None, None) == -1


def test_binding_refuses_host_tensors():
    x = torch.zeros(2, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        k.rmsnorm_residual(x, x)
