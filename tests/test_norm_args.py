"""Layer norm's C entry points refuse what they cannot take before anything is enqueued (no GPU)."""
import ctypes as C

import pytest

from zeno_amd import _lib

MIB = 1 << 20
S3 = C.c_int64 * 3


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def rows(**change):
    """Twelve rows of 16 floats along three dimensions, every array in a MiB of its own."""
    a = dict(dtype=0, weight_dtype=0, rows=(2, 3, 2), dim=16, eps=1e-5, x=MIB, residual=None, weight=2 * MIB, bias=3 * MIB, x_stride=(96, 32, 16),
             residual_stride=(96, 32, 16))
    a = {**a, **change}
    a["rows"] = (C.c_uint32 * 3)(*a["rows"])
    a["x_stride"], a["residual_stride"] = S3(*a["x_stride"]), S3(*a["residual_stride"])
    return _lib.ZenoAmdNormInputs(**a)


def refused(rc, words):
    assert rc == -6 and words in _lib.last_error(), (rc, _lib.last_error())


@pytest.mark.parametrize("change, words", [
    ({"dtype": 3, "weight_dtype": 3}, "dtype"), ({"dtype": 2, "weight_dtype": 1}, "weight_dtype"), ({"weight_dtype": 1}, "weight_dtype"),
    ({"rows": (2, 0, 2)}, "no rows"), ({"dim": 0}, "dim"), ({"dim": 16385}, "dim"), ({"rows": (65536, 32768, 1)}, "too many rows"),
    ({"rows": (4294967295, 4294967295, 4294967295)}, "too many rows"), ({"eps": float("nan")}, "eps"), ({"eps": -1e-9}, "eps"), ({"eps": float("inf")}, "eps")])
def test_sizes_and_types(lib, change, words):
    a = rows(**change)
    refused(lib.zeno_amd_norm_forward(a, 4 * MIB, S3(96, 32, 16), None, None, None), words)
    g = _lib.ZenoAmdNormGradients(d_y=5 * MIB, d_x=6 * MIB, d_y_stride=S3(96, 32, 16), d_x_stride=S3(96, 32, 16))
    refused(lib.zeno_amd_norm_backward(a, g, None, None), words)
    assert lib.zeno_amd_norm_workspace_bytes(a) == 0


def test_nulls(lib):
    y = S3(96, 32, 16)
    refused(lib.zeno_amd_norm_forward(None, 4 * MIB, y, None, None, None), "null")
    refused(lib.zeno_amd_norm_forward(rows(x=None), 4 * MIB, y, None, None, None), "null")
    refused(lib.zeno_amd_norm_forward(rows(), None, y, None, None, None), "null")
    refused(lib.zeno_amd_norm_forward(rows(), 4 * MIB, None, None, None, None), "null")
    refused(lib.zeno_amd_norm_forward(rows(), 4 * MIB, y, 5 * MIB, y, None), "residual")
    refused(lib.zeno_amd_norm_forward(rows(residual=5 * MIB), 4 * MIB, y, None, None, None), "residual")
    refused(lib.zeno_amd_norm_forward(rows(residual=5 * MIB), 4 * MIB, y, 6 * MIB, None, None), "residual")
    refused(lib.zeno_amd_norm_backward(rows(), None, None, None), "null")
    g = dict(d_y=5 * MIB, d_y_stride=y, d_x_stride=y)
    refused(lib.zeno_amd_norm_backward(rows(), _lib.ZenoAmdNormGradients(**g), None, None), "no gradient")
    refused(lib.zeno_amd_norm_backward(rows(), _lib.ZenoAmdNormGradients(d_x=6 * MIB), None, None), "null")
    refused(lib.zeno_amd_norm_backward(rows(), _lib.ZenoAmdNormGradients(d_weight=6 * MIB, **g), None, None), "workspace")
    refused(lib.zeno_amd_norm_backward(rows(), _lib.ZenoAmdNormGradients(d_bias=6 * MIB, **g), 7 * MIB + 4, None), "workspace")
    assert lib.zeno_amd_norm_workspace_bytes(None) == 0


@pytest.mark.parametrize("y, stride, words", [
    (MIB, (96, 32, 16), "overlaps an input"), (MIB + 700, (96, 32, 16), "overlaps an input"), (2 * MIB - 256, (96, 32, 16), "overlaps an input"),
    (3 * MIB + 63, (96, 32, 16), "overlaps an input"), (4 * MIB, (0, 32, 16), "overlaps itself"), (4 * MIB, (96, 32, 15), "overlaps itself"),
    (4 * MIB, (64, 32, 16), "overlaps itself"), (5 * MIB + 100, (96, 32, 16), "overlaps an input"), (6 * MIB - 4, (96, 32, 16), "outputs overlap")])
def test_outputs_that_overlap(lib, y, stride, words):
    a = rows(residual=5 * MIB)
    refused(lib.zeno_amd_norm_forward(a, y, S3(*stride), 6 * MIB, S3(96, 32, 16), None), words)


def test_gradients_that_overlap(lib):
    s = S3(96, 32, 16)
    fine = dict(d_y=5 * MIB, d_sum=6 * MIB, d_x=7 * MIB, d_weight=8 * MIB, d_bias=9 * MIB, d_y_stride=s, d_sum_stride=s, d_x_stride=s)
    for change, words in ((dict(d_x=MIB), "an input"), (dict(d_x=5 * MIB + 4), "an input"), (dict(d_x=6 * MIB), "an input"), (dict(d_weight=2 * MIB), "an input"),
                          (dict(d_bias=8 * MIB + 60), "outputs overlap"), (dict(d_weight=7 * MIB + 700), "outputs overlap"), (dict(d_x_stride=S3(96, 32, 0)), "itself")):
        refused(lib.zeno_amd_norm_backward(rows(), _lib.ZenoAmdNormGradients(**{**fine, **change}), 10 * MIB, None), words)


def test_workspaces(lib):
    """Two sums of every feature for each workgroup of at most 1024 of four waves."""
    assert lib.zeno_amd_norm_workspace_bytes(rows()) == 2 * 16 * 4  # twelve rows: one workgroup
    assert lib.zeno_amd_norm_workspace_bytes(rows(rows=(1, 1, 1 << 20), dim=1000)) == 1024 * 2 * 1000 * 4
    assert lib.zeno_amd_norm_workspace_bytes(rows(rows=(1, 1, 1 << 20), dim=16384)) == 256 * 2 * 16384 * 4
