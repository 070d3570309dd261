"""The norm of a policy's features: layer norm, alone or with the sum of a residual stream.

    y = (s - mean(s)) / sqrt(variance(s) + eps) * weight + bias

over the last dimension, where s is x or, with a residual, x + residual rounded to its type: a
block's output and the stream it is added to, in one pass. Runs on torch's current stream and has
gradients for every input; a trace records it as a call.

    x, residual    [..., dim]   float32, float16 or bfloat16, any strides
    weight, bias   [dim]        x's type or float32; None: 1 and 0

dim is 1 to 16384; a row of x may begin anywhere (a slice of wider rows needs no copy), its features
are contiguous or x is copied first. Each head's output [..., heads, dim] is normalised by the same
call. Sums and statistics are fp32, in the gradients of the weight and the bias too; results and
gradients are rounded once, and are the same from run to run. The sum of a row's values and of the
squares of their distances from its mean have to stay in fp32's range (values below 1e34 and distances below 1e17 do, whatever dim is); a NaN or an infinity spoils its own row, and of the gradients
its row's and those of the weight and the bias.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple, Union

import torch

from . import _lib as L
from ._torch import DTYPES, S3, dense_like, differentiated, fail, on, pointer, row, space, stream

_U3 = C.c_uint32 * 3
_NONE = S3()


def _strides(x: Optional[torch.Tensor]):
    if x is None:
        return _NONE
    s = x.stride()
    return S3(s[0], s[1], s[2]) if len(s) == 4 else S3(0, s[0], s[1]) if len(s) == 3 else S3(0, 0, s[0]) if len(s) == 2 else _NONE


def _inputs(x, residual, weight, bias, eps) -> L.ZenoAmdNormInputs:
    shape, dtype = x.shape, DTYPES[x.dtype]
    w = bias if weight is None else weight
    return L.ZenoAmdNormInputs(
        dtype, dtype if w is None else DTYPES[w.dtype], _U3(*(1,) * (4 - len(shape)), *shape[:-1]), shape[-1], eps, x.data_ptr(), pointer(residual),
        pointer(weight), pointer(bias), _strides(x), _strides(residual))


def _forward(x, weight, bias, residual, eps):
    with on(x):
        y = dense_like(x)
        total = None if residual is None else dense_like(x)
        rc = L.load().zeno_amd_norm_forward(_inputs(x, residual, weight, bias, eps), y.data_ptr(), _strides(y), pointer(total), _strides(total), stream(x))
        if rc:
            fail(rc, "layer_norm")
    return y, total


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps):
        y, total = _forward(x, weight, bias, residual, eps)
        ctx.save_for_backward(x if total is None else total, weight, bias)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        return y if total is None else (y, total)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_y, d_sum=None):
        if d_y is None and d_sum is None:
            return (None,) * 5
        s, weight, bias = ctx.saved_tensors
        want_x, want_weight, want_bias, want_residual = ctx.needs_input_grad[:4]
        with on(s):
            lib = L.load()
            d_y = torch.zeros_like(s) if d_y is None else row(d_y)
            d_sum = None if d_sum is None else row(d_sum)
            a = _inputs(s, None, weight, bias, ctx.eps)
            d_x = dense_like(s) if want_x or want_residual else None
            d_weight = torch.empty_like(weight) if want_weight else None
            d_bias = torch.empty_like(bias) if want_bias else None
            parts = space(lib.zeno_amd_norm_workspace_bytes(a), s) if want_weight or want_bias else None
            grads = L.ZenoAmdNormGradients(d_y.data_ptr(), pointer(d_sum), pointer(d_x), pointer(d_weight), pointer(d_bias),
                                           _strides(d_y), _strides(d_sum), _strides(d_x))
            rc = lib.zeno_amd_norm_backward(a, grads, pointer(parts), stream(s))
            if rc:
                fail(rc, "layer_norm's gradients")
        return d_x if want_x else None, d_weight, d_bias, d_x if want_residual else None, None


def _check(x, weight, bias, residual) -> None:
    dtype, shape, device = x.dtype, x.shape, x.device
    if dtype not in DTYPES:
        raise TypeError(f"x must be float32, float16 or bfloat16, not {dtype}")
    if not shape or 0 in shape:
        raise ValueError(f"x must hold rows of features, not {tuple(shape)}")
    if not x.is_cuda:
        raise ValueError("x must be on the GPU (there is no CPU fallback)")
    for name, w in (("weight", weight), ("bias", bias)):
        if w is None:
            continue
        if w.shape != shape[-1:]:
            raise ValueError(f"{name} must have the shape {tuple(shape[-1:])}, not {tuple(w.shape)}")
        if w.dtype is not dtype and w.dtype is not torch.float32:
            raise TypeError(f"{name} must be float32 or have x's type {dtype}, not {w.dtype}")
        if w.device != device:
            raise ValueError("the operands must be on one device")
    if weight is not None and bias is not None and weight.dtype is not bias.dtype:
        raise TypeError(f"weight and bias must have one type, not {weight.dtype} and {bias.dtype}")
    if residual is not None:
        if residual.shape != shape or residual.dtype is not dtype:
            raise ValueError(f"residual must be like x: {tuple(shape)}, {dtype}, not {tuple(residual.shape)}, {residual.dtype}")
        if residual.device != device:
            raise ValueError("the operands must be on one device")


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
               residual: Optional[torch.Tensor] = None, eps: float = 1e-5) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """The norm of x's rows; with a residual, the norm of the rows of x + residual and those sums, to
    which the gradient of either flows on. Differentiable in x, residual, weight and bias."""
    _check(x, weight, bias, residual)
    shape = x.shape
    if len(shape) > 4:  # rows lie along three dimensions at most
        x = x.flatten(0, len(shape) - 4)
        residual = None if residual is None else residual.flatten(0, len(shape) - 4)
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    x, residual = row(x), None if residual is None else row(residual)
    if differentiated(x, weight, bias, residual):
        out = _LayerNorm.apply(x, weight, bias, residual, float(eps))
    else:
        y, total = _forward(x, weight, bias, residual, float(eps))
        out = y if total is None else (y, total)
    if len(shape) > 4:
        return out.view(shape) if residual is None else tuple(y.view(shape) for y in out)
    return out
