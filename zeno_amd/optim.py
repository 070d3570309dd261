"""The update of a policy's matrices: orthogonalisation by Newton-Schulz products.

A momentum matrix G is replaced by a nearly orthogonal one, every singular value near 1, so that
a step moves all directions of the matrix alike:

    X = G / (|G| + eps);   steps times:   A = X X^T,  X <- a X + (b A + c A A) X

(on G^T where G has more rows than columns). With the usual coefficients and five steps the
singular values end between about 0.7 and 1.2. It is not differentiable: it makes an update.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import _lib as L
from ._torch import on, refuse_graph, refuse_trace

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_S3 = C.c_int64 * 3


@torch.no_grad()
def orthogonalize(update: torch.Tensor, steps: int = 5, coefficients: Tuple[float, float, float] = (3.4445, -4.7750, 2.0315),
                  eps: float = 1e-7, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """`update` [..., rows, cols]: one matrix or several of one shape, float32, float16 or
    bfloat16, on the GPU, of any strides. Returns matrices of its shape and type (`out` if given;
    out=update works in place). Results of every type are as exact as fp32 products give them,
    rounded once. Runs on torch's current stream."""
    refuse_trace("orthogonalize")
    refuse_graph()
    if update.dtype not in _DTYPES:
        raise TypeError(f"update must be float32, float16 or bfloat16, not {update.dtype}")
    if update.dim() < 2 or update.numel() == 0:
        raise ValueError(f"update must hold matrices, not {tuple(update.shape)}")
    if not update.is_cuda:
        raise ValueError("update must be on the GPU (there is no CPU fallback)")
    if not 1 <= steps <= 100:  # before it is cut to 32 bits
        raise ValueError(f"steps must be 1 to 100, not {steps}")
    if len(coefficients) != 3:
        raise ValueError("coefficients are three numbers")
    if out is None:
        out = torch.empty(update.shape, dtype=update.dtype, device=update.device)
    elif out.shape != update.shape or out.dtype != update.dtype or out.device != update.device:
        raise ValueError(f"out must be like update: {tuple(update.shape)}, {update.dtype}, on {update.device}")
    x = update.reshape(-1, *update.shape[-2:])
    y = out.view(-1, *update.shape[-2:])
    with on(update):
        lib = L.load()
        a = L.ZenoAmdOrthogonalize(_DTYPES[x.dtype], *x.shape, steps, *coefficients, eps, x.data_ptr(), _S3(*x.stride()),
                                   y.data_ptr(), _S3(*y.stride()))
        space = torch.empty(lib.zeno_amd_orthogonalize_workspace_bytes(a), dtype=torch.uint8, device=x.device)
        rc = lib.zeno_amd_orthogonalize(a, space.data_ptr(), torch.cuda.current_stream(x.device).cuda_stream)
    if rc == -6:
        raise ValueError(L.last_error())
    if rc:
        raise RuntimeError(f"orthogonalize failed: {rc}: {L.last_error()}")
    torch.autograd.graph.increment_version(out)  # autograd refuses a backward pass that needs what was here
    return out
