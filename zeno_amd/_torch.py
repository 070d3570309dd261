"""What the operators on torch tensors share: the library's errors, streams, devices and rows."""
from __future__ import annotations

import contextlib
import ctypes as C
from typing import Optional

import torch

from . import _lib as L

L.one_runtime()

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
S3 = C.c_int64 * 3
written = torch.autograd.graph.increment_version
_HERE = contextlib.nullcontext()


def fail(rc: int, what: str) -> None:
    if rc == -6:
        raise ValueError(L.last_error())
    raise RuntimeError(f"{what} failed: {rc}: {L.last_error()}")


def row(x: torch.Tensor) -> torch.Tensor:
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def dense_like(x: torch.Tensor) -> torch.Tensor:
    """Memory in x's order of dimensions, each value at a place of its own, rows contiguous."""
    y = torch.empty_like(x)
    return y if y.stride(-1) == 1 or x.shape[-1] == 1 else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def space(n: int, x: torch.Tensor) -> Optional[torch.Tensor]:
    return torch.empty(n, dtype=torch.uint8, device=x.device) if n else None


def stream(x: torch.Tensor) -> int:
    """torch.cuda.current_stream(x.device).cuda_stream, without an object around it (2 us less of a step's 20)."""
    return torch._C._cuda_getCurrentRawStream(x.device.index)


def on(x: torch.Tensor):
    """The context in which x's device is the current one, as the library's calls need it."""
    return _HERE if torch.cuda.current_device() == x.device.index else torch.cuda.device(x.device)


def differentiated(*operands: Optional[torch.Tensor]) -> bool:
    """Whether a call has to go through autograd: for gradients, or to be refused where tangents are carried forward."""
    return (torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in operands)) or torch.autograd.forward_ad._current_level >= 0


def pointer(x: Optional[torch.Tensor]) -> Optional[int]:
    return None if x is None else x.data_ptr()
