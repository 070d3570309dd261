"""What the operators on torch tensors share: the library's errors, streams, devices and rows."""
from __future__ import annotations

import contextlib
import ctypes as C
from typing import Optional

import torch
from torch.fx.experimental.proxy_tensor import get_proxy_mode

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


def refuse_graph() -> None:
    """Where make_fx records torch's operations: a graph of them has the memory that a call allocates and not the call. (It
    always sets a function mode, which is quicker to see.)"""
    if torch._C._len_torch_function_stack() and get_proxy_mode() is not None:
        raise RuntimeError("the library's calls are no torch operations and cannot be recorded into a graph of those")


def on(x: torch.Tensor):
    """The context in which x's device is the current one, as the library's calls need it."""
    refuse_graph()
    return _HERE if torch.cuda.current_device() == x.device.index else torch.cuda.device(x.device)


def differentiated(*operands: Optional[torch.Tensor]) -> bool:
    """Whether a call has to go through autograd: for gradients, to be refused where tangents are carried forward, or
    to be in a trace as a call, which without a function of autograd's would have the memory alone that it allocates."""
    return ((torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in operands)) or torch.autograd.forward_ad._current_level >= 0
            or torch._C._get_tracing_state() is not None)


def refuse_trace(what: str) -> None:
    """For calls that are no function of autograd's, of which a trace has nothing."""
    if torch._C._get_tracing_state() is not None:
        raise RuntimeError(f"{what} writes memory that a trace does not see: it cannot be traced")


def refuse_tangents(*operands: Optional[torch.Tensor]) -> None:
    """For calls that are no function of autograd's, which would refuse them."""
    forward = torch.autograd.forward_ad
    if forward._current_level >= 0 and any(x is not None and forward.unpack_dual(x).tangent is not None for x in operands):
        raise RuntimeError("an operand carries a tangent forward, of which a call without derivatives would make nothing")


def pointer(x: Optional[torch.Tensor]) -> Optional[int]:
    return None if x is None else x.data_ptr()
