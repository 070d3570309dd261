"""The memory layer of policies that act on partial observations: the gated delta rule.

Each environment (or recorded sequence) and head keeps a state S [key_dim, value_dim]. A token
brings a query, a key, a value, the log of a decay and a strength, and

    S <- exp(g) S                       (S <- 0 where an episode begins)
    S <- S + k (beta (v - S^T k))^T
    o  = scale S^T q

``gated_delta_step`` advances every environment's state by one token in place, beside a step of
the simulation; ``gated_delta`` runs whole sequences (rollouts, recorded episodes) and has
gradients for every input. Both take torch tensors on the GPU and run on torch's current stream.

Arguments, for B sequences (environments) of T tokens, Hk key heads and Hv value heads (a
multiple of Hk; value head h reads key head h // (Hv // Hk)):

    q, k       [B, T, Hk, key_dim]    float32, float16 or bfloat16
    v          [B, T, Hv, value_dim]  the same type
    g, beta    [B, T, Hv]             float32
    reset      [B, T]                 bool or uint8, or None: this token begins an episode
    state      [B, Hv, key_dim, value_dim] float32, or None for zeros

without T for a step. Dimensions are 1 to 128. Any strides will do where the last dimension of
q, k and v is contiguous, so views of one projection and time-major rollouts
(``x.transpose(0, 1)``) need no copy. scale defaults to key_dim ** -0.5; with ``normalize``,
queries and keys are divided by sqrt(sum of squares + 1e-6) first. All sums and states are 32-bit;
a token with g < -104 (its decay is 0 in fp32) counts as a reset. What lies before a reset, NaN
and infinity included, has no effect on what follows. A NaN or an infinity in an operand has
none on outputs before its token either; an infinity may make NaN of what it meets. Two limits:
gradients of up to 31 tokens on either side of it may be NaN too, and so may up to 31 outputs before
a token whose own sums overflow fp32.
"""
from __future__ import annotations

import contextlib
import ctypes as C
from typing import Optional, Tuple

import torch

from . import _lib as L

L.one_runtime()

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_S3 = C.c_int64 * 3
_HERE = contextlib.nullcontext()
_written = torch.autograd.graph.increment_version


def _fail(rc: int, what: str) -> None:
    if rc == -6:
        raise ValueError(L.last_error())
    raise RuntimeError(f"{what} failed: {rc}: {L.last_error()}")


def _check(q, k, v, g, beta, reset, state, lead: int) -> None:
    """Shapes, types and devices; `lead` is the number of dimensions before the heads."""
    dtype, device, qs, vs, gs = q.dtype, q.device, q.shape, v.shape, g.shape
    if dtype not in _DTYPES:
        raise TypeError(f"q, k and v must be float32, float16 or bfloat16, not {dtype}")
    if len(qs) != lead + 2 or len(vs) != lead + 2:
        raise ValueError(f"q and v must have {lead + 2} dimensions, not {len(qs)} and {len(vs)}")
    if k.shape != qs or vs[:lead] != qs[:lead] or gs != vs[:-1] or beta.shape != gs:
        raise ValueError(f"shapes do not agree: q {tuple(qs)}, k {tuple(k.shape)}, v {tuple(vs)}, "
                         f"g {tuple(gs)}, beta {tuple(beta.shape)}")
    if 0 in qs or 0 in vs:
        raise ValueError(f"empty operands: q {tuple(qs)}, v {tuple(vs)}")
    if k.dtype is not dtype or v.dtype is not dtype:
        raise TypeError(f"q, k and v must have one type, not {dtype}, {k.dtype}, {v.dtype}")
    if g.dtype is not torch.float32 or beta.dtype is not torch.float32:
        raise TypeError(f"g and beta must be float32, not {g.dtype} and {beta.dtype}")
    if not q.is_cuda:
        raise ValueError("the operands must be on the GPU (there is no CPU fallback)")
    apart = k.device != device or v.device != device or g.device != device or beta.device != device
    if reset is not None:
        if reset.shape != qs[:lead]:
            raise ValueError(f"reset must have the shape {tuple(qs[:lead])}, not {tuple(reset.shape)}")
        if reset.dtype not in (torch.bool, torch.uint8):
            raise TypeError(f"reset must be bool or uint8, not {reset.dtype}")
        apart = apart or reset.device != device
    if state is not None:
        want = (qs[0], vs[lead], qs[-1], vs[-1])
        if state.shape != want:
            raise ValueError(f"state must have the shape {want}, not {tuple(state.shape)}")
        if state.dtype is not torch.float32:
            raise TypeError(f"state must be float32, not {state.dtype}")
        apart = apart or state.device != device
    if apart:
        raise ValueError("the operands must be on one device")


def _row(x: torch.Tensor) -> torch.Tensor:
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _inputs(q, k, v, g, beta, reset, state, scale, normalize) -> L.ZenoAmdDeltaInputs:
    qs, ks, vs, gs, bs = q.stride(), k.stride(), v.stride(), g.stride(), beta.stride()
    rs = (0, 0) if reset is None else reset.stride()
    if len(qs) == 4:
        b, t, hk, dk = q.shape
        qs, ks, vs = qs[:3], ks[:3], vs[:3]
    else:
        (b, hk, dk), t = q.shape, 1
        qs, ks, vs, gs, bs = (qs[0], 0, qs[1]), (ks[0], 0, ks[1]), (vs[0], 0, vs[1]), (gs[0], 0, gs[1]), (bs[0], 0, bs[1])
        rs = (rs[0], 0)
    _, hv, dv = v.shape[-3:]
    return L.ZenoAmdDeltaInputs(
        _DTYPES[q.dtype], b, t, hk, hv, dk, dv, normalize, scale,
        q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(),
        None if reset is None else reset.data_ptr(), None if state is None else state.data_ptr(), qs, ks, vs, gs, bs, rs)


def _space(n: int, x: torch.Tensor) -> Optional[torch.Tensor]:
    return torch.empty(n, dtype=torch.uint8, device=x.device) if n else None


def _stream(x: torch.Tensor) -> int:
    return torch.cuda.current_stream(x.device).cuda_stream


def _on(x: torch.Tensor):
    """The context in which x's device is the current one, as the library's calls need it."""
    return _HERE if torch.cuda.current_device() == x.device.index else torch.cuda.device(x.device)


class _GatedDelta(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, reset, state, scale, normalize, train):
        with _on(q):
            lib = L.load()
            a = _inputs(q, k, v, g, beta, reset, state, scale, normalize)
            o = torch.empty_like(v)  # v's order of dimensions: time-major in, time-major out
            if o.stride(-1) != 1 and o.shape[-1] != 1:
                o = torch.empty(v.shape, dtype=v.dtype, device=v.device)
            last = torch.empty((q.shape[0], v.shape[2], q.shape[3], v.shape[3]), dtype=torch.float32, device=q.device)
            saved = torch.empty(max(lib.zeno_amd_delta_saved_bytes(a), 1), dtype=torch.uint8, device=q.device) if train else None
            space = _space(lib.zeno_amd_delta_workspace_bytes(a), q)
            rc = lib.zeno_amd_delta_forward(a, o.data_ptr(), _S3(*o.stride()[:3]), last.data_ptr(),
                                            None if saved is None else saved.data_ptr(), None if space is None else space.data_ptr(), _stream(q))
            if rc:
                _fail(rc, "gated_delta")
        if train:
            ctx.save_for_backward(q, k, v, g, beta, reset, state, last, saved)
            ctx.scale, ctx.normalize = scale, normalize
            ctx.set_materialize_grads(False)
        return o, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_o, d_last):
        q, k, v, g, beta, reset, state, last, saved = ctx.saved_tensors
        if d_o is None and d_last is None:
            return (None,) * 10
        with _on(q):
            lib = L.load()
            a = _inputs(q, k, v, g, beta, reset, state, ctx.scale, ctx.normalize)
            d_o = torch.zeros_like(v) if d_o is None else _row(d_o)
            d_last = None if d_last is None else d_last.contiguous()
            d_q, d_k, d_v = (_dense_like(x) for x in (q, k, v))
            d_g, d_beta = _dense_like(g), _dense_like(beta)
            d_state = torch.empty_like(state) if state is not None and ctx.needs_input_grad[6] else None
            space = _space(lib.zeno_amd_delta_workspace_bytes(a), q)
            grads = L.ZenoAmdDeltaGradients(
                d_o.data_ptr(), _S3(*d_o.stride()[:3]), None if d_last is None else d_last.data_ptr(),
                d_q.data_ptr(), d_k.data_ptr(), d_v.data_ptr(), d_g.data_ptr(), d_beta.data_ptr(),
                None if d_state is None else d_state.data_ptr(),
                *(_S3(*x.stride()[:3]) for x in (d_q, d_k, d_v, d_g, d_beta)))
            rc = lib.zeno_amd_delta_backward(a, last.data_ptr(), saved.data_ptr(), grads, None if space is None else space.data_ptr(),
                                             _stream(q))
            if rc:
                _fail(rc, "gated_delta's gradients")
        return d_q, d_k, d_v, d_g, d_beta, None, d_state, None, None, None


def _dense_like(x: torch.Tensor) -> torch.Tensor:
    """Memory for x's gradient in x's order of dimensions, each value at a place of its own."""
    y = torch.empty_like(x)
    return y if y.stride(-1) == 1 or x.shape[-1] == 1 or x.dim() == 3 else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def gated_delta(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                reset: Optional[torch.Tensor] = None, state: Optional[torch.Tensor] = None, *,
                scale: Optional[float] = None, normalize: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """The rule over whole sequences. Returns o [B, T, Hv, value_dim] in the type of v and the
    state after the last token, a new tensor. Differentiable in q, k, v, g, beta and state."""
    _check(q, k, v, g, beta, reset, state, 2)
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    q, k, v = _row(q), _row(k), _row(v)
    state = None if state is None else state.contiguous()
    train = torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, v, g, beta, state))
    return _GatedDelta.apply(q, k, v, g, beta, reset, state, scale, bool(normalize), train)


def gated_delta_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                     state: torch.Tensor, reset: Optional[torch.Tensor] = None, *, scale: Optional[float] = None,
                     normalize: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token for every sequence: q, k [B, Hk, key_dim], v [B, Hv, value_dim], g, beta
    [B, Hv], reset [B]. `state` (contiguous, refused if autograd follows it) is advanced in place; returns o [B, Hv, value_dim]
    (`out` if given; it may be v, but overlap nothing else that the step reads or writes). Without gradients, even where an operand asks for them: training runs
    gated_delta on the recorded rollout."""
    _check(q, k, v, g, beta, reset, state, 1)
    if not state.is_contiguous():
        raise ValueError("state must be contiguous: it is advanced in place")
    if (state.requires_grad or (out is not None and out.requires_grad)) and torch.is_grad_enabled():
        raise ValueError("state and out are written in place, which autograd does not see: give detached ones, or step under torch.no_grad()")
    q, k, v = _row(q), _row(k), _row(v)
    if out is None:
        out = torch.empty_like(v, memory_format=torch.contiguous_format)
    elif out.shape != v.shape or out.dtype != v.dtype or out.device != v.device or (out.stride(-1) != 1 and out.shape[-1] != 1):
        raise ValueError(f"out must be like v: {tuple(v.shape)}, {v.dtype}, on {v.device}, its last dimension contiguous")
    with _on(q):
        a = _inputs(q, k, v, g, beta, reset, state, q.shape[-1] ** -0.5 if scale is None else float(scale), bool(normalize))
        os = out.stride()
        rc = L.load().zeno_amd_delta_step(a, out.data_ptr(), _S3(os[0], 0, os[1]), state.data_ptr(), _stream(q))
        if rc:
            _fail(rc, "gated_delta_step")
    _written(state)  # autograd refuses a backward pass that needs what was here
    _written(out)
    return out
