"""Layer norm in 64 bits on the CPU, written from its definition; differentiable."""
import torch


def layer_norm(x, weight=None, bias=None, residual=None, eps=1e-5):
    """The rows' norm, and with a residual the sums, rounded to their type as the operator keeps
    them (their gradient passes the rounding)."""
    s = x.double()
    if residual is not None:
        exact = s + residual.double()
        s = exact + (exact.to(residual.dtype if residual.dtype != torch.float64 else exact.dtype).double() - exact).detach()
    mean = s.mean(-1, keepdim=True)
    y = (s - mean) / torch.sqrt(((s - mean) ** 2).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.double()
    if bias is not None:
        y = y + bias.double()
    return y if residual is None else (y, s)
