"""Linear attention with a decay for each head in 64 bits on the CPU, written from its definition."""
import torch


def linear_attention(q, k, v, g, reset=None, state=None, scale=None):
    """Token by token in float64; differentiable. A cleared state is a new one, not a product."""
    share, (b, t, _, dk) = v.shape[2] // q.shape[2], q.shape
    q, k, v, g = (x.double() for x in (q, k, v, g))
    q, k = q.repeat_interleave(share, 2), k.repeat_interleave(share, 2)
    scale = dk ** -0.5 if scale is None else scale
    s = torch.zeros(b, v.shape[2], dk, v.shape[3], dtype=torch.float64) if state is None else state.double()
    decay, out = torch.exp(g)[:, None, None], []
    for i in range(t):
        if reset is not None:
            s = torch.where(reset[:, i, None, None, None].bool(), torch.zeros_like(s), s)
        s = decay * s + k[:, i, :, :, None] * v[:, i, :, None, :]
        out.append(scale * (s * q[:, i, :, :, None]).sum(-2))
    return torch.stack(out, 1), s
