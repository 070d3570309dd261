"""The operators of policies in 64 bits on the CPU, written from their definitions, and the
tolerances that their tests use."""
import torch

EPS = 1e-6
HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def unit(x):
    return x / torch.sqrt((x * x).sum(-1, keepdim=True) + EPS)


def gated_delta(q, k, v, g, beta, reset=None, state=None, scale=None, normalize=False):
    """Token by token in float64; differentiable. A cleared state is a new one, not a product."""
    share, (b, t, _, dk) = v.shape[2] // q.shape[2], q.shape
    q, k, v, g, beta = (x.double() for x in (q, k, v, g, beta))
    if normalize:
        q, k = unit(q), unit(k)
    q, k = q.repeat_interleave(share, 2), k.repeat_interleave(share, 2)
    scale = dk ** -0.5 if scale is None else scale
    s = torch.zeros(b, v.shape[2], dk, v.shape[3], dtype=torch.float64) if state is None else state.double()
    out = []
    for i in range(t):
        keep = g[:, i] >= -104.0
        if reset is not None:
            keep = keep & ~reset[:, i, None].bool()
        decay = torch.exp(torch.where(keep, g[:, i], torch.zeros_like(g[:, i])))[..., None, None]
        s = torch.where(keep[..., None, None], s, torch.zeros_like(s)) * decay
        e = v[:, i] - (s * k[:, i, :, :, None]).sum(-2)
        s = s + k[:, i, :, :, None] * (beta[:, i, :, None] * e)[:, :, None, :]
        out.append(scale * (s * q[:, i, :, :, None]).sum(-2))
    return torch.stack(out, 1), s


def work_error(*lengths):
    """Largest relative error (2-norm) of sums in fp32 whose longest dependent chain has the sum
    of `lengths` terms: each addition rounds by 2^-24 of the partial sum, and a partial sum is
    at most a few times the result for the inputs of these tests (4)."""
    return 4 * sum(lengths) * 2.0 ** -24


def assert_near(got, want, tol, what=""):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)), f"{what}: finite values in other places"
    err, norm = float((got - want)[fine].norm()), float(want[fine].norm())
    assert err <= tol * norm + 1e-30, f"{what}: off by {err / max(norm, 1e-300):.3g} of its norm, {tol:.3g} allowed"


def orthogonalize(x, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7):
    """Newton-Schulz in float64, matrix by matrix, from the definition."""
    a, b, c = coefficients
    out = torch.empty(x.shape, dtype=torch.float64)
    for i, g in enumerate(x.double().reshape(-1, *x.shape[-2:])):
        y = g.T if g.shape[0] > g.shape[1] else g
        y = y / (torch.linalg.norm(y) + eps)
        for _ in range(steps):
            s = y @ y.T
            y = a * y + (b * s + c * s @ s) @ y
        out.view(-1, *x.shape[-2:])[i] = y.T if g.shape[0] > g.shape[1] else y
    return out
