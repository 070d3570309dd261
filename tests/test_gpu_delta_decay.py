"""Gradients of decays, down to those of the size of exp(-30), against the definition in 64 bits."""
import pytest
import torch

from tests.policy_reference import gated_delta, work_error

pytestmark = pytest.mark.gpu
NAMES = ("q", "k", "v", "g", "beta", "state")


def gradients(rule, x, do, ds, **options):
    x = {n: y.clone().requires_grad_() if n in NAMES else y for n, y in x.items()}
    o, s = rule(**x, **options)
    return dict(zip(NAMES, torch.autograd.grad((o, s), [x[n] for n in NAMES], (do, ds))))


def both(x, do, ds, **options):
    from zeno_amd.memory import gated_delta as ours

    want = gradients(gated_delta, {n: y.double() if n in NAMES else y for n, y in x.items()}, do.double(), ds.double(), **options)
    got = gradients(ours, {n: y.cuda() for n, y in x.items()}, do.cuda(), ds.cuda(), **options)
    return {n: y.double().cpu() for n, y in got.items()}, want


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("dim", [(64, 64), (128, 128), (24, 100)], ids=str)
@pytest.mark.parametrize("length", [32, 45])
def test_decays_of_heads_that_forget_fast(length, dim, dtype):
    """One strength of forgetting a head, and each head's gradient of g by itself: it is of the size of
    exp(g), and as exact as sums in fp32 relative to that."""
    strengths = [-0.5, -4.0, -8.0, -12.0, -16.0, -30.0]
    dk, dv = dim
    r = torch.Generator().manual_seed(length + dk)

    def normal(*s):
        return torch.randn(*s, generator=r)

    h = len(strengths)
    x = {"q": normal(2, length, h, dk).to(dtype), "k": normal(2, length, h, dk).to(dtype), "v": normal(2, length, h, dv).to(dtype),
         "g": torch.tensor(strengths).expand(2, length, h) * (1.0 + 0.1 * torch.rand(2, length, h, generator=r)), "beta": torch.sigmoid(normal(2, length, h)),
         "state": normal(2, h, dk, dv)}
    got, want = both(x, normal(2, length, h, dv).to(dtype), normal(2, h, dk, dv), normalize=True)
    for i, g in enumerate(strengths):
        error, norm = float((got["g"] - want["g"])[..., i].norm()), float(want["g"][..., i].norm())
        assert error <= 4 * work_error(length, dk, dv, 64) * norm, (g, error / norm)


def test_a_token_that_forgets_among_others_that_do_not():
    """Each token's gradient by itself: those of the strong decays are of the size of exp(-25)."""
    r = torch.Generator().manual_seed(5)
    t, d = 70, 64
    x = {n: torch.randn(1, t, 1, d, generator=r) for n in "qkv"}
    x.update(g=torch.full((1, t, 1), -0.01), beta=torch.sigmoid(torch.randn(1, t, 1, generator=r)), state=torch.randn(1, 1, d, d, generator=r))
    strong = [4, 11, 16, 31, 32, 50, 69]
    x["g"][:, strong] = -25.0
    got, want = both(x, torch.randn(1, t, 1, d, generator=r), torch.randn(1, 1, d, d, generator=r), normalize=True)
    error, norm = (got["g"] - want["g"])[0, strong, 0].norm(), want["g"][0, strong, 0].norm()
    assert float(error) <= 4 * work_error(t, d, d, 64) * float(norm), float(error / norm)
