"""Gradients of q and k behind their norms, which take away most of what is summed: the digits of
fp32 have to be there in every type. Against the definition in 64 bits."""
import pytest
import torch

from tests.policy_reference import gated_delta

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


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("dim", [(64, 64), (128, 128), (64, 128)], ids=str)
def test_what_the_norms_take_away(dtype, dim):
    """A state that is 1000 times the query (and key) but for a part across it: the gradients of q and
    k are that part, what remains of terms 1000 times as large when their share along q is taken
    away. Every term passes about 16 roundings of fp32, so the rest is off by 16 * 2^-24 * 1000 of it
    (twice that behind the result's own rounding, as in the orthogonalisation's test)."""
    dk, dv = dim
    r = torch.Generator().manual_seed(7)
    large = 1000.0
    q = torch.randn(1, 1, 1, dk, generator=r).to(dtype)
    unit = (q.double() / q.double().norm())[0, 0, 0]
    across = torch.randn(dk, generator=r).double()
    across = across / across.norm()
    column = (large * unit + across).float()
    state = torch.zeros(1, 1, dk, dv)
    state[0, 0, :, 0] = column
    x = {"q": q, "k": q.clone(), "v": torch.randn(1, 1, 1, dv, generator=r).to(dtype), "g": torch.zeros(1, 1, 1), "beta": torch.full((1, 1, 1), 0.5),
         "state": state}
    do = torch.zeros(1, 1, 1, dv)
    do[..., 0] = 1.0
    got, want = both(x, do.to(dtype), torch.zeros(1, 1, dk, dv), scale=1.0, normalize=True)
    for n in "qk":
        rounding = float((want[n].to(dtype).double() - want[n]).norm())
        error, norm = float((got[n] - want[n]).norm()), float(want[n].norm())
        assert error <= rounding + 2 * 16 * 2.0 ** -24 * large * norm, (n, error / norm, rounding / norm)
