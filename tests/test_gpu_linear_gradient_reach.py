"""Which gradients of linear attention a value that is not finite reaches, by the definition: from the gradient of o
and from q those of k and v (and of the first state) at tokens up to its own, back to the reset before it; from k and v
those of q from its token on, up to the next reset, and its own token's of v or k. The kernels' are finite in the same
places, and there have the definition's values."""
import pytest
import torch

from tests.linear_reference import linear_attention as definition
from tests.policy_reference import HALF_ULP, assert_near, work_error

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("where", ["q", "k", "v", "d_o"])
def test_one_value(where, bad, dtype):
    from zeno_amd.memory import linear_attention

    # One chunk, several, one segment and several; waves of 64 columns in the last.
    for b, t, at, dk, dv in ((2, 20, 5, 40, 64), (2, 90, 37, 40, 64), (1, 500, 140, 24, 33), (1030, 40, 21, 64, 64)):
        r = torch.Generator().manual_seed(at)

        def normal(*s):
            return torch.randn(*s, generator=r)

        x = {"q": normal(b, t, 1, dk).to(dtype), "k": normal(b, t, 1, dk).to(dtype), "v": normal(b, t, 2, dv).to(dtype), "state": normal(b, 2, dk, dv)}
        d_o, g, reset = normal(b, t, 2, dv).to(dtype), torch.tensor([-0.02, -0.3]), torch.zeros(b, t, dtype=torch.bool)
        if t > 20:
            reset[:, [at - 9, at + 12]] = True
        y = d_o if where == "d_o" else x[where]
        y[0, at, -1, 7] = bad
        some = slice(0, 2)  # the definition's share of many sequences
        ref = {n: z[some].double().requires_grad_() for n, z in x.items()}
        dev = {n: z.cuda().requires_grad_() for n, z in x.items()}
        want = torch.autograd.grad(definition(**ref, g=g, reset=reset[some])[0], list(ref.values()), d_o[some].double())
        got = torch.autograd.grad(linear_attention(**dev, g=g.cuda(), reset=reset.cuda())[0], list(dev.values()), d_o.cuda())
        work, half = work_error(t // 32 + 32, dk, dv), HALF_ULP[dtype]
        for n, p, w in zip(x, got, want):
            assert_near(p[some], w, (half if n != "state" else 0.0) + work, f"gradient of {n}, {t} tokens")
            assert torch.isfinite(p[2:]).all()
        spoilt = {n: ~torch.isfinite(w[0]).flatten(1).all(1) for n, w in zip(x, want)}
        if where in ("k", "v"):
            assert spoilt["q"][at:at + 12].all() and not spoilt["q"][:at].any() and not spoilt["q"][at + 12:].any() if t > 20 else spoilt["q"][at:].all()
        else:
            assert spoilt["k"][max(at - 9, 0):at + 1].all() and spoilt["v"][max(at - 9, 0):at + 1].all() and not spoilt["k"][at + 1:].any()
