"""Traced operators give the results that the calls give, for inputs other than those they were traced with, and their gradients."""
import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore")]


def inputs(b, t, seed):
    r = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, generator=r, device="cuda")

    return normal(b, t, 2, 24), normal(b, t, 2, 24), normal(b, t, 2, 40), -torch.rand(2, generator=r, device="cuda")


def attended(q, k, v, g):
    from zeno_amd.memory import linear_attention

    return linear_attention(q, k, v, g)


def normed(q, k, v, g):
    from zeno_amd.norm import layer_norm

    return layer_norm(q, residual=k)


def normed_alone(q, k, v, g):
    from zeno_amd.norm import layer_norm

    return layer_norm(v.flatten(2), v[0, 0].flatten())


@pytest.mark.parametrize("call", [attended, normed, normed_alone])
@pytest.mark.parametrize("grad", [False, True])
def test_traced(call, grad):
    example = inputs(2, 30, 1)
    with torch.enable_grad() if grad else torch.no_grad():
        traced = torch.jit.trace(call, tuple(x.requires_grad_(grad) for x in example))
    for b, t, seed in ((2, 30, 2), (3, 70, 3), (1, 400, 4)):
        x = inputs(b, t, seed)
        with torch.no_grad():
            want = call(*x)
            want = want if isinstance(want, tuple) else (want,)
            got = traced(*x)
            got = got if isinstance(got, tuple) else (got,)
        assert len(got) == len(want) and all(torch.equal(p, q) for p, q in zip(got, want))
        grads = []
        for f in (call, traced):
            leaves = [y.clone().requires_grad_() for y in x]
            out = f(*leaves)
            out = out if isinstance(out, tuple) else (out,)
            grads.append(torch.autograd.grad(sum(y.square().sum() for y in out), leaves, allow_unused=True))
        assert any(y is not None for y in grads[0])
        assert all(p is q is None or torch.equal(p, q) for p, q in zip(*grads))
