"""Values that are not finite reach no output before their token, in sequences as in single steps."""
import pytest
import torch

from tests.policy_reference import HALF_ULP, assert_near, gated_delta, work_error

pytestmark = pytest.mark.gpu
NAMES = ("q", "k", "v", "g", "beta")


def inputs(b, t, hk, hv, dk, dv, dtype, seed):
    r = torch.Generator().manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, generator=r)

    return {"q": normal(b, t, hk, dk).to(dtype), "k": normal(b, t, hk, dk).to(dtype), "v": normal(b, t, hv, dv).to(dtype),
            "g": -0.1 * torch.rand(b, t, hv, generator=r), "beta": torch.sigmoid(normal(b, t, hv)), "state": normal(b, hv, dk, dv)}


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")], ids=str)
@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("shape", [(2, 40, 1, 2, 64, 64), (1, 75, 2, 2, 128, 128), (3, 33, 1, 1, 24, 100)], ids=str)
def test_outputs_before_it_stay_as_they_are(shape, name, bad, dtype):
    from zeno_amd.memory import gated_delta as ours, gated_delta_step

    if name == "g" and bad == -float("inf"):
        pytest.skip("a reset")
    x = inputs(*shape, dtype, seed=sum(shape))
    for at in (5, 29):
        x[name][0, at, -1, ...] = bad  # one head (of g and beta), of q, k and v one row
    if name == "v":
        x[name][0, 5, -1, 1:] = 1.0    # and there one value
    # The reference takes a NaN for a decay below every other, a reset; an infinite one spoils the same values.
    want, last = gated_delta(**dict(x, g=torch.where(torch.isnan(x["g"]), torch.inf, x["g"])), normalize=True)
    d = {n: y.cuda() for n, y in x.items()}
    o, s = ours(**d, normalize=True)
    t, dk, dv = shape[1], shape[4], shape[5]
    assert_near(o, want, HALF_ULP[dtype] + work_error(t, dk, dv, 64), "o")
    assert_near(s, last, work_error(t, dk, dv, 64), "state")
    grown = {n: y.clone().requires_grad_(n == "q") for n, y in d.items()}  # with what training keeps: the same
    o2, _ = ours(**grown, normalize=True)
    assert torch.equal(torch.isfinite(o2), torch.isfinite(o))
    state = d["state"].clone()
    steps = torch.stack([gated_delta_step(*(d[n][:, i] for n in NAMES), state, normalize=True) for i in range(t)], 1)
    assert torch.equal(torch.isfinite(steps), torch.isfinite(o)) and torch.equal(torch.isfinite(state), torch.isfinite(s))


def test_in_a_segment_of_a_long_sequence():
    from zeno_amd.memory import gated_delta as ours

    x = inputs(1, 1500, 1, 1, 64, 64, torch.float32, seed=2)
    x["v"][0, 777, 0, 3] = float("nan")
    want, last = gated_delta(**x, normalize=True)
    o, s = ours(**{n: y.cuda() for n, y in x.items()}, normalize=True)
    assert_near(o, want, HALF_ULP[torch.float32] + work_error(1500, 64, 64, 64), "o")
    assert_near(s, last, work_error(1500, 64, 64, 64), "state")


def test_gradients_of_the_chunks_before_it():
    """A value that no gradient enters: what lies more than a chunk before it has the gradients of the
    sequence without it."""
    from zeno_amd.memory import gated_delta as ours

    x = inputs(1, 100, 1, 1, 64, 64, torch.float32, seed=4)
    results = []
    for value in (1.0, float("nan")):
        x["v"][0, 80, 0, :] = value
        d = {n: y.cuda().requires_grad_() for n, y in x.items()}
        o, _ = ours(**d, normalize=True)
        results.append(torch.autograd.grad(o[:, :64].sum(), [d[n] for n in NAMES]))
    for a, b in zip(*results):
        assert torch.isfinite(b[:, :64]).all() and torch.equal(a[:, :64], b[:, :64])
