"""Linear attention's heads that grow: what a whole chunk or segment would make of a state may pass fp32's
range, which is no matter while the state is zero, or so small that the result does not.

Tolerances as in the sequences' tests. No token adds to what is many tokens old, so the chains are no longer.
Scales and sizes keep every value of the definition within fp32 (and its type), which the tests look at first.
"""
import math

import pytest
import torch

from tests.linear_reference import linear_attention as definition
from tests.policy_reference import HALF_ULP, assert_near, work_error

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def inputs(b, t, h, dk, dv, dtype, seed):
    r = torch.Generator().manual_seed(seed)

    def normal(*s):
        return torch.randn(*s, generator=r)

    return {"q": normal(b, t, h, dk).to(dtype), "k": normal(b, t, h, dk).to(dtype), "v": normal(b, t, h, dv).to(dtype)}, normal(b, t, h, dv).to(dtype)


def check(x, d_o, g, scale, state=None, reset=None):
    """Outputs, the state and every gradient."""
    from zeno_amd.memory import linear_attention

    names = ["q", "k", "v", "g"] + (["state"] if state is not None else [])
    x = {**x, "g": torch.tensor(g), "state": state, "reset": reset}
    ref = {n: y.double().requires_grad_() if n in names else y for n, y in x.items()}
    dev = {n: y if y is None else y.cuda().requires_grad_(n in names) for n, y in x.items()}
    o, s = definition(**ref, scale=scale)
    want = torch.autograd.grad(o, [ref[n] for n in names], d_o.double())
    largest = torch.finfo(x["q"].dtype).max / 4
    assert all(float(y.detach().abs().max()) < min(largest, 1e38) for y in (o, *want[:3])) and all(float(y.detach().abs().max()) < 1e38 for y in (s, *want[3:]))
    po, ps = linear_attention(**dev, scale=scale)
    got = torch.autograd.grad(po, [dev[n] for n in names], d_o.cuda())
    (b, t, _, dk), dv = x["q"].shape, x["v"].shape[3]
    work, half = work_error(t // 32 + 32, dk, dv), HALF_ULP[x["q"].dtype]
    assert_near(po, o, half + work, "o")
    assert_near(ps, s, work, "state")
    for n, p, y in zip(names, got, want):
        assert_near(p, y, (half if n in "qkv" else 0.0) + work, "gradient of " + n)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("t", [16, 28, 29, 30, 31])
def test_a_chunk_that_passes_the_range(t, dtype):
    """exp(3 * 30) is beyond fp32; the states, of keys that small, are not. Scaled so that float16 holds the outputs."""
    x, d_o = inputs(2, t, 2, 32, 40, dtype, seed=t)
    x["k"] = (x["k"].float() * 2.0 ** -11).to(dtype)
    check(x, d_o, [3.0, -0.5], scale=2.0 ** (4 - int(3 * (t - 1) / math.log(2))))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_a_small_state_grows_to_its_digits(dtype):
    """1e-30 after 30 tokens of exp(3): 1e9, not an infinity."""
    x, d_o = inputs(2, 30, 1, 32, 40, dtype, seed=5)
    x["k"][:] = x["v"][:] = 0
    r = torch.Generator().manual_seed(6)
    check(x, d_o, [3.0], scale=2.0 ** -30, state=1e-30 * torch.randn(2, 1, 32, 40, generator=r))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("g", [0.4, 0.9, 1.5, 3.0])
def test_segments_that_pass_the_range(g, dtype):
    """One long sequence in segments. Its keys are zero up to the last tokens, so the state is, whatever a segment would
    make of it; the gradient comes from the first tokens only, so that of the state is zero behind them."""
    t, live = 500, int(60 / g)
    x, d_o = inputs(1, t, 1, 32, 40, dtype, seed=9)
    x["k"][:, :-live] = 0
    d_o[:, live:] = 0
    check(x, d_o, [g], scale=2.0 ** -87)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_long_segments_that_pass_the_range(dtype):
    """The same where many sequences leave segments of 256 tokens: exp(0.4 * 256)."""
    t, live, g = 1024, 150, 0.4
    x, d_o = inputs(64, t, 8, 4, 3, dtype, seed=10)
    x["k"][:, :-live] = 0
    d_o[:, live:] = 0
    check(x, d_o, [g] * 8, scale=2.0 ** -87)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("g", [88.0, 90.0, 170.0, 300.0])
def test_one_token_that_passes_the_range(g, dtype):
    """exp(90) is beyond fp32 by itself. Nothing is carried where every token begins an episode, and a state of
    zeros stays one; one of 2^-120 becomes 900."""
    from zeno_amd.memory import linear_attention, linear_attention_step

    x, d_o = inputs(3, 40, 2, 32, 40, dtype, seed=11)
    check(x, d_o, [g, -0.5], None, reset=torch.ones(3, 40, dtype=torch.bool))
    one, d_o = inputs(3, 1, 2, 32, 40, dtype, seed=12)
    check(one, d_o, [g, -0.5], None)
    states = [(torch.zeros(3, 2, 32, 40), None)]
    if g < 100:
        states.append((torch.full((3, 2, 32, 40), 2.0 ** -120), 2.0 ** -9))
        check(one, d_o, [g, -0.5], states[1][1], state=states[1][0])
    decays = torch.tensor([g, -0.5])
    for state, scale in states:
        o, s = definition(**one, g=decays, state=state, scale=scale)
        kept = state.clone().cuda()
        got = linear_attention_step(*(one[n][:, 0].cuda() for n in "qkv"), decays.cuda(), kept, scale=scale)
        whole, last = linear_attention(*(one[n].cuda() for n in "qkv"), decays.cuda(), None, state.clone().cuda(), scale=scale)
        for a, b in ((got, kept), (whole[:, 0], last)):
            assert_near(a, o[:, 0], HALF_ULP[dtype] + work_error(3, 32), "o")
            assert_near(b, s, work_error(3, 32), "state")
