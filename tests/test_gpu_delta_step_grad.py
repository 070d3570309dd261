"""A single step writes its state and its output in place and has no gradients: what autograd follows is
refused, as torch's own operations in place refuse a leaf."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def token():
    r = torch.Generator(device="cuda").manual_seed(2)

    def normal(*s):
        return torch.randn(*s, generator=r, device="cuda")

    return [normal(3, 2, 16), normal(3, 2, 16), normal(3, 2, 16), -torch.rand(3, 2, device="cuda"), torch.rand(3, 2, device="cuda")], normal(3, 2, 16, 16)


def test_a_state_or_output_with_gradients_is_refused():
    from zeno_amd.memory import gated_delta_step

    x, state = token()
    before = state.clone()
    leaf = state.clone().requires_grad_()
    for bad in (leaf, leaf * torch.ones_like(leaf), leaf.view_as(leaf)):
        with pytest.raises(ValueError, match="autograd"):
            gated_delta_step(*x, bad)
        assert torch.equal(bad, before)
    with pytest.raises(ValueError, match="autograd"):
        gated_delta_step(*x, state, out=torch.zeros(3, 2, 16, device="cuda", requires_grad=True))
    assert torch.equal(state, before)


def test_what_autograd_does_not_follow_is_stepped():
    from zeno_amd.memory import gated_delta_step

    x, state = token()
    want = gated_delta_step(*x, state)
    _, first = token()
    asked = [y.clone().requires_grad_() for y in x]
    s = first.clone()
    assert torch.equal(gated_delta_step(*asked, s), want) and torch.equal(s, state)  # operands may ask for gradients
    s = first.clone().requires_grad_()
    with torch.no_grad():
        assert torch.equal(gated_delta_step(*asked, s), want) and torch.equal(s, state)
    with torch.inference_mode():
        s = first.clone()
        assert torch.equal(gated_delta_step(*x, s), want) and torch.equal(s, state)
