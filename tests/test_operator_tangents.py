"""Single steps have no derivatives: operands that carry tangents forward are refused, as whole sequences refuse them, where
the result would have lost them without a word. (No GPU: the library's calls do nothing here.)"""
import pytest
import torch
import torch.autograd.forward_ad as forward

from tests.test_operator_traces import calls  # noqa: F401
from zeno_amd import memory


def operands(beta):
    x = {"q": torch.randn(2, 1, 8), "k": torch.randn(2, 1, 8), "v": torch.randn(2, 1, 8), "g": torch.zeros(2, 1) if beta else torch.zeros(1)}
    return {**x, **({"beta": torch.ones(2, 1)} if beta else {}), "state": torch.zeros(2, 1, 8, 8), "out": torch.zeros(2, 1, 8)}


@pytest.mark.parametrize("step", [memory.linear_attention_step, memory.gated_delta_step])
def test_tangents_are_refused(step, calls):  # noqa: F811
    x = operands(step is memory.gated_delta_step)
    for name in x:
        for grad in (torch.enable_grad, torch.no_grad):
            with grad(), forward.dual_level():
                dual = forward.make_dual(x[name], torch.ones_like(x[name]))
                with pytest.raises(RuntimeError, match="tangent"):
                    step(**{**x, name: dual})
    assert not calls
    with forward.dual_level():  # operands without tangents are stepped
        step(**x)
    step(**x)
    assert sum("step" in c for c in calls) == 2
