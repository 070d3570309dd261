"""The example's measure of how far acted outputs are from those that are differentiated: itself for the gated delta
rule, a share of the largest output for linear attention."""
import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("memory", ["delta", "linear"])
def test_large_outputs_that_differ(memory, monkeypatch):
    spec = importlib.util.spec_from_file_location("memory_policy", Path(__file__).resolve().parents[1] / "examples" / "memory_policy.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    remember, recall, largest = example.Policy.remember, example.Policy.recall, []

    def far(self, *a):
        o = recall(self, *a) + 1000.5
        largest.append(float(o.detach().abs().max()))
        return o

    monkeypatch.setattr(example.Policy, "remember", lambda self, *a: remember(self, *a) + 1000.0)
    monkeypatch.setattr(example.Policy, "recall", far)
    _, apart = example.train(envs=64, updates=1, length=8, log=lambda line: None, memory=memory)
    want = 0.5 if memory == "delta" else 0.5 / largest[0]
    assert largest[0] > 900.0
    assert abs(apart - want) < want / 2  # a number near 1000 is rounded by 2^-15
