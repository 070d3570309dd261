"""The example that trains a policy with memory: the environments, the single-token step, whole
rollouts with gradients and the orthogonalised update, together as they are used."""
import importlib.util
from pathlib import Path

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_rollouts_and_updates():
    spec = importlib.util.spec_from_file_location("memory_policy", Path(__file__).resolve().parents[1] / "examples" / "memory_policy.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    history, apart = example.train(envs=200, updates=8, length=40, log=lambda line: None)
    assert len(history) == 8 and np.isfinite(history).all() and min(history) > 10
    # What was acted token by token is what the training pass differentiates: sums of at most
    # 32 + 40 terms of order one in fp32, and the projections of other batch shapes, by 1e-5.
    assert apart < 1e-4
