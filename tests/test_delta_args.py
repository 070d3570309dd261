"""The gated delta rule's entry points on the CPU: argument checks that come before any GPU
work, and the sizes of what training keeps."""
import ctypes as C
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from zeno_amd import _lib, memory

ROOT = Path(__file__).resolve().parent.parent


def args(**change):
    a = dict(dtype=0, batch=2, length=70, key_heads=2, value_heads=4, key_dim=32, value_dim=32, normalize=1, scale=1.0, q=16, k=16, v=16, g=16, beta=16)
    return _lib.ZenoAmdDeltaInputs(**{**a, **change})


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


@pytest.mark.parametrize("change, words", [
    ({"dtype": 3}, "dtype"), ({"batch": 0}, "positive"), ({"length": 0}, "positive"), ({"value_heads": 5}, "multiple"),
    ({"key_dim": 129}, "1 to 128"), ({"value_dim": 0}, "1 to 128"), ({"q": None}, "null input"), ({"beta": None}, "null input"),
    ({"scale": float("inf")}, "scale"), ({"batch": 1 << 31}, "too many")])
def test_refused_before_any_gpu_work(lib, change, words):
    a, strides = args(**change), (C.c_int64 * 3)()
    assert lib.zeno_amd_delta_forward(a, 16, strides, 16, None, None, None) == -6
    assert words in _lib.last_error()
    assert lib.zeno_amd_delta_backward(a, 16, 16, _lib.ZenoAmdDeltaGradients(), 16, None) == -6
    assert lib.zeno_amd_delta_step(a, 16, strides, 16, None) == -6


def test_null_results_are_refused(lib):
    strides = (C.c_int64 * 3)()
    assert lib.zeno_amd_delta_forward(None, 16, strides, 16, None, None, None) == -6
    assert lib.zeno_amd_delta_forward(args(), None, strides, 16, None, None, None) == -6
    assert lib.zeno_amd_delta_forward(args(state=64), 16, strides, 64, None, None, None) == -6
    assert "overwrite" in _lib.last_error()
    assert lib.zeno_amd_delta_backward(args(), 16, 16, _lib.ZenoAmdDeltaGradients(), None, None) == -6
    assert lib.zeno_amd_delta_step(args(), 16, strides, 16, None) == -6  # 70 tokens
    assert "one token" in _lib.last_error()
    assert lib.zeno_amd_delta_step(args(length=1), 16, strides, None, None) == -6


def test_sizes_of_what_training_keeps(lib):
    """A state for every 32 tokens but the first ones, padded to the launch shape; gradients of
    q and k for each value head where heads share keys."""
    assert lib.zeno_amd_delta_saved_bytes(args()) == 4 * 2 * 4 * 2 * 64 * 64
    assert lib.zeno_amd_delta_saved_bytes(args(length=32)) == 0
    assert lib.zeno_amd_delta_saved_bytes(args(key_dim=300)) == 0
    assert lib.zeno_amd_delta_workspace_bytes(args()) == 4 * 2 * 2 * 70 * 4 * 32
    assert lib.zeno_amd_delta_workspace_bytes(args(key_heads=4)) == 0


def test_python_refuses_cpu_tensors_and_wrong_shapes():
    z = torch.zeros
    good = [z(1, 2, 1, 4), z(1, 2, 1, 4), z(1, 2, 1, 4), z(1, 2, 1), z(1, 2, 1)]
    with pytest.raises(ValueError, match="GPU"):
        memory.gated_delta(*good)
    with pytest.raises(ValueError, match="do not agree"):
        memory.gated_delta(good[0], z(1, 2, 1, 5), *good[2:])
    with pytest.raises(ValueError, match="dimensions"):
        memory.gated_delta_step(*good, z(1, 1, 4, 4))
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        memory.gated_delta(good[0].double(), *good[1:])


def test_segments_of_long_sequences(lib):
    """One head over 4096 tokens: 128 chunks, 32 segments of 4, states and matrices between them."""
    long = args(batch=1, key_heads=1, value_heads=1, length=4096)
    assert lib.zeno_amd_delta_workspace_bytes(long) == 4 * 31 * (64 * 64 + 3 * 64 * 64 + 4)
    assert lib.zeno_amd_delta_saved_bytes(long) == 4 * (127 * 64 * 64 + 31 * (3 * 64 * 64 + 4))
    assert lib.zeno_amd_delta_forward(long, 16, (C.c_int64 * 3)(), 16, None, None, None) == -6
    assert "workspace" in _lib.last_error()
    assert lib.zeno_amd_delta_forward(long, 16, (C.c_int64 * 3)(), 16, None, 8, None) == -6
    assert lib.zeno_amd_delta_workspace_bytes(args(batch=512, length=4096, key_heads=4)) == 0


@pytest.mark.parametrize("module", ["memory", "optim"])
def test_torch_has_to_come_before_the_library(module):
    """Two HIP runtimes in one process are refused by name, one shared by both is not."""
    def run(first, then):
        return subprocess.run([sys.executable, "-c", f"{first}; {then}"], cwd=ROOT, capture_output=True, text=True)

    load, use = "from zeno_amd import _lib; _lib.load()", f"import zeno_amd.{module}"
    late = run(load, use)
    assert late.returncode == 1 and "import torch before" in late.stderr, late.stderr
    early = run("import torch", f"{load}; {use}")
    assert early.returncode == 0, early.stderr
