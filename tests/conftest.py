"""Shared pytest setup: repo root on sys.path and the `gpu` marker."""
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

# torch's packages bring a HIP runtime of their own. Loaded first it is the one that libzeno.so and the
# tests' own calls use as well; loaded later it would be a second one in the process, which sees no GPU.
# Without torch the suite runs but for the files that name it (the policy operators' and their example's).
try:
    import torch  # noqa: E402,F401
except ImportError:
    import pathlib

    collect_ignore = sorted(f.name for f in pathlib.Path(__file__).parent.glob("test_*.py") if "torch" in f.read_text() or "memory_policy" in f.read_text())


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an AMD GPU (runs the HIP kernels through the C ABI)")
