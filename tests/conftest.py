"""Shared pytest setup: repo root on sys.path and the `gpu` marker."""
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

# torch's packages bring a HIP runtime of their own. Loaded first it is the one that libzeno.so and the
# tests' own calls use as well; loaded later it would be a second one in the process, which sees no GPU.
import torch  # noqa: E402,F401


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an AMD GPU (runs the HIP kernels through the C ABI)")
