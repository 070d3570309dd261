"""The library without torch, on the HIP runtime that it is linked to: what a program that only simulates
uses. The suite itself loads torch's runtime first."""
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

ROOT = Path(__file__).resolve().parent.parent

STEPS = """
import sys
import numpy as np
from zeno_amd import ASSETS
from zeno_amd.world import ZenoWorld

def run(scene, envs):
    w = ZenoWorld(mjcf_path=str(ASSETS / scene), num_envs=envs)
    r = np.random.default_rng(3)
    for _ in range(12):
        w.step(r.uniform(-1, 1, (envs, w.action_dim)).astype(np.float32))
    w.reset(np.arange(envs) % 3 == 0)
    w.step(r.uniform(-1, 1, (envs, w.action_dim)).astype(np.float32))
    return np.concatenate([np.asarray(w.get_observations()).ravel(), np.asarray(w.get_body_positions()).ravel(), np.asarray(w.get_rewards()).ravel()])
"""


def child(code):
    return subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=100)


@pytest.mark.gpu
@pytest.mark.parametrize("scene, envs", [("ant.xml", 200), ("cartpole.xml", 33)])
def test_a_world_steps_the_same_on_the_library_s_own_runtime(scene, envs, tmp_path):
    import torch  # noqa: F401  (here on its runtime)

    out = tmp_path / "state.npy"
    done = child(STEPS + f"""
np.save({str(out)!r}, run({scene!r}, {envs}))
assert "torch" not in sys.modules
runtimes = {{line.split()[-1] for line in open("/proc/self/maps") if "/libamdhip64.so" in line}}
assert len(runtimes) == 1 and "torch" not in runtimes.pop()
""")
    assert done.returncode == 0, done.stderr
    names = {}
    exec(STEPS, names)
    here, there = names["run"](scene, envs), np.load(out)
    assert np.isfinite(there).all() and np.array_equal(here, there)


def test_the_suite_loads_without_torch():
    """Its configuration leaves out the files that need torch, and the library loads and answers."""
    done = child("""
import sys
sys.modules["torch"] = None
import tests.conftest as c
assert "test_gpu_delta.py" in c.collect_ignore and "test_gpu_memory_policy.py" in c.collect_ignore and "test_gpu_sqrt.py" not in c.collect_ignore
from zeno_amd import _lib
assert _lib.load().zeno_amd_device_count() >= 0
""")
    assert done.returncode == 0, done.stderr
