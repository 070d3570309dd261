"""Linear attention's launch rules: sequences that are cut into segments have too few waves for the shape that the states
between segments have no kernel of, and a walk without a kernel is an error, never no launch (no GPU)."""
import shutil
import subprocess
from pathlib import Path

import pytest

from zeno_amd import _lib

CSRC = Path(__file__).resolve().parent.parent / "zeno_amd" / "csrc"
ROCM = Path("/opt/rocm")
CXX = shutil.which("g++")

pytestmark = pytest.mark.skipif(CXX is None or not (ROCM / "include" / "hip" / "hip_runtime.h").exists(), reason="needs g++ and the HIP headers")

PROGRAM = r"""
#include <cstdio>
#include "linear.h"
using namespace za::linear;

template <int TY> int launched(Kind kind, bool back, uint32_t batch, uint32_t segments, int length, int da, int dc) {
    Walk w{};
    w.batch = batch, w.heads = 1, w.segments = segments, w.length = length, w.da = da, w.dc = dc;
    return launch_walk<TY>(w, kind, back, nullptr) != hipErrorInvalidValue;
}

int main() {
    // Segments come with narrow waves only.
    long cut = 0;
    for (uint32_t batch = 1; batch <= 5000; batch += 1 + batch / 9)
        for (uint32_t heads : {1u, 2u, 3u, 8u, 64u})
            for (uint32_t length : {1u, 32u, 64u, 100u, 127u, 128u, 333u, 4096u, 1000000u})
                for (uint32_t dv = 1; dv <= 128; ++dv) {
                    ZenoAmdLinearInputs in{};
                    in.batch = batch, in.length = length, in.key_heads = 1, in.value_heads = heads, in.key_dim = 64, in.value_dim = dv;
                    const Segments s = segments_of(in);
                    if (s.count == 1) continue;
                    ++cut;
                    if (wide((uint64_t)batch * heads * s.count, (dv + 63) / 64, (dv + 31) / 32)) return std::printf("%u %u %u %u\n", batch, heads, length, dv), 1;
                }
    if (cut < 1000) return 2;
    // Enough sequences for waves of 64 columns, and states between segments all the same: no kernel.
    for (bool back : {false, true})
        for (int rows : {20, 64}) {
            if (launched<0>(STATES, back, 4096, 2, 64, rows, 64) || launched<1>(STATES, back, 4096, 2, 64, rows, 64) || launched<2>(STATES, back, 4096, 2, 64, rows, 64)) return 3;
        }
    return 0;
}
"""


def test_every_walk_has_a_kernel(tmp_path):
    _lib.load()
    source, program = tmp_path / "rules.cpp", tmp_path / "rules"
    source.write_text(PROGRAM)
    lib = _lib.LIB_PATH
    subprocess.run([CXX, "-std=c++17", "-w", "-D__HIP_PLATFORM_AMD__", f"-I{ROCM / 'include'}", f"-I{CSRC}", str(source), str(lib), f"-Wl,-rpath,{lib.parent}",
                    f"-L{ROCM / 'lib'}", f"-Wl,-rpath,{ROCM / 'lib'}", "-lamdhip64", "-o", str(program)], check=True)
    done = subprocess.run([str(program)], capture_output=True, text=True)
    assert done.returncode == 0, (done.returncode, done.stdout, done.stderr)
