"""Waits behind matrix instructions that tests/test_matrix_waits.py does not look for: a later matrix
instruction that takes the result as an operand other than its accumulator needs the same eight states
as any reader (only an accumulator that is passed on whole is the hardware's own matter), and some
instructions read the register that they write: multiply-adds into their destination, swaps between
lanes, and writes of a part of a register or of some of its lanes."""
import re
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from tests.test_matrix_waits import READ, WRITE, kernels, registers
from zeno_amd import build

READS_ITS_RESULT = re.compile(r"v_(pk_)?(fmac|mac|dot\w*c)_|_swap|v_swap|writelane|_sdwa|fma_mix(lo|hi)|d16_hi|_dpp")
BOTH_WRITTEN = re.compile(r"_swap|v_swap")


def split_operands(text):
    """Register operands at the top level, in order."""
    return [x.strip() for x in re.split(r",(?![^\[]*\])", text)]


def early(code):
    """Instructions that touch a matrix result before it is safe: (matrix instruction, user, wait states)."""
    at = {x: i for i, (op, x) in enumerate(code) if op == "label"}
    found = []
    for i, (op, operands) in enumerate(code):
        if "mfma" not in op:
            continue
        result = registers(split_operands(operands)[0])
        paths, seen = [(i + 1, 0, frozenset(result))], set()
        while paths:
            j, states, live = paths.pop()  # live: what no other matrix instruction has written since
            while j < len(code) and states < READ and live and (j, states, live) not in seen:
                seen.add((j, states, live))
                o, x = code[j]
                if o == "label":
                    j += 1
                    continue
                if o == "s_nop":
                    states += int(x, 0) + 1
                    j += 1
                    continue
                parts = split_operands(x)
                if "mfma" in o:
                    to, a, b, c = (registers(p) for p in parts[:4])
                    if (a | b) & live or (c & live and c != result):
                        found.append((f"{op} {operands}", f"{o} {x}", states))
                        break
                    live = live - to  # written in order; its own result is followed by itself
                elif o.startswith("v_"):
                    writes = registers(parts[0]) | (registers(parts[1]) if BOTH_WRITTEN.search(o) else set())
                    reads = set().union(*map(registers, parts[1:]))
                    if READS_ITS_RESULT.search(o) or re.search(r"quad_perm|row_|bound_ctrl|dst_unused:UNUSED_PRESERVE|op_sel", x):
                        reads |= writes
                    if reads & live or (states < WRITE and writes & live):
                        found.append((f"{op} {operands}", f"{o} {x}", states))
                        break
                elif o == "s_branch":
                    j, states = at[x], states + 1
                    continue
                elif o.startswith("s_cbranch"):
                    paths.append((at[x], states + 1, live))
                elif o == "s_endpgm":
                    break
                j, states = j + 1, states + 1
    return found


PRODUCT = "v_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[8:11], v[0:3]"


@pytest.mark.parametrize("user, waits, bad", [
    ("v_mfma_f32_16x16x32_bf16 v[20:23], v[0:3], v[8:11], v[20:23]", 7, True),
    ("v_mfma_f32_16x16x32_bf16 v[20:23], v[8:11], v[2:5], v[20:23]", 7, True),
    ("v_mfma_f32_16x16x32_bf16 v[20:23], v[8:11], v[2:5], v[20:23]", 8, False),
    ("v_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[8:11], v[0:3]", 0, False),        # accumulated on
    ("v_mfma_f32_16x16x32_bf16 v[2:5], v[24:27], v[8:11], v[2:5]", 0, True),       # a part of it
    ("v_fmac_f32_e32 v1, v20, v21", 7, True), ("v_fmac_f32_e32 v1, v20, v21", 8, False),
    ("v_permlane32_swap_b32 v20, v2", 7, True), ("v_permlane16_swap_b32 v2, v20", 7, True),
    ("v_mov_b32_dpp v1, v20 row_shr:1 row_mask:0xf bank_mask:0xf", 7, True),
    ("v_mov_b32_e32 v1, v20", 7, False), ("v_mov_b32_e32 v1, v20", 6, True), ("v_add_f32_e32 v20, v1, v2", 7, True)])
def test_the_check_sees_each(user, waits, bad):
    nop = f"s_nop {waits - 1}" if waits else ""
    (code,) = kernels(f"_Zk:\n    {PRODUCT}\n    {nop}\n    {user}\n    s_endpgm").values()
    assert [u for p, u, _ in early(code) if p == PRODUCT] == [user] * bad


@pytest.mark.skipif(not (shutil.which("hipcc") or shutil.which("/opt/rocm/bin/hipcc")), reason="no hipcc")
def test_every_kernel_of_the_policy_operators_waits_for_operands():
    sources = [s for s in build.POLICY_SOURCES if s != "delta.hip"]

    def assembly(source):
        return subprocess.run([build._hipcc(), *(f for f in build.policy_flags(source) if f not in ("-fPIC", "-Wall")), "-w", "--cuda-device-only", "-S", "-o", "-", str(build.CSRC / source)],
                              capture_output=True, text=True, check=True).stdout

    with ThreadPoolExecutor(len(sources)) as pool:
        for source, text in zip(sources, pool.map(assembly, sources)):
            found = kernels(text)
            assert found, source
            for name, code in found.items():
                assert not early(code), (source, name, early(code)[:3])
