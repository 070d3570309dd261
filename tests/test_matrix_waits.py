"""The compiler's waits behind matrix instructions, checked in the assembly of this build's own
kernels. A result of a four-pass matrix instruction may be read by another kind of instruction
after eight wait states and overwritten after seven; nothing in the hardware waits. The compiler
puts the waits in, but has been seen to leave one out where a branch lies between a matrix
instruction and the use of its result (values came out half written). Every path from every
matrix instruction is followed here, through branches, until its result is safe."""
import re
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from zeno_amd import build

READ, WRITE = 8, 7


def registers(text):
    found = set()
    for m in re.finditer(r"\b([va])\[(\d+):(\d+)\]|\b([va])(\d+)\b", text):
        found |= {(m[1], i) for i in range(int(m[2]), int(m[3]) + 1)} if m[1] else {(m[4], int(m[5]))}
    return found


def kernels(assembly):
    """{kernel: [(op, operands) or ("label", name)]}"""
    found, current = {}, None
    for line in assembly.splitlines():
        line = line.split(";")[0].rstrip()
        if m := re.match(r"^(_Z\S+):", line):
            current = found.setdefault(m[1], [])
        elif current is not None and (m := re.match(r"^(\.LBB\S+):", line)):
            current.append(("label", m[1]))
        elif current is not None and re.match(r"^\s+[a-z]", line) and not line.strip().startswith("."):
            op, _, operands = line.strip().partition(" ")
            current.append((op, operands.strip()))
    return {k: v for k, v in found.items() if any("mfma" in op for op, _ in v)}


def early(code):
    """Instructions that touch a matrix result before it is safe: (matrix instruction, user, wait states)."""
    at = {x: i for i, (op, x) in enumerate(code) if op == "label"}
    found = []
    for i, (op, operands) in enumerate(code):
        if "mfma" not in op:
            continue
        result = registers(operands.split(",")[0])
        paths, seen = [(i + 1, 0)], set()
        while paths:
            j, states = paths.pop()
            while j < len(code) and states < READ and (j, states) not in seen:
                seen.add((j, states))
                o, x = code[j]
                if o == "label":
                    j += 1
                    continue
                if o == "s_nop":
                    states += int(x, 0) + 1
                    j += 1
                    continue
                if "mfma" in o:  # chained results are the hardware's own matter
                    if registers(x.split(",")[0]) & result:
                        break
                elif o.startswith(("v_", "ds_", "global_", "scratch_", "buffer_")):
                    first, _, rest = x.partition(",")
                    writes = o.startswith(("v_", "ds_read", "ds_bpermute", "global_load", "scratch_load", "buffer_load"))
                    read = registers(rest if writes else x) & result
                    if read or (writes and states < WRITE and registers(first) & result):
                        found.append((f"{op} {operands}", f"{o} {x}", states))
                        break
                elif o == "s_branch":
                    j, states = at[x], states + 1
                    continue
                elif o.startswith("s_cbranch"):
                    paths.append((at[x], states + 1))
                elif o == "s_endpgm":
                    break
                j, states = j + 1, states + 1
    return found


def test_the_check_sees_a_missing_wait():
    loop = """_Zk:
        v_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[8:11], v[0:3]
        s_cbranch_vccnz .LBB0_1
        s_nop 7
        v_add_f32_e32 v20, v0, v1
    .LBB0_1:
        v_mov_b32_e32 v21, v2
        s_endpgm""".replace("\n    .LBB", "\n.LBB")
    (code,) = kernels(loop).values()
    assert [(user, states) for _, user, states in early(code)] == [("v_mov_b32_e32 v21, v2", 1)]
    (code,) = kernels(loop.replace("v21, v2", "v21, v22")).values()
    assert not early(code)


@pytest.mark.skipif(not (shutil.which("hipcc") or shutil.which("/opt/rocm/bin/hipcc")), reason="no hipcc")
def test_every_kernel_of_the_policy_operators_waits():
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
