"""The wait states that the hardware does not keep by itself, in the built kernels' own assembly.

A vector-memory instruction reads its buffer descriptor (and scalar offset) from scalar registers. A vector instruction
that wrote one of them (v_readlane, v_readfirstlane, a comparison) has to be 5 wait states away; the compiler keeps the
distance for the loads that it emits itself, but does not look into inline assembly. A load that lands in LDS takes its place
from M0, which has to be written 1 wait state before. One instruction is one wait state, ``s_nop n`` is n + 1.
"""
import re
import shutil
import subprocess

import pytest

from distributed_llm_training_gpu_manager_amd import _native

OBJDUMP = shutil.which("llvm-objdump", path="/opt/rocm/llvm/bin") or shutil.which("llvm-objdump")
APART = 5


def scalars(operand):
    """Numbers of the scalar registers of an operand: s7 -> {7}, s[4:7] -> {4, 5, 6, 7}, anything else -> {}."""
    m = re.fullmatch(r"s(?:(\d+)|\[(\d+):(\d+)\])", operand)
    if not m:
        return set()
    return {int(m[1])} if m[1] else set(range(int(m[2]), int(m[3]) + 1))


def too_close(lines):
    """(line, wait states) of every buffer instruction that reads a scalar register sooner than APART wait states after a
    vector instruction wrote it, or M0 in the very next one. Walks the text in its order: a jump only adds distance."""
    found, written, now, m0 = [], {}, 0, -1  # written: register -> time of the last vector write
    for line in lines:
        text = line.split("//")[0].strip()
        m = re.match(r"([a-z]\w+)\s*(.*)", text)
        if not m or text.endswith(":"):
            continue
        name, args = m[1], [a.strip().split(" ")[0] for a in m[2].split(",")]
        if name.startswith("buffer_"):
            near = [now - written[s] for a in args for s in scalars(a) if s in written and now - written[s] < APART]
            if "lds" in text.split() and m0 == now:
                near.append(0)
            if near:
                found.append((text, min(near)))
        if name.startswith("v_"):
            for a in args[:2]:  # the destination, and a carry's behind it
                if a is args[0] or "_co_" in name or name.startswith("v_div_scale"):
                    written.update((s, now + 1) for s in scalars(a))
        elif args:
            for s in scalars(args[0]):
                written.pop(s, None)  # written by the scalar unit since: the hardware waits for that
        if args[0] == "m0":
            m0 = now + 1
        now += int(args[0], 0) + 1 if name == "s_nop" else 1
    return found


def test_the_walk_counts_wait_states():
    load = "buffer_load_dwordx4 v1, s[24:27], 0 offen lds"
    body = ["v_readlane_b32 s26, v9, 3", "s_mov_b32 m0, s4"]
    assert too_close([*body, "s_nop 0", load]) == [(load, 2)]
    assert too_close([*body, "s_nop 2", load]) == [(load, 4)]
    assert not too_close([*body, "s_nop 3", load])
    assert not too_close(["v_readlane_b32 s28, v9, 3", load]) and not too_close(["v_readlane_b32 s26, v9, 3", "s_mov_b32 s26, s1", load])
    assert too_close(["s_add_u32 m0, m0, 0x1000", load]) == [(load, 0)] and not too_close(["s_mov_b32 m0, s4", "s_nop 0", load])
    assert too_close(["v_cmp_lt_i32_e64 s[24:25], v0, v1", "s_nop 3", load]) == [(load, 4)]


@pytest.mark.skipif(OBJDUMP is None or not _native.HIP_LIB.exists(), reason="needs llvm-objdump and the built library")
def test_descriptors_are_written_in_time(tmp_path):
    shutil.copy(_native.HIP_LIB, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    objects = sorted(tmp_path.glob("lib.so.*gfx950*"))
    assert objects
    loads, found = 0, []
    for o in objects:
        asm = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", str(o)], check=True, capture_output=True, text=True).stdout
        lines = asm.splitlines()
        loads += sum("buffer_load" in x and " lds" in x for x in lines)
        found += too_close(lines)
    assert loads > 100  # the attention and matrix kernels stage their tiles by LDS-DMA
    assert not found, f"{len(found)} of {loads} read a descriptor too early, the first: {found[:3]}"
