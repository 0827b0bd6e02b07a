"""The asm statements of the gradients' tiles.  Each that loads to LDS waits itself for the scalar registers it reads, whatever the compiler puts in front of it: a reload of a spilled word of
its buffer among them.  The MFMAs' operands are not written by a vector instruction right before, which the compiler does not look after either.  Runs without a GPU."""
import glob
import os
import re
import shutil
import subprocess

import pytest
from test_kernel_asm_host import KERNELS, MEMORY, OBJDUMP, OBJECTS, ROOT, WAIT_STATES, wait_states

from flux_amd import build

SOURCE = os.path.join(KERNELS, "grouped_gemm_grad_tiles.hip")
TILES = [o for o in OBJECTS if os.path.basename(o) == "grouped_gemm_grad_tiles.o"]


def statements(text):
    """The instructions of every asm statement of preprocessed source."""
    for found in re.finditer(r"asm volatile\s*\(", text):
        literals, at = [], found.end()
        while True:  # adjacent literals, up to the first colon or the end
            one = re.compile(r'\s*"((?:[^"\\]|\\.)*)"').match(text, at)
            if not one:
                break
            literals.append(one.group(1))
            at = one.end()
        yield [i.strip() for i in "".join(literals).replace("\\t", " ").split("\\n") if i.strip()]


def too_early(lines):
    """A load before which the statement itself has fewer than five wait states."""
    loads = [n for n, i in enumerate(lines) if i.startswith(MEMORY)]
    return bool(loads) and sum(wait_states(i) for i in lines[:loads[0]]) < WAIT_STATES


def test_the_scan_of_statements():
    one = 'asm volatile("buffer_load_dwordx4 %0, %1, 0 offen lds" : : "v"(off), "s"(rsrc) : "memory");'
    two = 'asm volatile("s_add_u32 m0, %0, %1\\n\\ts_nop 3\\n\\t" "buffer_load_ubyte" " %2, %3, 0 offen lds" : : "s"(base));'
    assert [too_early(s) for s in statements(one + two)] == [True, False]
    assert [too_early(s) for s in statements(two.replace("s_nop 3", "s_nop 2"))] == [True]


@pytest.mark.skipif(not os.path.exists(build.HIPCC), reason="needs hipcc")
def test_loads_to_lds_wait_in_their_statements():
    flags = [f for f in build.HIP_FLAGS if not f.startswith("-O")]
    text = subprocess.run([build.HIPCC, *flags, "-E", "--cuda-device-only", SOURCE], check=True, capture_output=True, text=True, cwd=ROOT).stdout
    found = [s for s in statements(text) if any(i.startswith(MEMORY) for i in s)]
    assert len(found) >= 2 and all("lds" in i for s in found for i in s if i.startswith(MEMORY))
    assert [s for s in found if too_early(s)] == []


REGISTERS = re.compile(r"\b([va])(\d+)\b|\b([va])\[(\d+):(\d+)\]")


def vectors(operands):
    out = set()
    for kind, one, kinds, first, last in REGISTERS.findall(operands):
        out |= {(kind, int(one))} if kind else {(kinds, r) for r in range(int(first), int(last) + 1)}
    return out


def mfma_too_close(lines):
    """MFMAs, in layout order, that read a register which a vector instruction wrote less than two wait states before."""
    now, written, found, seen = 0, {}, [], 0
    for line in lines:
        if not line.startswith("\t"):
            written = {}
            continue
        instruction = line.split("//")[0].strip()
        op, _, operands = instruction.partition(" ")
        to, _, rest = operands.partition(",")
        if op.startswith("v_mfma"):
            seen += 1
            found += [instruction for r in vectors(rest) if now - written.get(r, -9) - 1 < 2]
        elif op.startswith("v_"):
            written.update({r: now for r in vectors(to)})
        now += wait_states(instruction)
    return found, seen


def test_the_scan_of_mfmas():
    code = ["\tv_mov_b32_e32 v5, v9\n", "\ts_nop 0\n", "\tv_mfma_f32_16x16x32_bf16 a[0:3], v[4:7], v[8:11], a[0:3]\n"]
    assert len(mfma_too_close(code)[0]) == 1 and mfma_too_close([code[0], "\ts_nop 1\n", code[2]]) == ([], 1)


@pytest.mark.skipif(OBJDUMP is None or not TILES, reason="needs llvm-objdump and built objects")
def test_operands_of_mfmas_as_built(tmp_path):
    copy = shutil.copy(TILES[0], tmp_path)
    subprocess.run([OBJDUMP, "--offloading", copy], check=True, capture_output=True)
    for code in glob.glob(copy + ".*gfx950"):
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--mcpu=gfx950", code], check=True, capture_output=True, text=True).stdout
        found, seen = mfma_too_close(text.splitlines(True))
        assert seen >= 64 and found == []
