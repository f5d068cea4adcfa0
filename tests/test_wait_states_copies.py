"""Waits around the copies into LDS and the matrix instructions that are written in asm, in the built gfx950 code.
The compiler inserts what its own instructions need but cannot see into an asm block, so the disassembly of the whole
library is read, over all paths from an instruction that writes a register:

  * an SGPR written by a VALU instruction (a buffer's descriptor, made by v_readfirstlane, or one that comes back from
    a spill by v_readlane) is read by no memory instruction before five wait states have passed;
  * a register that a VALU instruction wrote is read by no matrix instruction before two have passed;
  * where matrix instructions are asm, their sums are touched by no other kind of instruction before they are there: a
    wait state a pass of four clocks, and four more.
"""
import concurrent.futures as cf
import glob
import multiprocessing
import os
import re
import subprocess

import pytest

from sparsesnn_amd import _lib
from tests.test_wait_states import OBJDUMP, _code, _sgprs, _vgprs, functions

MEMORY = ("buffer_", "global_", "flat_", "scratch_")
VALU_TO_MEMORY, VALU_TO_MATRIX = 5, 2


def _operands(text):
    name, _, rest = text.partition(" ")
    return name, re.split(r",(?![^\[]*\])", rest) if rest else []


def _is_matrix(name):
    return name.startswith(("v_mfma", "v_smfmac"))


def _writes_and_reads(name, ops):
    """Operands that a VALU or matrix instruction writes, and those that it reads."""
    if name.startswith("v_cmpx"):
        return [], ops
    if name.startswith(("v_swap", "v_permlane16_swap", "v_permlane32_swap")):
        return ops, ops
    n = 2 if "_co_" in name or name.startswith("v_div_scale") else 1
    return ops[:n], ops[n:]


def passes(name):
    """Passes of four clocks of the library's matrix instructions, rounded down: 16 x 16 x 32 of 16 bits, 16384 operations
    at 1024 a clock and SIMD (sparse ones do half of what their name says); x 128 of 8 bits, 65536 at 2048; 16 x 16 x 4
    of 32 bits, 2048 at 64."""
    m, n, k = map(int, re.search(r"(\d+)x(\d+)x(\d+)", name).groups())
    rate = 2048 if "f8f6f4" in name or name.startswith("v_smfmac") else 64 if re.search(r"x4(_f32|f32)", name) else 1024
    return max(1, 2 * m * n * k // rate // 4)


def _after(code, at, start, states):
    """The instructions within `states` wait states after instruction `start`, over all paths."""
    seen, work = {}, [(start + 1, 0)]
    while work:
        i, passed = work.pop()
        if i >= len(code) or passed >= states or seen.get(i, states) <= passed:
            continue
        seen[i] = passed
        name, _, rest = code[i][1].partition(" ")
        nxt = passed + (int(rest, 0) + 1 if name == "s_nop" else 1)
        if name == "s_endpgm":
            continue
        if code[i][2] is not None:
            work.append((at[code[i][2]], nxt))
        if name != "s_branch":
            work.append((i + 1, nxt))
    return seen


def hazards(code, sums=True):
    """(kind, writer, reader) of instructions that follow each other too closely, of one function; sums: of matrix
    instructions' sums too."""
    at = {a: i for i, (a, _, _) in enumerate(code)}
    found = []
    has_matrix = any(_is_matrix(t) for _, t, _ in code)
    for i, (_, text, _) in enumerate(code):
        name, ops = _operands(text)
        if not name.startswith("v_") or not ops:
            continue
        dst, _ = _writes_and_reads(name, ops)
        if _is_matrix(name):
            regs = _vgprs(dst[0])
            for j in _after(code, at, i, passes(name) + 4) if sums else ():
                other, rest = code[j][1].partition(" ")[::2]
                if not _is_matrix(other) and not other.startswith("s_") and _vgprs(rest) & regs:
                    found.append(("sums", text, code[j][1]))
            continue
        scalars = set().union(*(_sgprs(o) for o in dst)) if dst else set()
        if scalars:
            for j in _after(code, at, i, VALU_TO_MEMORY):
                other, rest = code[j][1].partition(" ")[::2]
                if other.startswith(MEMORY) and _sgprs(rest) & scalars:
                    found.append(("memory", text, code[j][1]))
        if has_matrix:
            regs = set().union(*(_vgprs(o) for o in dst)) if dst else set()
            for j in _after(code, at, i, VALU_TO_MATRIX) if regs else ():
                other, others = _operands(code[j][1])
                if _is_matrix(other) and set().union(*(_vgprs(o) for o in others[1:])) & regs:
                    found.append(("matrix", text, code[j][1]))
    return found


def _scan(path):
    found = []
    with subprocess.Popen([OBJDUMP, "-d", "--mcpu=gfx950", "--no-show-raw-insn", path], stdout=subprocess.PIPE,
                          text=True) as p:
        for name, code in functions(p.stdout):
            found += [(name, h) for h in hazards(code, "linear_tile" in name)]
    return p.returncode, found


@pytest.fixture(scope="module")
def findings(tmp_path_factory):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    tmp = tmp_path_factory.mktemp("lib")
    os.symlink(_lib.lib_path(), tmp / "lib.so")  # the code objects are extracted next to it
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp, check=True, stdout=subprocess.DEVNULL)
    objs = sorted(glob.glob(str(tmp / "lib.so.*gfx950")), key=os.path.getsize, reverse=True)
    assert objs
    with cf.ProcessPoolExecutor(4, mp_context=multiprocessing.get_context("spawn")) as ex:
        results = list(ex.map(_scan, objs))
    assert all(rc == 0 for rc, _ in results)
    return [h for _, found in results for h in found]


def _kinds(*texts):
    return [k for k, _, _ in hazards(_code(*texts))]


def test_hazards_finds_and_spares():
    copy = "buffer_load_dwordx4 v1, s[4:7], 0 offen lds"
    for write in ("v_readfirstlane_b32 s5, v3", "v_readlane_b32 s7, v3, 2"):
        assert _kinds(write, "s_mov_b32 m0, s9", "s_nop 0", copy) == ["memory"]
        assert _kinds(write, "s_mov_b32 m0, s9", "s_nop 2", copy) == ["memory"]
        assert not _kinds(write, "s_mov_b32 m0, s9", "s_nop 3", copy)
    assert not _kinds("v_readfirstlane_b32 s8, v3", copy) and not _kinds("s_mov_b32 s5, s9", copy)
    # by way of a branch
    assert _kinds("v_readfirstlane_b32 s5, v3", "s_cbranch_scc0 3", "s_nop 7", copy, "s_endpgm") == ["memory"]
    mma = "v_mfma_f32_16x16x32_f16 a[0:3], v[4:7], v[8:11], a[0:3]"
    assert _kinds("v_mov_b32_e32 v5, 0", "s_nop 0", mma) == ["matrix"]
    assert not _kinds("v_mov_b32_e32 v5, 0", "s_nop 1", mma) and not _kinds("v_mov_b32_e32 v12, 0", mma)
    read = "v_accvgpr_read_b32 v1, a2"
    assert _kinds(mma, mma, read) == ["sums", "sums"] and _kinds(mma, "s_nop 6", read) == ["sums"]
    assert not _kinds(mma, "s_nop 7", read) and not _kinds(mma, "v_accvgpr_read_b32 v1, a4")
    long = "v_mfma_f32_16x16x128_f8f6f4 a[0:3], v[4:11], v[12:19], a[0:3]"
    assert _kinds(long, "s_nop 10", read) == ["sums"] and not _kinds(long, "s_nop 11", read)


def test_library_waits_for_descriptors(findings):
    found = [f for f in findings if f[1][0] == "memory"]
    assert not found, f"{len(found)} memory instructions too close to a VALU write of an SGPR, first {found[:3]}"


def test_library_waits_for_operands_of_matrix_instructions(findings):
    found = [f for f in findings if f[1][0] == "matrix"]
    assert not found, f"{len(found)} matrix instructions too close to a VALU write, first {found[:3]}"


def test_library_waits_for_sums(findings):
    found = [f for f in findings if f[1][0] == "sums"]
    assert not found, f"{len(found)} uses of sums too close to their matrix instruction, first {found[:3]}"
