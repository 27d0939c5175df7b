"""The 8-bit products, as compiled: the tiles' K loop is one copy, adds every
product to the accumulator that it came from, moves none, touches no scratch
memory, waits for its loads with vmcnt(2) only, and nothing reads a sum before
the last products are through nor writes an operand right before its product;
the loads of the kernel of few rows leave in the order that its waits count
(test_gemm_isa.py has the same of bf16)."""
import functools
import os
import re
import shutil
import subprocess
import tempfile

import pytest

from conftest import ROOT
from test_gemm_isa import BAD, FLAGS, HIPCC, _body

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC),
                                reason="hipcc not installed")


@functools.lru_cache(maxsize=None)
def assembly():
    work = tempfile.mkdtemp(prefix="hk_int8_isa_")
    try:
        subprocess.run(
            [HIPCC, *FLAGS, "--save-temps", "-c",
             os.path.join(ROOT, "h3.c_amd", "csrc", "hk_int8.hip"), "-o",
             os.path.join(work, "x.o")], cwd=work, check=True,
            capture_output=True)
        asm, = (f for f in os.listdir(work)
                if f.endswith(".s") and "amdgcn" in f)
        return open(os.path.join(work, asm)).read().splitlines()
    finally:
        shutil.rmtree(work, ignore_errors=True)


def body_of(kernel):
    text = assembly()
    return _body(text, next(l for l in text if re.match(
        rf"_Z\d+{kernel}.*:", l)).split(":")[0])


def registers(operand):
    """{"v3", "v4"} of v[3:4]"""
    m = re.search(r"\b([av])(?:(\d+)|\[(\d+):(\d+)\])", operand)
    if not m:
        return set()
    first, last = (m[2], m[2]) if m[2] else (m[3], m[4])
    return {m[1] + str(i) for i in range(int(first), int(last) + 1)}


@pytest.mark.parametrize("jb", [4, 5, 6, 7, 8])
@pytest.mark.parametrize("epi", [0, 1, 3, 4, 5])
def test_k_loop(epi, jb):
    body = body_of(f"hk_int8_gemmILi{epi}ELb0ELi{jb}EE")
    mfma = [i for i, l in enumerate(body) if "v_mfma_" in l]
    assert len(mfma) == 16 * jb and not [l for l in body if "scratch_" in l]
    for i in mfma:
        dst, _, _, add = re.search(r"v_mfma_i32_16x16x64_i8 (.*)",
                                   body[i])[1].split("//")[0].split(", ")
        assert dst == add.strip(), body[i]
    back = next(i for i in range(mfma[-1], len(body))
                if body[i].strip().startswith("s_cbranch"))
    loop = body[mfma[0]:back]
    assert not [l for l in loop if BAD.search(l)]
    assert [l for l in loop if "vmcnt" in l] == [
        l for l in loop if re.search(r"s_waitcnt\b.*vmcnt\(2\)", l)]
    assert len([l for l in loop
                if re.search(r"buffer_load_dword\b.*\blds\b", l)]) == 2
    # 16 wait states before anything reads an accumulator, two between a vector
    # instruction and the MFMA that reads its result: the compiler counts none
    # for an MFMA in inline assembly
    after = [l.strip() for l in body[mfma[-1] + 1:]]
    read = next(i for i, l in enumerate(after) if re.match(
        r"(v_accvgpr|v_mov|global_store|ds_write|buffer_store|v_\w+ .*\ba\d)",
        l))
    assert "s_nop 15" in after[:read]
    code = [l.strip() for l in body if re.match(r"\s+[a-z]+_", l)]
    for i, line in enumerate(code):
        if "v_mfma_" not in line:
            continue
        sources = set().union(*map(registers, line.split(", ")[1:]))
        for before in code[i - 2:i]:
            if before.startswith("v_") and "v_mfma_" not in before:
                assert not registers(before.split(",")[0]) & sources, before


@pytest.mark.parametrize("gated", [0, 1])
@pytest.mark.parametrize("mb", [1, 2, 3, 4])
def test_loads_of_few_rows_leave_in_the_order_its_waits_count(mb, gated):
    body = body_of(f"hk_int8_skinnyILi{mb}ELb{gated}EE")
    loads = [(i, "X" if re.search(r"\blds\b", l) else "W")
             for i, l in enumerate(body) if "buffer_load_" in l]
    step = "X" * mb + "WWWW"
    assert "".join(w for _, w in loads) == 7 * step
    mfma = [i for i, l in enumerate(body) if "v_mfma_" in l]
    assert len(mfma) == 7 * 4 * mb
    turn = body[mfma[0]:mfma[4 * 4 * mb - 1]]
    assert not [l for l in turn if "s_cbranch" in l or "global_" in l]
    assert not [l for l in body if "scratch_" in l]
    asm = re.findall(r"#ASMSTART\n\s*s_waitcnt vmcnt\((\d+)\)",
                     "\n".join(body))
    assert [int(w) for w in asm] == [4 + 2 * (mb + 4)] * 4 + [
        4 + (2 - d) * (mb + 4) for d in range(3)] + [0]
