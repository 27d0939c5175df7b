"""The GEMM with adapters, as compiled: its K loop is one copy, moves no
accumulator, touches no scratch memory and waits for its loads with vmcnt(2)
only, as test_gemm_isa.py holds the plain GEMM's to."""
import os
import re
import shutil
import subprocess
import tempfile

import pytest

from conftest import ROOT
from test_gemm_isa import BAD, FLAGS, HIPCC, _body

INSTANCES = [(epi, jb) for epi in (0, 3, 5) for jb in (4, 5, 6, 7, 8)
             if (epi, jb) != (3, 7)]


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not installed")
def test_k_loop_with_adapters():
    work = tempfile.mkdtemp(prefix="hk_lora_isa_")
    try:
        subprocess.run(
            [HIPCC, *FLAGS, "--save-temps", "-c",
             os.path.join(ROOT, "h3.c_amd", "csrc", "hk_lora.hip"), "-o",
             os.path.join(work, "x.o")], cwd=work, check=True,
            capture_output=True)
        asm, = (f for f in os.listdir(work)
                if f.endswith(".s") and "amdgcn" in f)
        text = open(os.path.join(work, asm)).read().splitlines()
    finally:
        shutil.rmtree(work, ignore_errors=True)
    for epi, jb in INSTANCES:
        body = _body(text, f"_Z12hk_gemm_loraILi{epi}ELb0ELi{jb}EEv"
                           "12hk_gemm_args11hk_lora_ext")
        mfma = [i for i, l in enumerate(body) if "v_mfma_" in l]
        assert len(mfma) == 16 * jb, (epi, jb, len(mfma))
        back = next(i for i in range(mfma[-1], len(body))
                    if body[i].strip().startswith("s_cbranch"))
        loop = body[mfma[0]:back]
        assert not [l for l in loop if BAD.search(l)], (epi, jb)
        assert [l for l in loop if "vmcnt" in l] == [
            l for l in loop if re.search(r"s_waitcnt\b.*vmcnt\(2\)", l)]
        assert len([l for l in loop if re.search(
            r"buffer_load_dword\b.*\blds\b", l)]) == 2
        # no loop over the lanes' descriptors
        assert not [l for l in loop if "readfirstlane" in l], (epi, jb)
