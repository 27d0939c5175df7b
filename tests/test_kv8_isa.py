"""The attention kernels over the 8-bit cache, as compiled: what runs over
unpacked rows waits for its transposed reads as its bf16 kin does
(test_packed_plan.py), and none uses scratch memory."""
import os
import shutil
import subprocess
import tempfile

import pytest

from conftest import ROOT
from test_attn_isa import HIPCC, _offenders
from test_gemm_isa import FLAGS

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC),
                                reason="hipcc not installed")


def bodies(source, kernel, flags):
    work = tempfile.mkdtemp(prefix="hk_kv8_isa_")
    try:
        subprocess.run(
            [HIPCC, *FLAGS, "-mllvm", "-amdgpu-mfma-vgpr-form", *flags,
             "--save-temps", "-c", os.path.join(ROOT, "h3.c_amd", "csrc",
                                                source), "-o",
             os.path.join(work, "x.o")], cwd=work, check=True,
            capture_output=True)
        asm, = (f for f in os.listdir(work)
                if f.endswith(".s") and "amdgcn" in f)
        text = open(os.path.join(work, asm)).read().splitlines()
    finally:
        shutil.rmtree(work, ignore_errors=True)
    found, name = {}, None
    for line in text:
        if line.startswith(kernel) and ":" in line:
            name = line.split(":")[0]
            found[name] = []
        elif name and line.startswith(".Lfunc_end"):
            name = None
        elif name:
            found[name].append(line)
    return found


def test_many_rows():
    found = bodies("hk_packed.hip", "_Z15hk_packed_codesI",
                   ["-fno-signed-zeros", "-fno-trapping-math",
                    "-fassociative-math", "-freciprocal-math"])
    assert len(found) == 3
    for name, body in found.items():
        assert any("ds_read_b64_tr_b16" in l for l in body), name
        assert not _offenders(body), (name, _offenders(body)[:3])
        assert not [l for l in body if "scratch_" in l], name


def test_few_rows():
    found = bodies("hk_kv8.hip", "_Z10hk_kv8_fewI", [])
    assert len(found) == 4
    for name, body in found.items():
        assert not [l for l in body if "scratch_" in l], name
