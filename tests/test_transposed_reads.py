"""The transposing V^T reads are pairs in one asm statement: the second one's
address must not lie in the registers that the first one fills, which it would
read while that load is on its way.  Nothing but the outputs' early clobber
keeps the register allocator from it where the address is not used again."""
import os
import re
import shutil
import subprocess
import tempfile

import pytest

from conftest import ROOT
from test_attn_isa import FLAGS, HIPCC, _regs

READ = re.compile(r"ds_read_b64_tr_b16 (v\[\d+:\d+\]), (v\d+)")
CSRC = os.path.join(ROOT, "h3.c_amd", "csrc")
SOURCES = {"hk_attn.hip": FLAGS,
           "hk_packed.hip": [f for f in FLAGS if f != "-fno-honor-nans"]}


def overwritten(body):
    """The lines of a second read whose address its pair's first one fills."""
    reads = [(i, _regs(m.group(1)), _regs(m.group(2)))
             for i, m in ((i, READ.search(l)) for i, l in enumerate(body)) if m]
    return [body[b[0]] for a, b in zip(reads, reads[1:])
            if b[0] == a[0] + 1 and b[2] & a[1]]


def test_the_walk_sees_an_address_that_is_overwritten():
    first = "\tds_read_b64_tr_b16 v[10:11], v10 offset:0"
    assert overwritten([first, "\tds_read_b64_tr_b16 v[12:13], v10 offset:8"])
    assert not overwritten([first.replace(", v10", ", v9"),
                            "\tds_read_b64_tr_b16 v[12:13], v9 offset:8"])


@pytest.mark.parametrize("name", SOURCES)
def test_outputs_of_the_first_read_are_early_clobbers(name):
    """Also in the headers that hold the reads."""
    for part in [name] + re.findall(r'#include "(hk_\w+\.h)"', open(
            os.path.join(CSRC, name)).read()):
        text = open(os.path.join(CSRC, part)).read()
        for block in re.findall(r"asm volatile\((.*?)\);", text, re.S):
            if block.count("ds_read_b64_tr_b16") > 1:
                assert '"=v"' not in block and '"=&v"' in block, (part, block)


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not installed")
@pytest.mark.parametrize("name", SOURCES)
def test_no_address_is_overwritten(name):
    work = tempfile.mkdtemp(prefix="hk_reads_isa_")
    try:
        subprocess.run([HIPCC, *SOURCES[name], "--save-temps", "-c",
                        os.path.join(CSRC, name), "-o",
                        os.path.join(work, "x.o")], cwd=work, check=True,
                       capture_output=True)
        asm, = (f for f in os.listdir(work)
                if f.endswith(".s") and "amdgcn" in f)
        body = open(os.path.join(work, asm)).read().splitlines()
    finally:
        shutil.rmtree(work, ignore_errors=True)
    assert sum("ds_read_b64_tr_b16" in l for l in body) > 100
    assert not overwritten(body)
