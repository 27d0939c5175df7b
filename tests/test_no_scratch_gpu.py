"""The operators of packed requests where the context's scratch cannot grow
(small_memory.cpp): the same results, in larger pieces of work."""
import os
import shutil
import subprocess
import sys
import tempfile

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

START = """
import ctypes, sys
small = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
sys.path[:0] = sys.argv[2:]
import h3hip, numpy as np
import requests_oracle as ro
gpu = h3hip.Gpu()
def limit(size=-1):
    small.small_memory(ctypes.c_size_t(size))
limit(0)
assert not gpu.L.h3_gpu_tensor_new_bf16(gpu.h, 1 << 28), "not the limit's"
limit()
"""


def run(code):
    work = tempfile.mkdtemp(prefix="small_memory_")
    try:
        lib = os.path.join(work, "libsmall_memory.so")
        subprocess.run(["g++", "-O1", "-fPIC", "-shared", os.path.join(
            ROOT, "tests", "small_memory.cpp"), "-ldl", "-o", lib], check=True)
        done = subprocess.run(
            [sys.executable, "-c", START + code + "\nprint('fine')", lib] + [
                os.path.join(ROOT, d) for d in ("h3.c_amd", "oracle", "tests")],
            capture_output=True, text=True, timeout=100)
    finally:
        shutil.rmtree(work, ignore_errors=True)
    assert done.returncode == 0 and "fine" in done.stdout, done.stderr[-2000:]


@pytest.mark.skipif(not shutil.which("g++"), reason="needs g++")
@pytest.mark.parametrize("qn,kn,heads,kv_heads,dim", [
    ([1] * 8, [6144, 5000, 1, 0, 4097, 700, 9720, 6143], 64, 8, 128),
    ([128, 40], [9720, 9000], 32, 32, 64), ([300], [3000], 12, 4, 96)])
def test_packed_attention(qn, kn, heads, kv_heads, dim):
    """Items that the plan cuts run whole."""
    run(f"""
import test_packed_gpu as t
a = t.Case(31, {qn}, {kn}, {heads}, {kv_heads}, {dim}, gap=2)
plan = gpu.sdpa_packed_plan(a.qf, a.qn, a.kf, a.kn, a.heads, a.kv_heads, a.dim)
n = a.rows * a.heads * a.dim
y = gpu.bf16(np.full(n, 0x4141, np.uint16))
q, kv = gpu.bf16(a.q), gpu.bf16(a.kvs)
want, bound, covered = a.want()
for size in (0, -1):  # without and with scratch
    limit(size)
    gpu.run("h3_hip_sdpa_packed_bf16", y, q, 0, a.qs, kv, 0, kv,
            a.kv_heads * a.dim, a.ks, plan, a.scale)
    got = gpu.read_bf16(y).reshape(a.rows, a.heads, a.dim)
    ro.check(got[covered], want[covered], bound[covered], f"limit {{size}}")
    assert (got[~covered] == 0x4141).all()
""")


@pytest.mark.skipif(not shutil.which("g++"), reason="needs g++")
@pytest.mark.parametrize("rows,k,n", [(128, 64, 36000), (5, 128, 140000),
                                      (300, 320, 20480), (1000, 320, 5120)])
def test_adapters(rows, k, n):
    """Tiles where the skinny GEMM's sums of the whole output find no room."""
    run(f"""
import test_lora_gpu as t
a = t.make(32, t.spread({rows}, 3, 1), [16, 40, 3], {k}, {n})
x, w, b, ids = gpu.bf16(a["x"]), gpu.bf16(a["w"]), gpu.bf16(a["b"]), gpu.u32(
    a["ids"])
table, y = t.table_of(gpu, a), gpu.new_bf16({rows * n})
for act, name in ((False, ""), (True, "gelu_")):
    want, bound = ro.lora(act=act, **a)
    for size in (8 << 20, -1):  # room for the halves alone, and for all
        limit(size)
        gpu.run("h3_hip_linear_lora_" + name + "bf16", y, x, w, b, table, ids,
                {rows}, {k}, {n})
        ro.check(gpu.read_bf16(y), want, bound, f"limit {{size}}")
""")
