"""The 8-bit operators where the context's scratch cannot grow
(small_memory.cpp): the same results in larger pieces of work, or a refusal."""
import shutil

import pytest

from test_no_scratch_gpu import run

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not shutil.which("g++"),
                                                  reason="needs g++")]


@pytest.mark.parametrize("m,k,n", [(40, 7168, 640), (300, 5120, 2560),
                                   (2400, 2048, 2600)])
def test_product(m, k, n):
    """K whole, where its pieces' sums find no room."""
    run(f"""
import test_int8_gpu as t
p = t.Product({m}, {k}, {n})
sides = [t.quantize(gpu, a, r, {k}) for a, r in ((p.x, {m}), (p.w, {n}))]
y, got = gpu.new_bf16({m * n}), []
for size in (0, -1):
    limit(size)
    gpu.run("h3_hip_linear_int8_bf16", y, *sides, None, {m}, {k}, {n})
    got.append(gpu.read_bf16(y))
assert np.array_equal(*got)
want, bound = t.io.product(*p.sides())
ro.check(got[0].reshape({m}, {n}), want, t.io.rounded(want, bound))
""")


@pytest.mark.parametrize("qn,kn", [([1] * 4, [6144, 5000, 0, 1]),
                                   ([2], [9720])])
def test_attention_of_few_rows(qn, kn):
    """Items that the plan cuts run whole."""
    run(f"""
import test_kv8_gpu as t
a = t.Case(gpu, {qn}, {kn}, 16, 4, 128)
q, plan = gpu.bf16(a.q), gpu.sdpa_packed_plan(
    a.qf, a.qn, a.kf, a.kn, a.heads, a.kv_heads, a.dim)
y = gpu.new_bf16(a.rows * a.heads * a.dim)
want, bound, covered = t.io.attention(
    ro.wide(a.q, a.rows, a.heads, a.dim), a.kv.wide,
    list(zip(a.qf, a.qn, a.kf, a.kn)), a.heads, a.kv_heads, a.dim,
    float(np.float32(a.scale)))
for size in (0, -1):
    limit(size)
    gpu.run("h3_hip_sdpa_packed_int8_bf16", y, q, 0, a.stride, a.kv.t, plan,
            a.scale)
    ro.check(gpu.read_bf16(y).reshape(want.shape)[covered], want[covered],
             bound[covered], f"limit {{size}}")
""")


def test_what_needs_scratch_is_refused():
    """The blocks of many rows, and the gated block's hidden values."""
    run("""
import test_int8_gpu as i, test_kv8_gpu as t
a = t.Case(gpu, [6144], [500], 8, 8, 64)  # items of 128 rows
m, k, h, n = 200, 300, 700, 128
rng = np.random.default_rng(0)
x, w1, w2 = (i.quantize(gpu, i.rand_bf16(rng, r * c), r, c)
             for r, c in ((m, k), (2 * h, k), (n, h)))
q, z = gpu.bf16(a.q), gpu.new_bf16(m * n)
plan = gpu.sdpa_packed_plan(a.qf, a.qn, a.kf, a.kn, a.heads, a.kv_heads, a.dim)
y = gpu.bf16(np.full(a.rows * a.heads * a.dim, i.MARK, np.uint16))
limit(0)
gpu.begin()
assert not gpu.L.h3_hip_sdpa_packed_int8_bf16(gpu.h, y, q, 0, a.stride, a.kv.t,
                                              plan, a.scale)
assert not gpu.L.h3_hip_mlp_int8_bf16(gpu.h, z, x, w1, w2, m, k, h, n)
assert gpu.error()
gpu.submit()
assert (gpu.read_bf16(y) == i.MARK).all()
limit()
a.check()
""")
