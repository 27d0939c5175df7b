"""The 8-bit products and gated block at shapes that are cut along K, where the
pieces' sums find no room (small_memory.cpp): the same bits, uncut; and the
attention of many rows. test_int8_routes.py holds each to its kernel."""
import shutil

import pytest

from test_no_scratch_gpu import run

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not shutil.which("g++"),
                                                  reason="needs g++")]

# of test_int8_kernels_gpu.py's: the kernel that runs then, hk_int8_ left out.
# Few rows' pieces fit what a context has from its start, if it finds that.
WHOLE = {
    (243, 2885, 1048): "skinny<1, false>", (327, 5013, 1905): "skinny<4, false>",
    (293, 4031, 12329): "gemm<0, false, 5>",
    (466, 4852, 8611): "gemm<0, false, 8>",
}
BLOCKS = {
    (1096, 5022, 202): "skinny<3, true>", (1473, 7142, 150): "skinny<4, true>",
    (284, 4274, 6136): "gemm<1, false, 5>",
    (1029, 4946, 1869): "gemm<1, false, 8>",
}
ROOM = {s: 4 << 20 if "skinny" in k else 16 << 20  # for the hidden values
        for s, k in BLOCKS.items()}

BARE = """
limit(0)
bare = h3hip.Gpu()  # which finds no scratch
limit()
y, z = (g.new_bf16(m * n) for g in (bare, gpu))
"""


@pytest.mark.parametrize("m,k,n", WHOLE)
def test_product(m, k, n):
    run(f"""
import test_int8_gpu as t
m, k, n = {m}, {k}, {n}
p = t.Product(m, k, n)
{BARE}
for g, out, size in ((bare, y, 0), (gpu, z, -1)):
    sides = [t.quantize(g, a, r, k) for a, r in ((p.x, m), (p.w, n))]
    limit(size)
    g.run("h3_hip_linear_int8_bf16", out, *sides, None, m, k, n)
    limit()
got = bare.read_bf16(y)
assert np.array_equal(got, gpu.read_bf16(z))
want, bound = t.io.product(*p.sides())
ro.check(got.reshape(m, n), want, t.io.rounded(want, bound))
""")


@pytest.mark.parametrize("m,k,h", BLOCKS)
def test_gated_block(m, k, h):
    run(f"""
import test_int8_gpu as t
m, k, h, n = {m}, {k}, {h}, 130
rng = np.random.default_rng((m, k, h))
sides = [(t.rand_bf16(rng, r * c, std), r, c) for r, c, std in (
    (m, k, 1), (2 * h, k, 1.5 * k ** -0.5), (n, h, h ** -0.5))]
{BARE}
for g, out, size in ((bare, y, {ROOM[m, k, h]}), (gpu, z, -1)):
    made = [t.quantize(g, *s) for s in sides]
    limit(size)
    g.run("h3_hip_mlp_int8_bf16", out, *made, m, k, h, n)
    limit()
got = bare.read_bf16(y)
assert np.array_equal(got, gpu.read_bf16(z))
want, bound = t.io.mlp(*(t.io.rows_of(ro.wide(b, r, c)) for b, r, c in sides))
ro.check(got.reshape(m, n), want, t.io.rounded(want, bound))
""")


def test_attention_of_many_rows():
    """Items that the plan cuts run whole, in a context that has room for the
    unpacked keys and values alone."""
    run("""
import test_kv8_gpu as t
limit(0)
bare = h3hip.Gpu()
limit()
a = t.Case(bare, [16384], [9720], 8, 8, 128)  # whole items
b = t.Case(bare, [128], [9720], 8, 8, 128)
def plan(c):
    return bare.sdpa_packed_plan(c.qf, c.qn, c.kf, c.kn, 8, 8, 128)
q = [bare.bf16(c.q) for c in (a, b)]
y = [bare.new_bf16(c.rows * 1024) for c in (a, b)]
plans = [plan(c) for c in (a, b)]
got = []
for i, size in ((0, -1), (1, 0), (1, -1)):
    limit(size)
    bare.run("h3_hip_sdpa_packed_int8_bf16", y[i], q[i], 0, 1024, (a, b)[i].kv.t,
             plans[i], b.scale)
    limit()
    got.append(bare.read_bf16(y[i]))
want, bound, _ = t.io.attention(ro.wide(b.q, 128, 8, 128), b.kv.wide,
                                [(0, 128, 0, 9720)], 8, 8, 128,
                                float(np.float32(b.scale)))
for g in got[1:]:
    ro.check(g.reshape(want.shape), want, bound)
# another order of sums
assert not np.array_equal(got[1], got[2])
""")
