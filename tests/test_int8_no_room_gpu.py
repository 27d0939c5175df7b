"""The 8-bit products and gated block at shapes that are cut along K, where the
pieces' sums find no room (small_memory.cpp): the same bits, uncut.
test_int8_routes.py holds each to its kernel."""
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
