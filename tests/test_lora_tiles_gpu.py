"""Projections with adapters that go over the GEMM's tiles, every kernel of that
way, against the same in 64 bits at the bounds of requests_oracle.
test_lora_routes.py holds each shape to the kernels named here."""
import shutil

import numpy as np
import pytest

import requests_oracle as ro
from conftest import to_f32
from test_lora_gpu import blocks, check, make, ro_bits, run, spread, table_of
from test_no_scratch_gpu import run as run_small

pytestmark = pytest.mark.gpu

# (rows, K, N, ranks): the first product's <16-rank blocks, 16-row blocks> and
# the GEMM's <epilogue, 32-row blocks of a tile>, 3 of a launch cut along K
SHAPES = {
    (1645, 64, 4056, (16,)): ("low<1, 2>", "gemm<0, 8>"),
    (7554, 512, 1324, (9, 2)): ("low<1, 4>", "gemm<0, 6>"),
    (5244, 64, 1696, (32, 8)): ("low<2, 2>", "gemm<0, 8>"),
    (7725, 320, 1684, (32, 8)): ("low<2, 4>", "gemm<0, 8>"),
    (549, 64, 12720, (33,)): ("low<4, 2>", "gemm<0, 8>"),
    (9045, 64, 1076, (128, 5)): ("low<4, 4>", "gemm<0, 8>"),
    (6413, 768, 1236, (32, 8)): ("low<2, 2>", "gemm<0, 4>"),
    (2669, 768, 2944, (200,)): ("low<4, 4>", "gemm<0, 4>"),
    (1177, 768, 6600, (64, 16)): ("low<4, 2>", "gemm<0, 5>"),
    (534, 320, 16808, (128, 5)): ("low<4, 2>", "gemm<0, 6>"),
    (386, 512, 21528, (16,)): ("low<1, 2>", "gemm<0, 7>"),
    (284, 5120, 6428, (33,)): ("low<4, 2>", "gemm<3, 5>"),
    (374, 5120, 6972, (32, 8)): ("low<2, 2>", "gemm<3, 6>"),
    (2725, 2560, 1432, (64, 16)): ("low<4, 4>", "gemm<3, 8>"),
}
# several adapters over each tile height, whole and cut
SEVEN = (4, 16, 0, 33, 64, 8, 128)
SEVERAL = {
    (2601, 64, 2872): SEVEN, (2669, 768, 2944): SEVEN,
    (1177, 768, 6600): SEVEN, (534, 320, 16808): SEVEN,
    (386, 512, 21528): SEVEN, (284, 5120, 6428): (16, 8, 33, 64),
    (374, 5120, 6972): (16, 8, 33, 64), (562, 2560, 9664): SEVEN,
    (2725, 2560, 1432): SEVEN,
}
# two adapters for every three rows of a tile, and more
MANY = [(8553, 1024, 992), (6773, 512, 1604), (5586, 128, 5488)]
CUT = (374, 5120, 6972)
SMALL = (2601, 64, 2872)


def parts(rows, adapters):
    """Runs of every adapter and of none whose ends lie within tiles."""
    count = adapters + 1
    sizes = [rows * (i + 1) // count - rows * i // count
             for i in range(count)]
    return blocks(*((n, i if i < adapters else ro.NONE)
                    for i, n in enumerate(sizes)))


@pytest.mark.parametrize("act", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_every_kernel(gpu, shape, act):
    rows, k, n, ranks = shape
    check(gpu, make(rows, parts(rows, len(ranks)), ranks, k, n, scale=0.02),
          act)


@pytest.mark.parametrize("act", [False, True])
@pytest.mark.parametrize("shape", SEVERAL)
def test_adapters_in_any_order(gpu, shape, act):
    """All in every tile, and rows of none."""
    rows, k, n = shape
    ranks = SEVERAL[shape]
    check(gpu, make(rows + 1, spread(rows, len(ranks), rows), ranks, k, n,
                    bias=not act, scale=0.02), act)


@pytest.mark.parametrize("rank", [1, 2, 7, 8, 9, 15, 16, 17, 24, 31, 32, 33, 40,
                                  63, 64, 65, 96, 127, 128, 129, 200, 320])
def test_ranks(gpu, rank):
    rows, k, n = SMALL
    check(gpu, make(rank, parts(rows, 2), [rank, 8], k, n))


@pytest.mark.parametrize("rank", [4, 33, 64, 1024])
def test_ranks_of_a_cut_launch(gpu, rank):
    rows, k, n = CUT
    check(gpu, make(rank, parts(rows, 2), [rank, 8], k, n, scale=0.02))


@pytest.mark.parametrize("shape", MANY)
def test_an_adapter_for_almost_every_row(gpu, shape):
    """More of them than a wave has lanes, in each tile's list."""
    rows, k, n = shape
    check(gpu, make(rows + 2, np.arange(rows) * 7 % 281, [2] * 281, k, n,
                    scale=0.02))


@pytest.mark.parametrize("shape", [SMALL, (386, 512, 21528),
                                   (284, 5120, 6428)])
def test_a_row_reaches_no_other(gpu, shape):
    """NaN and infinities in rows of one request stay there."""
    rows, k, n = shape
    a = make(5, spread(rows, 3, 1), [16, 33, 8], k, n, scale=0.02)
    want, bound = ro.lora(**a)
    x = a["x"].reshape(rows, k).copy()
    x[::7, 3] = 0x7FC0
    x[3::7, k - 2] = 0xFF80
    bad = np.zeros(rows, bool)
    bad[::7] = bad[3::7] = True
    a["x"] = x.reshape(-1)
    got = run(gpu, a).reshape(rows, n)
    ro.check(got[~bad], want[~bad], bound[~bad])
    assert not np.isfinite(to_f32(got[bad])).any()


@pytest.mark.parametrize("rank", [1, 4, 20, 33, 40])
def test_an_infinity_against_positive_adapters_is_one(gpu, rank):
    """It meets the ranks there are, not their padding (0 times it is NaN)."""
    rows, k, n = SMALL
    a = make(16, np.zeros(rows), [rank], k, n)
    x = np.ones((rows, k))
    x[::3, 5] = np.inf
    a.update(x=ro_bits(x.reshape(-1)), w=ro_bits(np.ones(n * k)),
             down=[ro_bits(np.ones(rank * k))], up=[ro_bits(np.ones(rank * n))])
    got = to_f32(run(gpu, a)).reshape(rows, n)
    assert (got[::3] == np.inf).all()
    assert np.isfinite(np.delete(got, np.s_[::3], 0)).all()


def test_products_past_the_types_range_are_infinite(gpu):
    rows, k, n = SMALL
    a = make(6, np.zeros(rows), [8], k, n)
    a.update(x=ro_bits(np.full(rows * k, 3e38)), w=ro_bits(np.zeros(n * k)),
             down=[ro_bits(np.ones(8 * k))], up=[ro_bits(np.ones(8 * n))])
    assert (to_f32(run(gpu, a)) == np.inf).all()


@pytest.mark.parametrize("shape", [SMALL, (284, 5120, 6428)])
def test_gelu_of_the_sum_itself(gpu, shape):
    """One rounding, in whole tiles and behind pieces.  The sums are exact,
    multiples of 2^-11 below 2^5, and the activation's arithmetic is off by
    2^-20 of the argument, from -1 up at most 2^-17.3 of the result: under one
    result in 2^8 lies so near a border between two bf16 values, 2^-8 apart,
    that it may fall to the other.  Rounded twice, many do."""
    rows, k, n = shape
    rng = np.random.default_rng(17)
    a = dict(x=rng.integers(-2, 3, rows * k),
             w=rng.integers(-8, 9, n * k) / 1024, b=rng.integers(-8, 9, n) / 64)
    a = {name: ro_bits(v) for name, v in a.items()}
    a.update(down=[ro_bits(rng.integers(-1, 2, 16 * k))],
             up=[ro_bits(rng.integers(-2, 3, 16 * n) / 1024)], ranks=[16],
             scales=[0.5], ids=np.zeros(rows, np.uint32), k=k, n=n)
    got = to_f32(run(gpu, a, True)).astype(np.float64)
    sums = ro.lora(**a)[0].reshape(-1)
    assert (sums * 2048 == np.round(sums * 2048)).all()
    assert np.abs(sums).max() < 32
    up = sums > -1

    def others(values):
        nearest = to_f32(ro_bits(ro.gelu(sums))).reshape(-1)
        return (values != nearest)[up].mean()
    twice = to_f32(ro_bits(ro.gelu(to_f32(ro_bits(sums))))).reshape(-1)
    assert others(twice) > 2.0 ** -5
    assert others(got) < 2.0 ** -8


@pytest.mark.parametrize("shape", [SMALL, (284, 5120, 6428)])
def test_the_same_call_gives_the_same_bits(gpu, shape):
    rows, k, n = shape
    a = make(9, spread(rows, 4, 2), [16, 8, 33, 64], k, n, scale=0.02)
    table = table_of(gpu, a)
    first = run(gpu, a, table=table)
    run(gpu, make(10, spread(700, 2, 3), [128, 4], 192, 20480))
    assert (run(gpu, a, table=table) == first).all()


@pytest.mark.skipif(not shutil.which("g++"), reason="needs g++")
@pytest.mark.parametrize("rows,k,n", [(128, 2048, 8192), (40, 1024, 4100),
                                      (1, 2048, 8192)])
def test_up_to_128_rows_over_cut_tiles(rows, k, n):
    """A context whose scratch finds room only at the second attempt."""
    run_small(f"""
import test_lora_gpu as t
a = t.make(33, t.spread({rows}, 3, 1), [16, 40, 3], {k}, {n}, scale=0.02)
want, bound = ro.lora(**a)
limit(2 << 20)
second = h3hip.Gpu()  # without the scratch that contexts begin with
limit()
x, w, b, ids = (second.bf16(a["x"]), second.bf16(a["w"]), second.bf16(a["b"]),
                second.u32(a["ids"]))
table, y = t.table_of(second, a), second.new_bf16({rows * n})
small.fail_once(ctypes.c_size_t(1 << 20))
second.run("h3_hip_linear_lora_bf16", y, x, w, b, table, ids, {rows}, {k}, {n})
ro.check(second.read_bf16(y), want, bound)
""")
