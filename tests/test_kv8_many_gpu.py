"""Attention over the 8-bit cache by items of more than 32 rows and of fewer
(MANY, FEW and ROWS; test_int8_routes.py holds them to their kernels), also where
scores and factors lie far from zero or one, against the same in 64 bits at the
bounds of int8_oracle."""
import numpy as np
import pytest

import int8_oracle as io
import requests_oracle as ro
from test_int8_gpu import plain  # noqa: F401 (a fixture)
from test_kv8_gpu import Case, Kv

pytestmark = pytest.mark.gpu

FEW, ROWS = 20, 129  # query rows of items of each kind, with up to 128 keys

# query rows, first key rows (None: side by side) and key rows of each request,
# heads, key heads, head size: the kernels between unpacking and join
MANY = [
    *(([129, 1, 40], None, [70, 128, 33], 4, 2, dim, kernels)
      for dim, kernels in (
        (8, ["codes<64>", "few<32>"]), (40, ["codes<64>", "few<64>"]),
        (64, ["codes<64>", "few<64>"]), (72, ["codes<96>", "few<96>"]),
        (80, ["codes<96>", "few<96>"]), (96, ["codes<96>", "few<96>"]),
        (104, ["codes<128>", "few<128>"]),
        (128, ["codes<128>", "few<128>"]))),
    *(([170], None, [n], 2, 2, dim, [f"codes<{dim}>"])
      for n in (1, 31, 32, 33, 63, 64, 65, 127, 128) for dim in (64, 128)),
    ([1, 200, 8, 129, 40], [0, 0, 320, 448, 320], [100, 100, 65, 128, 64], 4,
     2, 128, ["codes<128>", "few<128>"]),
    ([2000, 1, 300, 20], [0, 0, 704, 704], [700, 500, 200, 64], 10, 10, 80,
     ["codes<96>", "few<96>"]),
    ([2048, 1], [0, 0], [300, 300], 16, 2, 128, ["codes<128>", "few<128>"]),
    ([4096], None, [700], 8, 8, 96, ["codes<96>"]),
    # in pieces
    ([128], None, [9720], 8, 8, 128, ["codes<128>", "joined<128>"]),
    ([256], None, [5000], 8, 2, 64, ["codes<64>", "joined<64>"]),
    ([256], None, [5000], 8, 2, 96, ["codes<96>", "joined<128>"]),
    ([300, 1], [0, 0], [5000, 4000], 8, 2, 128,
     ["codes<128>", "few<128>", "joined<128>"]),
    # what the matrix cores do not take
    ([129, 1], None, [70, 128], 2, 2, 100, ["simple"]),
    ([129, 1], None, [70, 128], 2, 2, 136, ["simple"]),
]


def many(gpu, qn, kf, kn, heads, kv_heads, dim, **more):
    c = Case(gpu, qn, kn if not kf else [
        max(f + n for f, n in zip(kf, kn))] * len(kn), heads, kv_heads, dim,
        share=bool(kf), **more)
    if kf:
        c.kf, c.kn = kf, kn
    return c


@pytest.mark.parametrize("case", MANY, ids=lambda c: str(c[:6]))
def test_many(gpu, case):
    c = many(gpu, *case[:-1], pad=8, gap=2)
    assert np.array_equal(c.check(), c.run()), "other bits the second time"


@pytest.mark.parametrize("std", [30.0, 1e4, 1e-4])
@pytest.mark.parametrize("rows", [FEW, ROWS])
def test_scores_large_and_small(gpu, rows, std):
    """One key has all the weight, or all have the same."""
    for dim in (64, 96, 128):
        Case(gpu, [rows, 1], [100, 128], 2, 2, dim, std=std).check()


@pytest.mark.parametrize("powers", [[0, 9], [-9, 0], [0, 40], [-60, -70],
                                    [30, -30]])
def test_keys_of_unlike_scales(gpu, powers):
    """Of the first block and the second."""
    for rows in (FEW, ROWS):
        c = Case(gpu, [rows], [100], 2, 2, 128)

        def change(kv):
            v = ro.wide(kv, *kv.shape)
            for block, power in enumerate(powers):
                v[64 * block:64 * block + 64, :256] *= 2.0 ** power
            kv[:] = io.bits(v.astype(np.float32)).reshape(kv.shape)
        c.kv.store([0], [100], change=change)
        c.scale *= 2.0 ** -max(powers)
        c.check()


def numbers(c):
    """A case's query rows in 64 bits, [row][head][dim]."""
    return ro.wide(c.q, c.rows, c.heads, c.dim).copy()


def put(c, q):
    c.q = io.bits(q.astype(np.float32)).ravel()


@pytest.mark.parametrize("rows", [FEW, ROWS])
@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("stored", [False, True])
def test_far_scores_and_a_last_block_of_zeros(gpu, rows, dim, stored):
    """Scores to +-1e3 of one block of keys, then part of a block whose keys are
    zeros, stored or not."""
    c = Case(gpu, [rows], [70], 2, 2, dim)
    c.kv = Kv(gpu, 128, 2, dim)

    def change(kv):
        kv[:64, 0] = kv[:64, dim] = 0x42c8  # 100
        kv[64:, :2 * dim] = 0
    c.kv.store([0], [70 if stored else 64], change=change)
    q = numbers(c)
    q[:, :, 0] = 0
    q[::5, 0, 0], q[3::7, 1, 0] = 200, -200
    put(c, q)
    c.check()


FACTORS = [
    (5e37, 1e-34, 1e-5), (1e36, 1e-33, 4.6e-5), (1e34, 1e-31, 4.6e-5),
    (1e30, 1e-32, 1e-1), (1e-30, 1e30, 0.2), (1e-35, 1e30, 1e4),
    (1e-30, 1.0, 1e29), (1e-3, 1e-33, 1e35)]


@pytest.mark.parametrize("rows", [FEW, ROWS])
@pytest.mark.parametrize("dim", [64, 80, 128])
@pytest.mark.parametrize("size,std,scale", FACTORS)
def test_scores_of_large_and_small_factors(gpu, rows, dim, size, std, scale):
    """Queries, keys and the scale near the ends of F32's range, scores of
    ordinary size."""
    c = Case(gpu, [rows], [100], 2, 2, dim, std=std)
    put(c, numbers(c) * size)
    c.scale = float(np.float32(scale))
    c.check()


@pytest.mark.parametrize("dim", [64, 136, 256])
@pytest.mark.parametrize("size,std,scale", FACTORS)
def test_factors_in_the_simple_kernel(plain, dim, size, std,  # noqa: F811
                                      scale):
    test_scores_of_large_and_small_factors(plain, FEW, dim, size, std, scale)


@pytest.mark.parametrize("rows", [FEW, ROWS])
def test_rows_never_stored_are_zeros_to_large_queries(gpu, rows):
    """In memory that held something else."""
    c = Case(gpu, [rows], [70], 2, 2, 64)
    old = Kv(gpu, 128, 2, 64)
    old.store([0], [128], std=30.0)
    gpu.free(old.t)
    c.kv = Kv(gpu, 128, 2, 64)
    c.kv.store([0], [64], std=1e-33)
    put(c, numbers(c) * 1e35)
    c.scale = float(np.float32(4.6e-4))
    c.check()


@pytest.mark.parametrize("qn", [[FEW] * 20, [ROWS] * 3])
@pytest.mark.parametrize("dim", [64, 96, 128])
def test_a_row_is_the_same_beside_any_others(gpu, qn, dim):
    """Its bits, with rows beside it of scores far from zero, of infinities and
    of NaN."""
    c = Case(gpu, qn, [110] * len(qn), 2, 2, dim, share=True)
    put(c, numbers(c) * 40)
    want = c.check()
    q = numbers(c)
    other = np.arange(c.rows) % 3 > 0
    q[other] *= 100 * np.random.default_rng(1).uniform(-1, 1,
                                                       (other.sum(), 1, 1))
    put(c, q)
    got = c.check()
    assert np.array_equal(got[~other], want[~other])
    assert (got[other] != want[other]).any()
    bits = c.q.reshape(c.rows, 2, dim)
    bits[1, 0, 3], bits[4, 0, 5], bits[5, 1, 6] = 0x7f80, 0x7fc0, 0xff80
    spoilt = c.run()
    assert np.array_equal(spoilt[~other], want[~other])
    assert np.isnan(ro.wide(spoilt, *spoilt.shape)[4, 0]).all()


def test_values_of_the_smallest_sizes(gpu):
    """Near 2^-113, the mean of 1475 of them."""
    c = Case(gpu, [4096], [1475], 8, 8, 64)

    def change(kv):
        v = ro.wide(kv, *kv.shape)
        v[:, 512:] = 1.5e-34 * (1 + 0.01 * np.tanh(v[:, 512:]))
        kv[:] = io.bits(v.astype(np.float32)).reshape(kv.shape)
    c.kv.store([0], [1475], change=change)
    put(c, numbers(c) * 0)
    c.check()


@pytest.mark.parametrize("count", [63, 64, 65, 150])
def test_many_requests(gpu, count):
    """Each with a range of blocks of its own, or one of several of a text."""
    kn = [1 + 37 * i % 128 for i in range(count)]
    Case(gpu, [33 + i % 3 for i in range(count)], kn, 5, 5, 64).check()
    c = Case(gpu, [40] * count, [700] * count, 5, 5, 64, share=True)
    c.kf = [64 * (i % 7) for i in range(count)]
    c.kn = [1 + 23 * i % 250 for i in range(count)]
    c.check()
