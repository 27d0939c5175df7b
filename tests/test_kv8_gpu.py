"""The cache of keys and values in 8 bits and attention over it, against the
same in 64 bits at the bounds of int8_oracle."""
import os

import numpy as np
import pytest

import int8_oracle as io
import requests_oracle as ro
from conftest import rand_bf16
from test_int8_gpu import MARK, ctx, plain, same  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


def blocks(n):
    return (n + 63) // 64


class Kv:
    """A cache on the device and in 64 bits, side by side."""

    def __init__(self, gpu, rows, heads, dim, seed=0):
        self.gpu, self.rows = gpu, blocks(rows) * 64
        self.heads, self.dim = heads, dim
        self.t = gpu.kv_int8(rows, heads, dim)
        self.wide = io.Cache(rows, heads, dim)
        self.rng = np.random.default_rng((rows, heads, dim, seed))

    def store(self, first, counts, std=1.0, pad=0, change=None):
        """Random rows at each place of `first`, all in one call."""
        width = self.heads * self.dim
        stride, total = 2 * width + pad, max(1, sum(counts))
        kv = rand_bf16(self.rng, total * stride, std).reshape(total, stride)
        if change:
            change(kv)
        d = self.gpu.bf16(kv)
        source = [int(s) for s in np.cumsum([0, *counts])[:-1]]
        self.gpu.begin()
        self.gpu.kv_int8_store(self.t, first, source, counts, d, 0, d, width,
                               stride)
        self.gpu.submit()
        wide = ro.wide(kv, total, stride)[:, :2 * width].reshape(
            total, 2, self.heads, self.dim)
        for f, s, n in zip(first, source, counts):
            if n:
                self.wide.store(f, wide[s:s + n])

    def read(self, first, rows):
        n = rows * self.heads * self.dim
        k, v = (self.gpu.bf16(np.full(n + 64, MARK, np.uint16))
                for _ in range(2))
        self.gpu.run("h3_hip_kv_int8_read", k, v, self.t, first, rows)
        got = [self.gpu.read_bf16(t) for t in (k, v)]
        assert all((g[n:] == MARK).all() for g in got)
        return np.stack([g[:n].reshape(rows, self.heads, self.dim)
                         for g in got], axis=1)

    def check(self, first, rows):
        got = self.read(first, rows)
        w = slice(first, first + rows)
        doubt = self.wide.doubtful[w]
        want = io.values(self.wide.c[w], self.wide.steps()[w])
        same(np.where(doubt, 0, got), np.where(doubt, 0, want))
        if doubt.any():
            step = np.abs(self.wide.steps()[w] + 0 * self.wide.c[w])[doubt]
            off = np.abs(ro.wide(got, *got.shape) - self.wide.values()[w])
            assert (off[doubt] <= 1.01 * step + io.BF16 * 128 * step).all()
            assert doubt.mean() < 0.02


@pytest.mark.parametrize("dim", [1, 8, 31, 32, 64, 72, 80, 96, 128, 129, 256])
@pytest.mark.parametrize("heads", [1, 3])
def test_store_whole(gpu, heads, dim):
    """Lengths around a block, rows of no range between them."""
    counts = [1, 63, 64, 65, 130, 0, 17]
    first = [int(f) for f in np.cumsum([0] + [
        64 * (blocks(c) + 1) for c in counts])[:-1]]
    kv = Kv(gpu, first[-1] + 64, heads, dim)
    kv.store(first, counts, pad=8 if dim % 8 == 0 else 3)
    for f, c in zip(first, counts):
        if c:
            kv.check(f, blocks(c) * 64)
            kv.check(f + c - 1, 1)


@pytest.mark.parametrize("dim", [64, 100, 128])
def test_store_goes_on(gpu, dim):
    """Row by row and in runs behind what the blocks have: smaller rows, then
    larger ones, which widen the scales."""
    kv = Kv(gpu, 400, 2, dim)
    at = 0
    for i, n in enumerate([1, 1, 5, 56, 1, 1, 70, 63, 2, 64, 3]):
        kv.store([at], [n], std=[1.0, 0.3, 2.0, 0.1, 5.0][i % 5])
        at += n
        kv.check(0, blocks(at) * 64)


def test_store_begins_anew(gpu):
    """A block's first row on: what it held has no part in its scales."""
    kv = Kv(gpu, 128, 2, 64)
    kv.store([0], [128], std=100.0)
    kv.store([0], [10])
    kv.check(0, 128)
    kv.store([64 + 0], [64], std=0.01)
    kv.check(0, 128)


@pytest.mark.parametrize("std", [0.5, 3.0])
def test_store_inside(gpu, std):
    """Rows in a block's middle: the ones before and behind stay."""
    for first, n in ((64 + 1, 1), (64 + 5, 3), (64 + 30, 34), (64 + 62, 2),
                     (64 + 7, 60)):
        kv = Kv(gpu, 192, 2, 80)
        kv.store([0], [192])
        kv.store([first], [n], std=std)
        kv.check(0, 192)


def test_new_cache_is_zeros(gpu):
    """Also in memory that held something else."""
    for _ in range(2):
        kv = Kv(gpu, 5000, 3, 64)
        kv.check(0, 5000)
        kv.store([3, 200], [2, 5], std=1e-3)
        kv.check(0, 5000)
        kv.store([0], [5000], std=30.0)
        gpu.free(kv.t)


def test_store_many_ranges(gpu):
    """More ranges than a launch takes, out of order."""
    order = np.random.default_rng(3).permutation(150)
    kv = Kv(gpu, 150 * 64, 1, 64)
    kv.store([int(o) * 64 for o in order], [1 + int(o) % 64 for o in order])
    kv.check(0, 150 * 64)
    kv.store([int(o) * 64 + 1 + int(o) % 64 for o in order if o % 64 < 63],
             [1 for o in order if o % 64 < 63])
    kv.check(0, 150 * 64)


def test_store_not_finite(gpu):
    """Infinities and NaN make their block's scale NaN, of the keys or the
    values of their head alone; going on behind them keeps it."""
    kv = Kv(gpu, 192, 2, 32)

    def change(rows):
        rows[70, 3], rows[130, 64 + 32] = 0x7f80, 0x7fc0
    kv.store([0], [140], change=change)
    kv.check(0, 192)
    kv.store([140], [10])
    kv.check(0, 192)
    kv.store([128], [64])
    kv.check(0, 192)


def test_store_extremes(gpu):
    """Zeros, then rows that make the scale; the ends of the range."""
    kv = Kv(gpu, 64, 1, 32)
    kv.store([0], [3], std=0.0)
    kv.store([3], [2])
    kv.check(0, 64)

    def change(rows):
        rows[0, 0], rows[1, 40] = 0x7f7f, 0x0001
    kv.store([5], [2], std=1e-20, change=change)
    kv.check(0, 64)


class Case:
    def __init__(self, gpu, qn, kn, heads, kv_heads, dim, seed=0, share=False,
                 pad=0, std=1.0, gap=0):
        self.gpu, self.heads, self.kv_heads, self.dim = \
            gpu, heads, kv_heads, dim
        self.qn, self.kn = qn, kn
        self.qf = [int(v) for v in np.cumsum(
            [0] + [n + gap for n in qn])[:-1]]
        self.kf = [0] * len(kn) if share else [64 * int(v) for v in np.cumsum(
            [0] + [blocks(n) for n in kn])[:-1]]
        self.rows = self.qf[-1] + qn[-1] + gap
        self.kv = Kv(gpu, max(64, max(f + n for f, n in zip(self.kf, kn))),
                     kv_heads, dim, seed)
        if share:
            self.kv.store([0], [max(kn)], std=std)
        else:
            self.kv.store(self.kf, kn, std=std)
        rng = np.random.default_rng(seed + 7)
        self.stride = heads * dim + pad
        self.q = rand_bf16(rng, self.rows * self.stride)
        self.scale = dim ** -0.5

    def run(self, scale=None):
        plan = self.gpu.sdpa_packed_plan(
            self.qf, self.qn, self.kf, self.kn, self.heads, self.kv_heads,
            self.dim)
        n = self.rows * self.heads * self.dim
        y = self.gpu.bf16(np.full(n + 256, MARK, np.uint16))
        self.gpu.run("h3_hip_sdpa_packed_int8_bf16", y, self.gpu.bf16(self.q),
                     0, self.stride, self.kv.t, plan,
                     self.scale if scale is None else scale)
        got = self.gpu.read_bf16(y)
        assert (got[n:] == MARK).all(), "wrote behind the last row"
        return got[:n].reshape(self.rows, self.heads, self.dim)

    def check(self):
        got = self.run()
        q = ro.wide(self.q, self.rows, self.stride)[
            :, :self.heads * self.dim].reshape(self.rows, self.heads, self.dim)
        want, bound, covered = io.attention(
            q, self.kv.wide, list(zip(self.qf, self.qn, self.kf, self.kn)),
            self.heads, self.kv_heads, self.dim,
            float(np.float32(self.scale)))
        ro.check(got[covered], want[covered], bound[covered])
        assert (got[~covered] == MARK).all(), "wrote rows of no request"
        return got


LENGTHS = [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 257, 513]


@pytest.mark.parametrize("n", LENGTHS)
def test_lengths(ctx, n):  # noqa: F811
    Case(ctx, [n], [n], 2, 2, 128).check()
    Case(ctx, [37], [n], 3, 1, 64).check()
    Case(ctx, [1], [n], 4, 2, 128).check()
    Case(ctx, [n], [70], 2, 1, 128).check()


@pytest.mark.parametrize("dim", [1, 8, 16, 31, 32, 40, 64, 72, 80, 96, 100,
                                 112, 128, 129, 192, 256])
def test_head_sizes(ctx, dim):  # noqa: F811
    Case(ctx, [70, 1, 9], [33, 130, 64], 4, 2, dim, pad=8).check()


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 5), (6, 3), (8, 1),
                                            (64, 8), (33, 1), (40, 1)])
def test_shared_heads(gpu, heads, kv_heads):
    Case(gpu, [1, 3, 50], [100, 65, 129], heads, kv_heads, 128).check()
    Case(gpu, [2, 40], [64, 300], heads, kv_heads, 64).check()


def test_empty_and_shared(ctx):  # noqa: F811
    """Requests without keys get zeros, without queries nothing; rows between
    requests stay; a text that requests share."""
    got = Case(ctx, [40, 3, 0, 1], [0, 65, 9, 0], 2, 2, 64, gap=2).check()
    assert not got[:40].any() and not got[-3].any()
    Case(ctx, [200, 1, 33], [100, 64, 7], 2, 1, 128, share=True).check()


def test_long_context(gpu):
    """Pieces of long contexts, joined."""
    Case(gpu, [1, 1], [4097, 9000], 8, 1, 128).check()
    Case(gpu, [3], [5000], 2, 2, 96).check()
    Case(gpu, [150], [3000], 1, 1, 64).check()


def test_many_rows(gpu):
    Case(gpu, [700, 333], [513, 90], 6, 6, 128).check()
    Case(gpu, [1000], [1000], 2, 1, 80).check()


@pytest.mark.parametrize("std", [30.0, 1e4, 1e-4])
def test_scores_large_and_small(gpu, std):
    """One key has all the weight, or all have the same."""
    Case(gpu, [70, 1], [300, 700], 2, 2, 128, std=std).check()


@pytest.mark.parametrize("powers", [
    [0, 3, 5, -3, -7, 4, 0, -5], [-90, 0, 30, -90, 60, 60, 90, 0],
    [60, -60, -61, -59, 60, -60, 0, -99], [0, -8, -9, -10, -7, -7, -6, -5]])
def test_blocks_of_unlike_scales(gpu, powers):
    """Values whose blocks' scales lie near and far from each other, the keys'
    the other way round, so that some rows attend to small values alone."""
    def change(rows):
        v = ro.wide(rows, *rows.shape)
        for block, power in enumerate(powers):
            at = slice(64 * block, 64 * block + 64)
            v[at, 2 * 128:] *= 2.0 ** power
            v[at, :2 * 128] *= 1 + 0.2 * (block % 3)
        rows[:] = io.bits(v.astype(np.float32)).reshape(rows.shape)
    c = Case(gpu, [70, 1, 1], [512, 512, 300], 2, 2, 128, share=True)
    c.kv.store([0], [512], change=change)
    c.check()
    # one block has all the weight of each row, by turns
    q = np.zeros((c.rows, 2, 128))
    q[np.arange(c.rows), :, np.arange(c.rows) % 8] = 1000
    c.q = io.bits(q.astype(np.float32)).ravel()

    def mark(rows):
        change(rows)
        k = rows[:, :2 * 128].reshape(-1, 2, 128)
        for block in range(8):
            k[64 * block:64 * block + 64, :, :8] = 0
            k[64 * block:64 * block + 64, :, block] = 0x3f80
    c.kv.store([0], [512], change=mark)
    c.check()


def test_queries_out_of_f16(gpu):
    """Query rows far from F16's range, zeros and rows of one large element."""
    for factor in (1e-30, 1e20):
        c = Case(gpu, [70, 1], [200, 400], 2, 2, 128, std=1.0)
        q = ro.wide(c.q, c.rows, c.stride) * factor
        q[3] = 0
        q[5, 1] *= 1000
        c.q = io.bits(q.astype(np.float32)).ravel()
        c.scale = float(np.float32(0.1 / factor))
        c.check()


def test_scale_of_zero(ctx):  # noqa: F811
    """Every key has the same weight."""
    c = Case(ctx, [40, 1], [100, 300], 2, 2, 64)
    c.scale = 0.0
    c.check()


def test_rows_behind_the_keys_have_no_part(gpu):
    """Fewer keys than the block holds: the result is that of the keys."""
    for n in (1, 30, 65):
        c = Case(gpu, [50, 2], [n, n], 2, 2, 64, share=True)
        c.kv = Kv(gpu, 128, 2, 64)
        c.kv.store([0], [128])
        c.check()


def test_a_bad_block_stays_with_its_readers(ctx):  # noqa: F811
    c = Case(ctx, [40, 1, 33], [100, 70, 64], 2, 2, 64)

    def change(rows):
        rows[2, 64 + 5] = 0x7f80  # keys of head 1 of the second request
    c.kv.store([c.kf[1]], [70], change=change)
    got = ro.wide(c.run(), c.rows, 2, 64)
    assert np.isnan(got[40, 1]).all()
    assert np.isfinite(got[40, 0]).all() and np.isfinite(got[:40]).all() and \
        np.isfinite(got[41:]).all()


def test_next_tokens(gpu):
    """A cache that grows by a row a step, read after each."""
    c = Case(gpu, [1, 1], [62, 5], 8, 2, 128)
    c.kv = Kv(gpu, 256, 2, 128, 5)
    c.kf = [0, 128]
    c.kv.store(c.kf, c.kn)
    for _ in range(5):
        c.kv.store([f + n for f, n in zip(c.kf, c.kn)], [1, 1], std=1.5)
        c.kn = [n + 1 for n in c.kn]
        c.check()


@pytest.mark.parametrize("powers", [[0, 9, -9, 4], [-60, -70, -50, -55],
                                    [60, 70, 50, 66], [0, 40, -40, 3]])
def test_many_rows_of_unlike_scales(gpu, powers):
    """Items of 128 rows, whose values share a unit."""
    def change(rows):
        v = ro.wide(rows, *rows.shape)
        for block, power in enumerate(powers):
            v[64 * block:64 * block + 64, 8 * 64:] *= 2.0 ** power
        rows[:] = io.bits(v.astype(np.float32)).reshape(rows.shape)
    c = Case(gpu, [4096], [256], 8, 8, 64)
    c.kv.store([0], [256], change=change)
    c.check()
    assert np.isfinite(ro.wide(c.run(), 4096, 512)).all()


@pytest.mark.parametrize("qn", [[6144], [1, 6144, 3], [2]])
def test_requests_without_keys(gpu, qn):
    """A plan that has nothing to unpack."""
    c = Case(gpu, qn, [0] * len(qn), 8, 8, 64)
    assert not c.check().any()


def test_keys_of_others_have_no_part(gpu):
    """Two requests share their first blocks; the longer one's last blocks are
    larger by 2^90 or not finite."""
    c = Case(gpu, [4096, 4096], [128, 256], 8, 8, 64, share=True)
    first = c.check()[:4096]

    def change(rows):
        v = ro.wide(rows, *rows.shape) * 2.0 ** 90
        rows[:] = io.bits(v.astype(np.float32)).reshape(rows.shape)
        rows[70] = 0x7f80
    c.kv.store([128], [128], change=change)
    assert np.array_equal(first, c.run()[:4096])
