"""Attention of packed requests against the same in 64 bits, at the bounds of
requests_oracle."""
import os
import subprocess
import sys

import numpy as np
import pytest

import requests_oracle as ro
from conftest import ROOT, rand_bf16, to_f32

pytestmark = pytest.mark.gpu


def starts(counts, gap=0):
    return [int(s) for s in np.cumsum([0, *[c + gap for c in counts]])[:-1]]


class Case:
    """Inputs and ranges; `gap` rows of no request behind each range."""

    def __init__(self, seed, qn, kn, heads, kv_heads, dim, qf=None, kf=None,
                 gap=0, std=1.0, pad=0):
        rng = np.random.default_rng(seed)
        self.qf = starts(qn, gap) if qf is None else qf
        self.kf = starts(kn, gap) if kf is None else kf
        self.qn, self.kn = qn, kn
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        self.rows = max(f + n for f, n in zip(self.qf, qn)) + gap
        self.kv = max(1, max(f + n for f, n in zip(self.kf, kn)) + gap)
        # the fused rows' widths, `pad` elements wider than what they hold
        self.qs, self.ks = heads * dim + pad, 2 * kv_heads * dim + pad
        self.q = rand_bf16(rng, self.rows * self.qs, std)
        self.kvs = rand_bf16(rng, self.kv * self.ks, std)
        self.scale = dim ** -0.5

    def parts(self):
        q = ro.wide(self.q, self.rows, self.qs)[:, :self.heads * self.dim]
        kv = ro.wide(self.kvs, self.kv, self.ks)
        w = self.kv_heads * self.dim
        return (q.reshape(self.rows, self.heads, self.dim),
                kv[:, :w].reshape(self.kv, self.kv_heads, self.dim),
                kv[:, w:2 * w].reshape(self.kv, self.kv_heads, self.dim))

    def want(self):
        return ro.packed(*self.parts(), list(zip(self.qf, self.qn, self.kf,
                                                 self.kn)),
                         self.heads, self.kv_heads, self.dim, self.scale)

    def run(self, gpu, plan=None, scale=None):
        plan = plan or gpu.sdpa_packed_plan(
            self.qf, self.qn, self.kf, self.kn, self.heads, self.kv_heads,
            self.dim)
        n = self.rows * self.heads * self.dim
        y = gpu.bf16(np.full(n + 256, 0x4141, np.uint16))
        kv = gpu.bf16(self.kvs)
        gpu.run("h3_hip_sdpa_packed_bf16", y, gpu.bf16(self.q), 0, self.qs, kv,
                0, kv, self.kv_heads * self.dim, self.ks, plan,
                self.scale if scale is None else scale)
        got = gpu.read_bf16(y)
        assert (got[n:] == 0x4141).all(), "wrote behind the last row"
        return got[:n].reshape(self.rows, self.heads, self.dim)

    def check(self, gpu, **how):
        got = self.run(gpu, **how)
        want, bound, covered = self.want()
        ro.check(got[covered], want[covered], bound[covered])
        assert (got[~covered] == 0x4141).all(), "wrote rows of no request"
        return got


LENGTHS = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 130, 192,
           255, 256, 257, 320, 511, 513]


@pytest.mark.parametrize("n", LENGTHS)
def test_lengths(gpu, n):
    """One request, query and key rows around the tiles' steps."""
    Case(n, [n], [n], 2, 2, 128).check(gpu)
    Case(n, [n], [67], 2, 1, 128).check(gpu)
    Case(n, [37], [n], 3, 1, 64).check(gpu)
    Case(n, [1], [n], 4, 2, 128).check(gpu)


@pytest.mark.parametrize("dim", [1, 3, 8, 16, 24, 40, 56, 64, 72, 80, 96, 100,
                                 112, 120, 127, 128, 129, 136, 192, 256])
def test_head_sizes(gpu, dim):
    Case(dim, [70, 1, 9], [33, 130, 64], 4, 2, dim).check(gpu)


@pytest.mark.parametrize("dim", [8, 64, 72, 96, 128])
@pytest.mark.parametrize("kn", [1, 31, 32, 33, 64, 65, 95, 97, 127, 128, 129, 161,
                                256, 300, 1025])
def test_few_rows_share_the_waves(gpu, dim, kn):
    """Up to 32 virtual rows a key head: keys split over the waves, of which
    some have none; and the 33rd."""
    Case(25, [1, 4, 5, 32, 33], [kn, 33, kn, 0, kn], 1, 1, dim, gap=1,
         pad=8).check(gpu)
    Case(26, [4, 1, 3, 36], [kn, kn, 2, kn], 16, 2, dim).check(gpu)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 5), (6, 3), (8, 1),
                                            (12, 4), (64, 8), (33, 1),
                                            (40, 1)])
@pytest.mark.parametrize("dim", [64, 128])
def test_shared_heads(gpu, heads, kv_heads, dim):
    """The heads of a group side by side, more and fewer than a tile holds."""
    Case(heads, [1, 3, 50], [100, 65, 129], heads, kv_heads, dim).check(gpu)


@pytest.mark.parametrize("dim", [64, 80, 128])
@pytest.mark.parametrize("pad", [0, 8, 40])
def test_many_requests(gpu, dim, pad):
    rng = np.random.default_rng(dim)
    qn = [int(v) for v in rng.choice([0, 1, 1, 2, 7, 40, 129, 300], 40)]
    kn = [int(v) for v in rng.choice([0, 1, 5, 63, 64, 65, 200, 513], 40)]
    Case(1, qn, kn, 4, 2, dim, gap=3, pad=pad).check(gpu)


def test_requests_in_any_order_that_share_keys(gpu):
    Case(2, [50, 1, 70, 4], [90, 90, 33, 0], 4, 4, 128, qf=[80, 79, 0, 140],
         kf=[10, 10, 47, 500]).check(gpu)


def test_strides_and_offsets_that_are_not_multiples_of_eight(gpu):
    Case(3, [40, 9], [70, 5], 3, 3, 64, pad=3).check(gpu)
    Case(3, [40, 9], [70, 5], 3, 3, 128, pad=4).check(gpu)


def test_fused_rows(gpu):
    """Q, K and V of self-attention in the rows of one tensor."""
    rng = np.random.default_rng(4)
    heads, kv_heads, dim, qn = 6, 2, 128, [130, 1, 64, 299]
    w, rows = (heads + 2 * kv_heads) * dim, sum(qn)
    bits = rand_bf16(rng, rows * w)
    first = starts(qn)
    plan = gpu.sdpa_packed_plan(first, qn, first, qn, heads, kv_heads, dim)
    y, t = gpu.new_bf16(rows * heads * dim), gpu.bf16(bits)
    gpu.run("h3_hip_sdpa_packed_bf16", y, t, 0, w, t, heads * dim, t,
            (heads + kv_heads) * dim, w, plan, 0.1)
    all_ = ro.wide(bits, rows, heads + 2 * kv_heads, dim)
    want, bound, _ = ro.packed(
        all_[:, :heads], all_[:, heads:heads + kv_heads],
        all_[:, heads + kv_heads:], list(zip(first, qn, first, qn)), heads,
        kv_heads, dim, float(np.float32(0.1)))
    ro.check(gpu.read_bf16(y), want, bound)


@pytest.mark.parametrize("qn,kn,heads,kv_heads", [
    ([1] * 3, [9720, 4097, 1], 16, 2), ([2, 1], [6144, 0], 8, 8),
    ([1], [20000], 8, 1), ([1500], [3000], 2, 2), ([40, 600], [5000, 77], 4, 1),
    ([33], [33240], 1, 1)])
def test_long_contexts(gpu, qn, kn, heads, kv_heads):
    """Key rows cut over the CUs and joined."""
    Case(5, qn, kn, heads, kv_heads, 128).check(gpu)
    Case(6, qn, kn, heads, kv_heads, 64).check(gpu)


@pytest.mark.parametrize("std", [8.0, 30.0])
def test_scores_far_apart(gpu, std):
    """Scores of some hundreds: the running maximum moves many times."""
    a = Case(7, [100, 1, 33], [300, 1000, 65], 4, 2, 128, std=std)
    a.scale = 2.0 / std
    a.check(gpu)


def test_ascending_scores(gpu):
    """Every tile's keys score higher than the last one's."""
    a = Case(8, [70, 3], [640, 200], 2, 2, 128)
    kv = to_f32(a.kvs).reshape(a.kv, 4, 128)
    kv[:, :2] = np.linspace(-40, 40, a.kv)[:, None, None] / 11
    a.kvs = ro_bits(kv)
    q = to_f32(a.q)
    q[:] = np.abs(q)
    a.q = ro_bits(q)
    a.check(gpu)


def ro_bits(values):
    import oracle
    return oracle.bf16(np.ascontiguousarray(values, np.float32).reshape(-1))


def test_a_zero_scale_takes_the_mean(gpu):
    a = Case(9, [40, 2], [100, 7], 2, 2, 128)
    a.scale = 0.0
    a.check(gpu)


@pytest.mark.parametrize("dim", [64, 80, 128])
def test_rows_of_other_requests_are_not_read(gpu, dim):
    """NaN and infinities behind a request's keys, in other requests' rows and
    in rows of none, leave it as it is."""
    a = Case(10, [40, 2, 1], [70, 7, 130], 4, 2, dim, gap=5)
    want = a.run(gpu)
    k = a.kvs.reshape(a.kv, -1).copy()
    live = np.zeros(a.kv, bool)
    for f, n in zip(a.kf, a.kn):
        live[f:f + n] = True
    k[~live] = 0x7FC0
    k[~live, ::2] = 0x7F80
    a.kvs = k.reshape(-1)
    assert (a.run(gpu) == want).all()
    k[a.kf[1]:a.kf[1] + a.kn[1]] = 0xFF80
    a.kvs = k.reshape(-1)
    got = a.run(gpu)
    assert (got[:40] == want[:40]).all()
    assert (got[a.qf[2]] == want[a.qf[2]]).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_a_query_row_that_is_nan(gpu, dim):
    """It is NaN in the result, and no other row is."""
    a = Case(11, [40, 3], [70, 200], 4, 2, dim)
    want = a.run(gpu)
    q = a.q.reshape(a.rows, -1).copy()
    q[5, 0] = q[41, 0] = 0x7FC0
    a.q = q.reshape(-1)
    got = a.run(gpu)
    bad = np.zeros((a.rows, 4), bool)
    bad[5, 0] = bad[41, 0] = True
    assert np.isnan(to_f32(got[bad])).all()
    assert (got[~bad] == want[~bad]).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_a_row_is_the_same_beside_any_others(gpu, dim):
    """Its bits, with rows beside it whose maximum moves at other keys."""
    a = Case(19, [64, 9], [700, 300], 4, 2, dim)
    want = a.run(gpu)
    q = to_f32(a.q).reshape(a.rows, -1).copy()
    other = np.arange(a.rows) % 3 > 0
    q[other] *= 200 * np.random.default_rng(1).uniform(-1, 1, (other.sum(), 1))
    a.q = ro_bits(q)
    got = a.run(gpu)
    assert (got[~other] == want[~other]).all()
    assert (got[other] != want[other]).any()


@pytest.mark.parametrize("dim", [64, 128])
def test_a_key_that_is_nan_or_infinite(gpu, dim):
    """A NaN key makes its request's rows NaN; an infinite one as well, where
    its score is (inf - inf)."""
    for bits in (0x7FC0, 0x7F80):
        a = Case(12, [40, 3], [70, 200], 4, 2, dim)
        want = a.run(gpu)
        k = a.kvs.reshape(a.kv, -1).copy()
        k[3, 0] = bits
        a.kvs = k.reshape(-1)
        got = a.run(gpu)
        s = to_f32(a.q).reshape(a.rows, 4, dim)[:40, :2, 0] * (
            np.inf if bits == 0x7F80 else np.nan)
        # a score of -inf has no weight: such rows stay finite
        lost = ~(s == -np.inf)
        assert np.isnan(to_f32(got[:40, :2][lost])).all()
        assert np.isfinite(to_f32(got[:40, :2][~lost])).all()
        assert (got[40:] == want[40:]).all()
        assert (got[:, 2:] == want[:, 2:]).all()


@pytest.mark.parametrize("dim", [64, 80, 100, 128])
def test_keys_of_no_weight_before_far_lower_ones(gpu, dim):
    """Scores of -inf for the first tiles, or all of a piece, and then scores
    whose weights against a maximum of 0 would all be 0; the last request has
    no others and gets zeros."""
    for qn, kn, out in (([40, 2, 3], [200, 331, 70], [70, 129, 70]),
                        ([1, 1], [9720, 500], [5000, 500])):
        a = Case(18, qn, kn, 4, 2, dim)
        q = to_f32(a.q).reshape(a.rows, -1)
        a.q = ro_bits(1 + np.abs(q) / 4)
        kv = to_f32(a.kvs).reshape(a.kv, -1).copy()
        kv[:, :2 * dim] = kv[:, :2 * dim] / 4 - 18
        bits = ro_bits(kv).reshape(a.kv, -1)
        for f, n in zip(a.kf, out):
            bits[f:f + n, 0] = bits[f:f + n, dim] = 0xFF80
        a.kvs = bits.reshape(-1)
        got = a.run(gpu)
        # the oracle is not shown the keys of no weight
        whole = a.kf, a.kn
        a.kf = [f + n for f, n in zip(a.kf, out)]
        a.kn = [k - n for k, n in zip(a.kn, out)]
        want, bound, _ = a.want()
        a.kf, a.kn = whole
        assert np.abs(want[0]).max() > 0
        ro.check(got, want, bound)


@pytest.mark.parametrize("dim", [64, 72, 128])
def test_rows_that_lie_past_four_gigabytes(gpu, dim):
    """Row strides of 16 MB: 330 key rows over 5 GB."""
    a = Case(23, [3, 2], [129, 201], 1, 1, dim)
    compact = gpu.bf16(a.kvs)
    stride = (1 << 23) + 8
    q, kv = gpu.bf16(a.q), gpu.new_bf16((a.kv - 1) * stride + 2 * dim)
    gpu.begin()
    for r in range(a.kv):
        gpu.check(gpu.L.h3_gpu_copy_bf16(gpu.h, kv, r * stride, compact,
                                         r * 2 * dim, 2 * dim))
    gpu.submit()
    plan = gpu.sdpa_packed_plan(a.qf, a.qn, a.kf, a.kn, 1, 1, dim)
    y = gpu.new_bf16(a.rows * dim)
    gpu.run("h3_hip_sdpa_packed_bf16", y, q, 0, a.qs, kv, 0, kv, dim, stride,
            plan, a.scale)
    got = gpu.read_bf16(y).reshape(a.rows, 1, dim)
    gpu.free(kv)
    want, bound, _ = a.want()
    ro.check(got, want, bound)
    assert (got == a.run(gpu)).all()


def test_two_contexts_at_once(gpu):
    """Each with its own sums of pieces; a plan serves both."""
    import h3hip
    with h3hip.Gpu() as other:
        a = Case(24, [1, 2], [9720, 5000], 8, 2, 128)
        plan = gpu.sdpa_packed_plan(a.qf, a.qn, a.kf, a.kn, 8, 2, 128)
        n = a.rows * 8 * 128
        made = [(g, [g.new_bf16(n) for _ in range(4)], g.bf16(a.q),
                 g.bf16(a.kvs)) for g in (gpu, other)]
        gpu.begin()
        other.begin()
        for turn in range(4):
            for g, y, q, kv in made:
                g.check(g.L.h3_hip_sdpa_packed_bf16(
                    g.h, y[turn], q, 0, a.qs, kv, 0, kv, 256, a.ks, plan,
                    a.scale))
        other.submit()
        gpu.submit()
        want, bound, _ = a.want()
        for g, y, *_ in made:
            for t in y:
                ro.check(g.read_bf16(t).reshape(a.rows, 8, 128), want, bound)


def test_the_same_call_gives_the_same_bits(gpu):
    for a in (Case(13, [1, 1, 2], [9000, 33, 700], 8, 1, 128),
              Case(14, [300, 40], [400, 1300], 4, 4, 64)):
        plan = gpu.sdpa_packed_plan(a.qf, a.qn, a.kf, a.kn, a.heads,
                                    a.kv_heads, a.dim)
        first = a.run(gpu, plan=plan)
        Case(15, [500], [5000], 4, 1, 128).run(gpu)
        assert (a.run(gpu, plan=plan) == first).all()


def test_plans_queued_one_after_the_other(gpu):
    cases = [Case(16, [1, 2], [9000, 33], 8, 1, 128),
             Case(17, [700], [700], 4, 4, 128),
             Case(18, [1], [20000], 8, 8, 64)] * 2
    made = []
    for a in cases:
        kv = gpu.bf16(a.kvs)
        made.append((a, gpu.new_bf16(a.rows * a.heads * a.dim), gpu.bf16(a.q),
                     kv, gpu.sdpa_packed_plan(a.qf, a.qn, a.kf, a.kn, a.heads,
                                              a.kv_heads, a.dim)))
    gpu.begin()
    for a, y, q, kv, plan in made:
        assert gpu.L.h3_hip_sdpa_packed_bf16(
            gpu.h, y, q, 0, a.qs, kv, 0, kv, a.kv_heads * a.dim, a.ks, plan,
            a.scale)
    gpu.submit()
    for a, y, *_ in made:
        want, bound, _ = a.want()
        ro.check(gpu.read_bf16(y), want, bound)


def test_simple_kernel(gpu):
    """H3_HIP_REFERENCE=1 takes the sequential kernel, at the same bounds."""
    code = """
import sys
sys.path[:0] = sys.argv[1:]
import h3hip, test_packed_gpu as t
gpu = h3hip.Gpu()
for dim in (64, 100, 128):
    t.Case(1, [1, 40, 0, 70], [300, 64, 9, 0], 4, 2, dim, gap=2).check(gpu)
print("fine")
"""
    done = subprocess.run(
        [sys.executable, "-c", code] + [os.path.join(ROOT, d) for d in (
            "h3.c_amd", "oracle", "tests")], capture_output=True, text=True,
        env={**os.environ, "H3_HIP_REFERENCE": "1"}, timeout=100)
    assert done.returncode == 0 and "fine" in done.stdout, done.stderr[-2000:]
