"""Packed attention with scores far from zero, against the same in 64 bits.

Scores are exact in F32: a query's first dim times a key's first is the score's
distance from zero, a multiple of a power of two, its second times the key's
second a small number beside it, so that the weights differ as in any softmax
however far the scores lie."""
import numpy as np
import pytest

import requests_oracle as ro
from conftest import to_f32
from test_packed_gpu import Case, ro_bits

pytestmark = pytest.mark.gpu

SHAPES = [([1, 3], [200, 77], 2, 1),          # up to 32 virtual rows
          ([70, 2], [300, 65], 2, 2),         # rows over the waves
          ([1, 2], [9720, 5000], 4, 1),       # pieces of few rows
          ([128], [9720], 8, 8)]              # and of 128
DIMS = [64, 72, 100, 128]  # 100: the sequential kernel


def far(seed, shape, dim, base, low, scale):
    """Scores base + j / 4, |j| <= 32, of most keys, `low` + j / 4 of the
    others, every tile's first keys among them."""
    qn, kn, heads, kv_heads = shape
    a = Case(seed, qn, kn, heads, kv_heads, dim)
    a.scale = scale
    rng = np.random.default_rng(seed)
    q = np.zeros((a.rows, heads, dim))
    q[..., 0] = 2.0 ** 12
    q[..., 1] = 0.25
    kv = to_f32(a.kvs).reshape(a.kv, 2, kv_heads, dim).copy()
    kv[:, 0] = 0
    at = np.full((a.kv, kv_heads), base)
    # the first 100 keys of each request, and some others
    for f, n in zip(a.kf, a.kn):
        at[f:f + min(100, n // 2)] = low
    at[rng.random(at.shape) < 0.2] = low
    kv[:, 0, :, 0] = at / 2.0 ** 12
    # a fine part where F32 has room for it
    if abs(base) < 2.0 ** 21:
        kv[:, 0, :, 1] = rng.integers(-32, 33, at.shape)
    a.q, a.kvs = ro_bits(q), ro_bits(kv)
    s = to_f32(a.kvs).reshape(kv.shape)[:, 0, :, 0].astype(np.float64)
    assert (s * 2.0 ** 12 == at).all(), "not the scores that were meant"
    return a


def want(a):
    """(o, bound).  The exponent's argument, (s - top) scale log2(e) of a top up
    to 1024 away from the one that it is taken against, is off by 2^-14, of
    scores exact as here: two roundings of 2^-15 of references below 1024, and
    2^-23 of differences up to 24, below which a weight is under 2^-34."""
    q, k, v = a.parts()
    o, bound = np.zeros_like(q), np.zeros_like(q)
    group = a.heads // a.kv_heads
    for qf, qn, kf, kn in zip(a.qf, a.qn, a.kf, a.kn):
        for h in range(a.heads):
            s = q[qf:qf + qn, h] @ k[kf:kf + kn, h // group].T
            p = np.exp((s - s.max(1, keepdims=True)) * a.scale)
            p /= p.sum(1, keepdims=True)
            vs = v[kf:kf + kn, h // group]
            o[qf:qf + qn, h] = p @ vs
            bound[qf:qf + qn, h] = p @ np.abs(vs) * (
                ro.BF16 + 2 * np.expm1(2.0 ** -13) + 2 * (kn + 64) * ro.F32
                + 2.0 ** -30)
    return o, bound * (1 + ro.BF16) + ro.BF16 * np.abs(o) + 1e-37


@pytest.mark.parametrize("base", [2.0 ** 8, 2.0 ** 11, 2.0 ** 20, 1.5 * 2.0 ** 33,
                                  1.25 * 2.0 ** 40, 2.0 ** 60])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("dim", DIMS)
def test_scores_far_from_zero(gpu, dim, shape, base):
    scale = 0.3125
    for sign, low in ((1, 0.0), (-1, 2 * -base), (1, base / 2), (1, -base)):
        a = far(41, SHAPES[shape], dim, sign * base, low, scale)
        got = a.run(gpu)
        ro.check(got, *want(a), what=f"{sign * base} beside {low}")


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("scale", [2.0 ** 60, 3e38])
def test_scales_of_any_size(gpu, dim, scale):
    """The keys of the largest score share the weight, those of others have
    none, also where the scaled scores pass the type's range."""
    for shape in SHAPES:
        a = far(43, shape, dim, 2.0 ** 12, 2.0 ** 11, float(np.float32(scale)))
        ro.check(a.run(gpu), *want(a))


def test_rows_beside_far_ones_keep_their_bits(gpu):
    for shape in SHAPES:
        a = Case(44, *shape, 128)
        want_bits = a.run(gpu)
        q = to_f32(a.q).reshape(a.rows, a.heads, 128).copy()
        q[:, 0] *= 2.0 ** 30
        a.q = ro_bits(q)
        got = a.run(gpu)
        assert (got[:, 1:] == want_bits[:, 1:]).all()
        assert np.isfinite(to_f32(got)).all()
