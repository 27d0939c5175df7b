"""The 8-bit operators in 64 bits, with bounds on what a correct F32 kernel may
be off.

One rounding to bf16 is off by at most 2^-8 of the value, one in F32 by 2^-24
(both half a step); F32 sums and the hardware's exponentials and reciprocals as
in requests_oracle."""
import numpy as np

from conftest import to_f32
from requests_oracle import BF16, F32, gelu

HALF = 2.0 ** -24  # an F32 rounding


def bits(x):
    """bf16 bits of F32 values, ties to even."""
    b = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    nan = np.isnan(np.asarray(x, np.float32))
    out = ((b + 0x7fff + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(nan, np.uint16(0x7fc0), out)


def rows_of(x):
    """(codes, scales) of bf16 values given as float64 rows: exact.  127 x and
    the quotient's halves are exact in 64 bits, and a quotient that is no half
    lies 2^-17 of its size or more from one."""
    x = np.asarray(x, np.float64)
    most = np.abs(x).max(1)
    good = np.isfinite(most)
    safe = np.where(good & (most > 0), most, 1.0)[:, None]
    c = np.rint(127 * np.where(good[:, None], x, 0) / safe)
    s = np.float32(most.astype(np.float32)) / np.float32(127)
    return c, np.where(good, s, np.float32(np.nan)).astype(np.float32)


def values(c, s):
    """bf16 bits of the values that codes and F32 scales stand for."""
    with np.errstate(invalid="ignore"):
        return bits(c.astype(np.float32) * s)


def product(x, w, bias=None, act=False):
    """(y, bound) of the product of two (codes, scales)."""
    acc = x[0] @ w[0].T
    s = x[1].astype(np.float64)[:, None] * w[1].astype(np.float64)
    y, size = acc * s, np.abs(acc * s)
    if bias is not None:
        b = to_f32(bias).astype(np.float64)
        y, size = y + b, size + np.abs(b)
    # the sum's conversion, the scales' product (which may be subnormal), its
    # product with the sum, the bias
    bound = 5 * HALF * size + np.abs(acc) * 2.0 ** -149 + 2.0 ** -149
    if act:
        bound = 1.13 * bound + 2.0 ** -20 * np.abs(y)
        y = gelu(y)
    return y, bound


def rounded(y, bound):
    """The bound of a result rounded to bf16."""
    return bound * (1 + BF16) + BF16 * np.abs(y) + 1e-37


def norm(x, weight, bias, mod, row_map, shift, scale, eps, layer):
    """(v, bound) of adaLN rows in F32.  A row's sums are those of 256 threads,
    n / 256 terms each, joined over a wave of 64 and the waves."""
    n = x.shape[1] // 256 + 16
    size = np.abs(x)
    mean = x.mean(1, keepdims=True) if layer else 0.0
    if layer:
        # the mean: a sum of n terms
        off = (n + 1) * HALF * size.mean(1, keepdims=True)
        size = size + np.abs(mean)
    else:
        off = 0.0
    v = x - mean
    var = (v * v).mean(1, keepdims=True)
    inv = 1 / np.sqrt(var + eps)
    # 1 / sqrt of a sum of n squares, each off by the mean's error too
    rel = (n + 8) * HALF + (2 * off * np.abs(v).mean(1, keepdims=True) +
                           off * off) / (var + eps)
    v, bound = v * inv, (off + HALF * size) * inv
    bound = bound + rel * np.abs(v)
    if weight is not None:
        v, bound = v * weight, bound * np.abs(weight) + HALF * np.abs(v *
                                                                      weight)
    if bias is not None:
        v, bound = v + bias, bound + HALF * (np.abs(v) + np.abs(bias))
    if mod is not None:
        a, b = 1 + mod[row_map, scale], mod[row_map, shift]
        bound = bound * np.abs(a) + 3 * HALF * (np.abs(v * a) + np.abs(b))
        v = v * a + b
    return v, bound


def quantized(v, bound):
    """(codes, scales, doubtful, scale bound): rows of F32 values v known to
    `bound`; the codes of doubtful ones may be off by one."""
    most = np.abs(v).max(1, keepdims=True)
    off = bound.max(1, keepdims=True)
    safe = np.where(most > 0, most, 1.0)
    q = 127 * v / safe
    # value, maximum, and the quotient's own roundings
    may = 127 * (bound + off) / safe + 127 * 4 * HALF
    doubtful = np.abs(q - np.floor(q) - 0.5) <= may
    return (np.rint(q), (most / 127)[:, 0], doubtful,
            (off / 127 + HALF * most / 127)[:, 0])


def mlp(x, w1, w2):
    """(y, bound) of the gated block of (codes, scales)."""
    h = w1[0].shape[0] // 2
    gu, off = product(x, w1)
    g, u, og, ou = gu[:, :h], gu[:, h:], off[:, :h], off[:, h:]
    with np.errstate(over="ignore"):
        sig = 1 / (1 + np.exp(-g))
    v = g * sig * u
    # silu's slope is within 1.1; its exponential's argument rounds, which
    # moves the result by 2^-22 |g| of itself, exponential and reciprocal and
    # the products by a few more
    bound = 1.1 * og * np.abs(u) + np.abs(g * sig) * ou + og * ou + \
        np.abs(v) * (np.abs(g) + 6) * 2.0 ** -22
    c, s, doubtful, scale_off = quantized(v, bound)
    t = w2[1].astype(np.float64)
    acc = c @ w2[0].T
    y = acc * s[:, None] * t
    bound = (doubtful @ np.abs(w2[0]).T) * s[:, None] * t + \
        np.abs(acc) * t * scale_off[:, None] + 5 * HALF * np.abs(y)
    return y, bound


class Cache:
    """A cache of keys and values as the store leaves it: codes float64
    [rows][2][heads][dim], scales F32 [blocks][2][heads]."""

    def __init__(self, rows, heads, dim):
        blocks = (rows + 63) // 64
        self.c = np.zeros((blocks * 64, 2, heads, dim))
        self.s = np.zeros((blocks, 2, heads), np.float32)
        # codes that the store may have rounded the other way
        self.doubtful = np.zeros(self.c.shape, bool)

    def store(self, first, kv):
        """kv: float64 of bf16 values, [rows][2][heads][dim]."""
        end = first + len(kv)
        for block in range(first // 64, (end + 63) // 64):
            at = block * 64
            r0, r1 = max(first, at), min(end, at + 64)
            new = kv[r0 - first:r1 - first]
            most = np.abs(new).max((0, 3))
            s = most.astype(np.float32) / np.float32(127)
            # not finite: a NaN scale, codes of 0
            bad = ~np.isfinite(most)
            s = np.where(bad, np.float32(np.nan), s)
            rest = slice(at, at + 64)
            if r0 > at:
                old = self.s[block]
                grows = old < s
                keep = np.where(grows, old.astype(np.float64) /
                                np.where(grows, s, 1), 1.0)
                was = self.c[rest] * keep[None, :, :, None]
                self.c[rest] = np.rint(was)
                # the factor and the product round in F32
                self.doubtful[rest] |= np.abs(
                    was - np.floor(was) - 0.5) <= 4 * HALF * np.abs(was)
                top = np.where(grows, most, 127 * old.astype(np.float64))
                s = np.where(bad | np.isnan(old), np.float32(np.nan),
                             np.where(grows, s, old))
                # 127 * scale rounds where the scale stays
                off = 127 * 4 * HALF
            else:
                self.c[rest] = 0
                self.doubtful[rest] = False
                top, off = most, -1.0
            top = np.where(np.isnan(s) | (top == 0), 1.0, top)
            q = np.where(np.isnan(s)[None, :, :, None], 0,
                         127 * np.nan_to_num(new, posinf=0, neginf=0) /
                         top[None, :, :, None])
            self.c[r0:r1] = np.rint(q)
            self.doubtful[r0:r1] = np.abs(q - np.floor(q) - 0.5) <= off
            self.s[block] = s

    def steps(self):
        return np.repeat(self.s, 64, axis=0)[:, :, :, None]

    def values(self):
        """float64 [rows][2][heads][dim]"""
        return self.c * self.steps().astype(np.float64)


def attention(q, cache, ranges, heads, kv_heads, dim, scale):
    """(o, bound, covered rows) as requests_oracle.packed, over a cache."""
    kv = cache.values()
    step = np.abs(cache.steps().astype(np.float64)) * cache.doubtful
    o, bound = np.zeros_like(q), np.zeros_like(q)
    covered = np.zeros(len(q), bool)
    group = heads // kv_heads
    for qf, qn, kf, kn in ranges:
        covered[qf:qf + qn] = True
        if not kn or not qn:
            continue
        for h in range(heads):
            qs = q[qf:qf + qn, h]
            ks, vs = (kv[kf:kf + kn, i, h // group] for i in range(2))
            dk, dv = (step[kf:kf + kn, i, h // group] for i in range(2))
            s = qs @ ks.T * scale
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            o[qf:qf + qn, h] = p @ vs
            # a score: the products' sum (f16 holds a row of q, scaled to
            # 2^13, but for what is under 2^-25 there), the scales, doubtful
            # codes, the rounding of the exponent's argument
            top = np.abs(qs).max(1, keepdims=True)
            off = ((dim + 6) * F32 * (np.abs(qs) @ np.abs(ks).T) +
                   2.0 ** -38 * top * np.abs(ks).sum(1) +
                   np.abs(qs) @ dk.T).max(1, keepdims=True) * scale + \
                2.0 ** -22
            # P rounds to 11 bits, or by 2^-25 at most, lifted by 2^7 against a
            # reference that is at most the largest; of many rows of a key head
            # the values round to 11 bits too, or by 2^-25 of a unit that is at
            # most 2^-14 of the largest value its blocks have codes for
            bound[qf:qf + qn, h] = (p @ np.abs(vs)) * (
                (2.0 ** -11 if qn * group <= 32 else 2.01 * 2.0 ** -11) +
                2 * np.expm1(off) + 2 * (kn + 64) * F32) + \
                p @ dv + 2.0 ** -32 * p.max(1, keepdims=True) * \
                np.abs(vs).sum(0)
            if qn * group > 32:
                top = cache.s[kf // 64:(kf + kn + 63) // 64, 1, h // group]
                bound[qf:qf + qn, h] += 2.0 ** -39 * 127 * top.max()
    return o, rounded(o, bound), covered
