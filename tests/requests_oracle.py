"""The operators of packed requests in 64 bits, with bounds on what a correct
F32 kernel may be off, and a way to call the backend without a GPU.

One rounding to bf16 is off by at most 2^-8 of the value (half a step of the
8-bit significand).  An F32 sum of n terms is off by at most n 2^-23 of the sum
of their magnitudes (each addition by 2^-23, which also allows a matrix core
that cuts instead of rounding)."""
import json
import math
import os
import subprocess
import sys

import numpy as np

from conftest import ROOT, to_f32
from launches import _fake

BF16, F32 = 2.0 ** -8, 2.0 ** -23
NONE = 0xFFFFFFFF


def wide(bits, *shape):
    return to_f32(bits).astype(np.float64).reshape(shape)


def gelu(y):
    return 0.5 * y * (1 + np.tanh(
        math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))


def lora(x, w, b, down, up, ranks, scales, ids, k, n, act=False):
    """(y, bound) of a projection with adapters; bf16 bits in, float64 out."""
    rows = len(ids)
    x, w = wide(x, rows, k), wide(w, n, k)
    y = x @ w.T
    size = np.abs(x) @ np.abs(w).T
    if b is not None:
        y, size = y + wide(b, n), size + np.abs(wide(b, n))
    bound = np.zeros((rows, n))
    most = 0
    for a, (rank, scale) in enumerate(zip(ranks, scales)):
        at = np.flatnonzero(ids == a)
        if not len(at) or not rank:
            continue
        scale = float(np.float32(scale))
        d, u = wide(down[a], rank, k), wide(up[a], n, rank)
        low = scale * (x[at] @ d.T)
        low_size = abs(scale) * (np.abs(x[at]) @ np.abs(d).T)
        y[at] += low @ u.T
        size[at] += np.abs(low) @ np.abs(u).T
        # the first sum and its scaling, then the two bf16 halves: the second
        # rounds what the first leaves, 2^-8 of 2^-8
        bound[at] += ((k + 1) * F32 * low_size +
                      BF16 * BF16 * np.abs(low)) @ np.abs(u).T
        most = max(most, rank)
    # every half of the low products is a term
    bound += (k + 2 * most + 1) * F32 * size
    if act:
        # the derivative of gelu is under 1.13; the activation's own F32
        # arithmetic is under 2^-20 of the argument
        bound = 1.13 * bound + 2.0 ** -20 * np.abs(y)
        y = gelu(y)
    return y, bound * (1 + BF16) + BF16 * np.abs(y) + 1e-37


def packed(q, k, v, ranges, heads, kv_heads, dim, scale):
    """(o, bound, covered rows): q [rows][heads][dim], k and v
    [rows][kv_heads][dim] float64, ranges (q_first, q_rows, kv_first, kv_rows)
    of each request."""
    o = np.zeros_like(q)
    bound = np.zeros_like(q)
    covered = np.zeros(len(q), bool)
    group = heads // kv_heads
    for qf, qn, kf, kn in ranges:
        covered[qf:qf + qn] = True
        if not kn or not qn:
            continue
        for h in range(heads):
            qs = q[qf:qf + qn, h]
            ks, vs = k[kf:kf + kn, h // group], v[kf:kf + kn, h // group]
            s = qs @ ks.T * scale
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            o[qf:qf + qn, h] = p @ vs
            # a score: the sum of the products, the scaling in F32, and the
            # rounding of the exponent's argument; exp2 itself 2^-22
            off = (dim + 4) * F32 * (np.abs(qs) @ np.abs(ks).T).max(
                1, keepdims=True) * scale + 2.0 ** -22
            # numerator and denominator each carry it; P rounds to bf16, and
            # both sums have kn terms (and up to 64 joins of pieces)
            bound[qf:qf + qn, h] = (p @ np.abs(vs)) * (
                BF16 + 2 * np.expm1(off) + 2 * (kn + 64) * F32)
    return o, bound * (1 + BF16) + BF16 * np.abs(o) + 1e-37, covered


def check(got_bits, want, bound, what=""):
    got = wide(got_bits, *want.shape)
    assert np.isfinite(got).all(), f"{what}: not finite"
    over = np.abs(got - want) - bound
    assert over.max() <= 0, (
        f"{what}: {int((over > 0).sum())}/{over.size} beyond the bound, worst "
        f"by {over.max():.3g} at {np.unravel_index(over.argmax(), over.shape)}")


def on_fake(code, env=None, **values):
    """What `code` leaves in `out`, run in a child whose HIP runtime launches
    nothing (fake_hip.cpp); it has h3hip, np, C (ctypes), gpu and `values`."""
    program = f"""
import ctypes as C, json, os, sys
import numpy as np
fake = C.CDLL({_fake()!r}, mode=C.RTLD_GLOBAL)
sys.path.insert(0, {os.path.join(ROOT, "h3.c_amd")!r})
import h3hip
globals().update(json.loads(sys.stdin.read()))
gpu = h3hip.Gpu()
def launches():
    got = []
    for i in range(fake.fake_launches()):
        text, words = C.create_string_buffer(400), (C.c_uint64 * 18)()
        fake.fake_launch(C.c_size_t(i), text, 400, words)
        got.append([text.value.decode()] + list(words[:5]))
    return got
def contents(t, words):
    at = C.c_void_p.from_address(t).value
    return np.ctypeslib.as_array((C.c_uint32 * words).from_address(at))
out = None
{code}
print("\\n" + json.dumps(out), flush=True)
os._exit(0)
"""
    done = subprocess.run([sys.executable, "-c", program],
                          input=json.dumps(values), text=True,
                          capture_output=True, timeout=120,
                          env={**os.environ, **(env or {})})
    assert done.returncode == 0, done.stderr[-2000:]
    return json.loads(done.stdout.splitlines()[-1])
