"""8-bit matrices and caches of more than 2^32 bytes, at rows on both sides of
every 2^32."""
import numpy as np
import pytest

import int8_oracle as io
import requests_oracle as ro
from conftest import rand_bf16
from test_int8_gpu import quantize

pytestmark = pytest.mark.gpu

COLUMNS, ROWS = 4096, 1100000  # 4.5e9 bytes of codes


@pytest.fixture(scope="module")
def far(gpu):
    """An 8-bit matrix of rows that repeat every 1000, in another order at both
    ends, and the rows at `at` in 64 bits."""
    rng = np.random.default_rng(1)
    x = rand_bf16(rng, 1000 * COLUMNS).reshape(1000, COLUMNS)
    source = gpu.new_bf16(ROWS * COLUMNS)
    part = gpu.bf16(x)
    gpu.begin()
    for i in range(ROWS // 1000):
        gpu.check(gpu.L.h3_gpu_copy_bf16(gpu.h, source, i * x.size, part, 0,
                                         x.size), "copy")
    gpu.submit()
    border = 2 ** 32 // COLUMNS
    at = np.r_[0:40, border - 40:border + 40, ROWS - 40:ROWS]
    t = gpu.int8(ROWS, COLUMNS)
    gpu.run("h3_hip_quantize_int8", t, source, ROWS, COLUMNS)
    gpu.free(source)
    yield t, at, io.rows_of(ro.wide(x, 1000, COLUMNS)), at % 1000
    gpu.free(t)


@pytest.mark.parametrize("n", [8, 300])
def test_rows(gpu, far, n):
    t, at, rows, which = far
    w = rand_bf16(np.random.default_rng(n), n * COLUMNS, 0.05)
    y = gpu.new_bf16(ROWS * n)
    gpu.run("h3_hip_linear_int8_bf16", y, t, quantize(gpu, w, n, COLUMNS),
            None, ROWS, COLUMNS, n)
    got = gpu.read_bf16(y).reshape(ROWS, n)
    want, bound = io.product(rows, io.rows_of(ro.wide(w, n, COLUMNS)))
    ro.check(got[at], want[which], io.rounded(want, bound)[which])
    # and all the others of the same row
    whole = got.reshape(ROWS // 1000, 1000, n)
    assert (whole == whole[:1]).all()
    gpu.free(y)


@pytest.mark.parametrize("m", [1, 5])
def test_weights(gpu, far, m):
    """(which the simple kernel takes)"""
    t, at, rows, which = far
    x = rand_bf16(np.random.default_rng(m), m * COLUMNS)
    y = gpu.new_bf16(m * ROWS)
    gpu.run("h3_hip_linear_int8_bf16", y, quantize(gpu, x, m, COLUMNS), t,
            None, m, COLUMNS, ROWS)
    got = gpu.read_bf16(y).reshape(m, ROWS)
    want, bound = io.product(io.rows_of(ro.wide(x, m, COLUMNS)), rows)
    ro.check(got[:, at], want[:, which], io.rounded(want, bound)[:, which])
    whole = got.reshape(m, ROWS // 1000, 1000)
    assert (whole == whole[:, :1]).all()
    gpu.free(y)


@pytest.mark.parametrize("qn", [1, 200])
def test_cache(gpu, qn):
    """Rows around byte 2^32 of the cache, and at its end."""
    heads, kv_heads, dim, room = 16, 8, 128, 2200000
    border = 2 ** 32 // (2 * kv_heads * dim) // 64 * 64
    places = [0, border - 64, 64 * ((room - 200) // 64)]
    counts = [70, 130, 190]
    rng = np.random.default_rng(qn)
    width = kv_heads * dim
    kv = rand_bf16(rng, sum(counts) * 2 * width)
    d, t = gpu.bf16(kv), gpu.kv_int8(room, kv_heads, dim)
    source = [0, 70, 200]
    gpu.begin()
    gpu.kv_int8_store(t, places, source, counts, d, 0, d, width, 2 * width)
    gpu.submit()
    rows = ro.wide(kv, sum(counts), 2, kv_heads, dim)
    wide, near = io.Cache(64 * 8, kv_heads, dim), [0, 128, 320]
    for f, s, n in zip(near, source, counts):
        wide.store(f, rows[s:s + n])
    k, v = gpu.new_bf16(190 * width), gpu.new_bf16(190 * width)
    for f, to, n in zip(places, near, counts):
        gpu.run("h3_hip_kv_int8_read", k, v, t, f, n)
        want = io.values(wide.c, wide.steps())[to:to + n]
        for i, got in enumerate((k, v)):
            got = gpu.read_bf16(got)[:n * width].reshape(n, kv_heads, dim)
            assert np.array_equal(got & 0x7fff, want[:, i] & 0x7fff)
    q = rand_bf16(rng, 3 * qn * heads * dim)
    first, scale = [0, qn, 2 * qn], float(np.float32(dim ** -0.5))
    plan = gpu.sdpa_packed_plan(first, [qn] * 3, places, counts, heads,
                                kv_heads, dim)
    y = gpu.new_bf16(3 * qn * heads * dim)
    gpu.run("h3_hip_sdpa_packed_int8_bf16", y, gpu.bf16(q), 0, heads * dim, t,
            plan, scale)
    want, bound, _ = io.attention(
        ro.wide(q, 3 * qn, heads, dim), wide,
        list(zip(first, [qn] * 3, near, counts)), heads, kv_heads, dim, scale)
    ro.check(gpu.read_bf16(y).reshape(3 * qn, heads, dim), want, bound)
    for p in (t, d, k, v, y):
        gpu.free(p)
