"""Rows in 8 bits, their products and the gated block, against the same in 64
bits at the bounds of int8_oracle."""
import ctypes as C

import numpy as np
import pytest

import int8_oracle as io
import requests_oracle as ro
from conftest import rand_bf16

pytestmark = pytest.mark.gpu

MARK = 0x4141  # what outputs hold before a call


@pytest.fixture(scope="module")
def plain():
    """A context of the simple kernels."""
    import os
    import h3hip
    os.environ["H3_HIP_REFERENCE"] = "1"
    try:
        g = h3hip.Gpu()
    finally:
        del os.environ["H3_HIP_REFERENCE"]
    yield g
    g.close()


@pytest.fixture(params=["fast", "simple"])
def ctx(request, gpu):
    return gpu if request.param == "fast" else \
        request.getfixturevalue("plain")


def quantize(gpu, x, rows, columns, room=None):
    t = gpu.int8(room or rows, columns)
    gpu.run("h3_hip_quantize_int8", t, gpu.bf16(x), rows, columns)
    return t


def read(gpu, t, rows, columns):
    y = gpu.bf16(np.full(rows * columns + 64, MARK, np.uint16))
    gpu.run("h3_hip_dequantize_int8", y, t, rows, columns)
    got = gpu.read_bf16(y)
    assert (got[rows * columns:] == MARK).all(), "wrote behind the last row"
    return got[:rows * columns].reshape(rows, columns)


def same(got, want):
    nan = (want & 0x7fff) > 0x7f80
    assert np.array_equal(nan, (got & 0x7fff) > 0x7f80)
    # -0 is 0
    a, b = (np.where(v == 0x8000, 0, v)[~nan] for v in (got, want))
    assert np.array_equal(a, b), f"{int((a != b).sum())} of {a.size} differ"


WIDTHS = [1, 2, 7, 8, 63, 64, 127, 128, 129, 256, 1000, 2048, 2056, 5376, 8192,
          8200, 14336, 16384, 16392, 20001]


@pytest.mark.parametrize("columns", WIDTHS)
@pytest.mark.parametrize("rows", [1, 3, 65])
def test_rows(ctx, rows, columns):
    x = rand_bf16(np.random.default_rng(columns), rows * columns)
    got = read(ctx, quantize(ctx, x, rows, columns), rows, columns)
    same(got, io.values(*(v if v.ndim == 2 else v[:, None] for v in io.rows_of(
        ro.wide(x, rows, columns)))))


def test_rows_at_borders(ctx):
    """Halves of the largest, one value alone, zeros, the ends of the range,
    subnormal values, infinities and NaN in one row."""
    n = 320
    x = np.zeros((12, n))
    x[0, :3] = 1.0, 0.5, -0.5
    x[1, 5] = -3.0
    x[3] = np.arange(n) / 64
    x[4, :4] = 3.3895313892515355e38, 1.69e38, -3e36, 1e-38
    x[5, :4] = 2.0 ** -133, 2.0 ** -132, -2.0 ** -133, 0
    x[6, :3] = 1.0, np.inf, 2.0
    x[7, :3] = 1.0, np.nan, 2.0
    x[8] = 1.0
    x[9, :3] = 254.0, 1.0, 127.0  # steps of 2: halves all along
    x[9, 3:258] = np.arange(255)
    x[10, -1] = -np.inf
    x[11, :2] = 2.0 ** -126, 2.0 ** -127
    with np.errstate(over="ignore"):
        b = io.bits(x.astype(np.float32))
    got = read(ctx, quantize(ctx, b.ravel(), 12, n), 12, n)
    c, s = io.rows_of(ro.wide(b, 12, n))
    same(got, io.values(c, s[:, None]))


def test_rows_behind_the_call_stay(gpu):
    x = rand_bf16(np.random.default_rng(1), 9 * 200)
    t = quantize(gpu, x, 9, 200)
    before = read(gpu, t, 9, 200)
    gpu.run("h3_hip_quantize_int8", t, gpu.bf16(x[::-1].copy()), 4, 200)
    after = read(gpu, t, 9, 200)
    assert np.array_equal(before[4:], after[4:])
    assert not np.array_equal(before[:4], after[:4])


@pytest.mark.parametrize("layer,parts", [(False, "all"), (True, "all"),
                                         (True, "bare")])
@pytest.mark.parametrize("rows,width", [(1, 8), (5, 513), (70, 1024),
                                        (3, 5376), (2, 9000), (2, 17000)])
def test_adaln(ctx, layer, rows, width, parts):
    """With every part, and (the LayerNorm) with none."""
    rng = np.random.default_rng(width)
    slots, shift, scale, eps = 3, 2, 0, 1e-5
    x = rand_bf16(rng, rows * width, 2.0, 0.5)
    w, b = rand_bf16(rng, width, 0.2, 1.0), rand_bf16(rng, width, 0.2)
    mod = rand_bf16(rng, 2 * slots * width, 0.3)
    at = rng.integers(0, 2, rows).astype(np.uint32)
    t = ctx.int8(rows, width)
    if not layer:
        ctx.run("h3_hip_adaln_int8", t, ctx.bf16(x), ctx.bf16(w),
                ctx.bf16(mod), ctx.u32(at), rows, width, slots, shift, scale,
                eps)
    elif parts == "all":
        ctx.run("h3_hip_layer_adaln_int8", t, ctx.bf16(x), ctx.bf16(w),
                ctx.bf16(b), ctx.bf16(mod), ctx.u32(at), rows, width, slots,
                shift, scale, eps)
    else:
        ctx.run("h3_hip_layer_adaln_int8", t, ctx.bf16(x), None, None, None,
                None, rows, width, 0, 0, 0, eps)
    wide = parts == "all"
    v, bound = io.norm(
        ro.wide(x, rows, width), ro.wide(w, width) if wide else None,
        ro.wide(b, width) if wide and layer else None,
        ro.wide(mod, 2, slots, width) if wide else None, at, shift, scale,
        float(np.float32(eps)), layer)
    c, s, doubtful, off = io.quantized(v, bound)
    want = c * s[:, None]
    # a doubtful code is one step off, every value by its scale's error
    ro.check(read(ctx, t, rows, width), want, io.rounded(
        want, doubtful * s[:, None] + np.abs(c) * off[:, None] +
        io.HALF * np.abs(want)))
    assert doubtful.mean() < 0.05


SHAPES = [(1, 1, 1), (1, 128, 4), (2, 130, 31), (5, 64, 33), (32, 256, 128),
          (33, 300, 129), (64, 1024, 96), (65, 129, 257), (97, 640, 500),
          (128, 2000, 260), (129, 128, 128), (130, 500, 1000), (200, 1283, 513),
          (256, 512, 256), (257, 384, 255), (300, 2049, 771), (513, 257, 300),
          (700, 896, 130), (1025, 128, 2), (1100, 640, 1111),
          (40, 256, 1030), (70, 3000, 640), (100, 2000, 2100),
          (150, 1283, 1411), (180, 2176, 129), (1500, 300, 100)]


class Product:
    def __init__(self, m, k, n, seed=0, std=1.0):
        rng = np.random.default_rng((m, k, n, seed))
        self.m, self.k, self.n = m, k, n
        self.x, self.w = rand_bf16(rng, m * k, std), rand_bf16(rng, n * k)
        self.b = rand_bf16(rng, n, 5.0)

    def sides(self):
        return (io.rows_of(ro.wide(self.x, self.m, self.k)),
                io.rows_of(ro.wide(self.w, self.n, self.k)))

    def run(self, gpu, act=False, bias=True, room=0):
        m, k, n = self.m, self.k, self.n
        y = gpu.bf16(np.full(m * n + 512, MARK, np.uint16))
        gpu.run("h3_hip_linear_gelu_int8_bf16" if act else
                "h3_hip_linear_int8_bf16", y,
                quantize(gpu, self.x, m, k, m + room),
                quantize(gpu, self.w, n, k, n + room),
                gpu.bf16(self.b) if bias else None, m, k, n)
        got = gpu.read_bf16(y)
        assert (got[m * n:] == MARK).all(), "wrote behind the last row"
        return got[:m * n].reshape(m, n)

    def check(self, gpu, act=False, bias=True, room=0):
        got = self.run(gpu, act, bias, room)
        y, bound = io.product(*self.sides(), self.b if bias else None, act)
        ro.check(got, y, io.rounded(y, bound))
        return got


@pytest.mark.parametrize("m,k,n", SHAPES)
def test_product(ctx, m, k, n):
    p = Product(m, k, n)
    p.check(ctx)
    p.check(ctx, bias=False, room=3)
    p.check(ctx, act=True)


@pytest.mark.parametrize("m,k,n", [(1, 14336, 200), (40, 7168, 640),
                                   (128, 14336, 1024), (129, 14336, 256),
                                   (512, 5376, 640), (2378, 512, 5376),
                                   (1536, 1024, 13824), (39, 2688, 40000)])
def test_product_sizes_of_models(gpu, m, k, n):
    """Pieces of K, several rounds of tiles, and their last, sparse round."""
    Product(m, k, n).check(gpu)


def test_sums_do_not_overflow(ctx):
    """The longest rows, all codes at the end of the range."""
    k = 131072
    x = np.full((3, k), 1.0, np.float32)
    x[1] = -1
    x[2, ::2] = -1
    w = np.full((5, k), 2.0, np.float32)
    w[3] = -2
    p = Product(3, k, 5)
    p.x, p.w = io.bits(x).ravel(), io.bits(w).ravel()
    got = p.check(ctx, bias=False)
    assert io.bits(np.float32(2 * k)) == got[0, 0]


def test_a_bad_row_stays_alone(ctx):
    """Infinities and NaN of one row or channel reach no other."""
    p = Product(200, 300, 150)
    x, w = p.x.reshape(200, 300), p.w.reshape(150, 300)
    x[7, 3], x[150, 299], w[40, 0] = 0x7f80, 0x7fc0, 0xff80
    got = ro.wide(p.run(ctx), 200, 150)
    bad = np.zeros((200, 150), bool)
    bad[[7, 150]] = True
    bad[:, 40] = True
    assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()


def test_scales_far_apart(ctx):
    """Rows of 1e30 and 1e-30, weights of 1e-20 and 1e8."""
    p = Product(130, 256, 140)
    x = ro.wide(p.x, 130, 256) * np.where(np.arange(130) % 2, 1e30,
                                          1e-30)[:, None]
    w = ro.wide(p.w, 140, 256) * np.where(np.arange(140) % 3, 1e-20,
                                          1e4)[:, None]
    p.x, p.w = (io.bits(v.astype(np.float32)).ravel() for v in (x, w))
    p.check(ctx, bias=False)


MLPS = [(1, 8, 1, 1), (1, 130, 64, 32), (3, 200, 333, 70), (33, 512, 640, 512),
        (128, 256, 130, 129), (129, 128, 128, 128), (200, 300, 777, 129),
        (257, 1001, 300, 255), (600, 512, 1536, 512)]


@pytest.mark.parametrize("m,k,h,n", MLPS)
def test_gated_block(ctx, m, k, h, n):
    rng = np.random.default_rng((m, k, h))
    x, w1 = rand_bf16(rng, m * k), rand_bf16(rng, 2 * h * k, 1.5 * k ** -0.5)
    w2 = rand_bf16(rng, n * h, h ** -0.5)
    y = ctx.bf16(np.full(m * n + 512, MARK, np.uint16))
    ctx.run("h3_hip_mlp_int8_bf16", y, quantize(ctx, x, m, k),
            quantize(ctx, w1, 2 * h, k), quantize(ctx, w2, n, h), m, k, h, n)
    got = ctx.read_bf16(y)
    assert (got[m * n:] == MARK).all(), "wrote behind the last row"
    want, bound = io.mlp(io.rows_of(ro.wide(x, m, k)),
                         io.rows_of(ro.wide(w1, 2 * h, k)),
                         io.rows_of(ro.wide(w2, n, h)))
    ro.check(got[:m * n].reshape(m, n), want, io.rounded(want, bound))


def test_results_repeat(gpu):
    """Sums in whole numbers: the same bits each time."""
    for m, k, n in ((300, 2049, 771), (40, 7168, 640)):
        p = Product(m, k, n)
        first = p.run(gpu)
        for _ in range(3):
            assert np.array_equal(first, p.run(gpu))


def test_fast_and_simple_agree(gpu, plain):
    """The same sums, scales and roundings: the same bits."""
    for m, k, n in SHAPES[4:16:3]:
        p = Product(m, k, n)
        assert np.array_equal(p.run(gpu), p.run(plain))
