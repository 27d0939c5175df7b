"""The 8-bit products and gated block at shapes that between them run every
kernel (PRODUCTS and GATED; test_int8_routes.py holds each to its kernels), at
odd sizes, against the same in 64 bits and, bit for bit, the simple kernels."""
import numpy as np
import pytest

import int8_oracle as io
import requests_oracle as ro
from conftest import rand_bf16
from test_int8_gpu import MARK, Product, plain, quantize  # noqa: F401

pytestmark = pytest.mark.gpu

# rows, input and output columns: the kernels, hk_int8_ left out
PRODUCTS = {
    (1, 300, 77): ["dot<1, false>"], (1, 1283, 20001): ["dot<2, false>"],
    (106, 104, 129): ["narrow<2, false>"],
    (417, 1943, 600): ["narrow<1, false>"],
    (513, 130, 1287): ["skinny<1, false>"],
    (116, 134, 9708): ["skinny<2, false>"],
    (139, 134, 11313): ["skinny<3, false>"],
    (510, 129, 5517): ["skinny<4, false>"],
    (243, 2885, 1048): ["skinny<1, false>", "skinny_reduce<false>"],
    (294, 4108, 1026): ["skinny<2, false>", "skinny_reduce<false>"],
    (702, 5089, 651): ["skinny<3, false>", "skinny_reduce<false>"],
    (327, 5013, 1905): ["skinny<4, false>", "skinny_reduce<false>"],
    (572, 1831, 11655): ["gemm<0, false, 4>"],
    (776, 836, 11577): ["gemm<0, false, 5>"],
    (516, 680, 8548): ["gemm<0, false, 6>"],
    (416, 794, 11619): ["gemm<0, false, 7>"],
    (1517, 104, 3021): ["gemm<0, false, 8>"],
    # the tiles of a last, sparse round, or all, in pieces of K
    (1409, 1261, 11987): ["gemm<0, false, 8>", "gemm<3, false, 8>",
                          "tile_reduce"],
    (293, 4031, 12329): ["gemm<3, false, 5>", "tile_reduce"],
    (516, 4559, 7238): ["gemm<3, false, 6>", "tile_reduce"],
    (466, 4852, 8611): ["gemm<3, false, 8>", "tile_reduce"],
}

# rows, input and hidden columns: the kernels of the first product
GATED = {
    (1, 300, 77): ["dot<2, true>"], (63, 110, 65): ["narrow<2, true>"],
    (1693, 107, 68): ["narrow<1, true>"],
    (100, 129, 2966): ["skinny<1, true>"],
    (131, 135, 3844): ["skinny<2, true>"],
    (4501, 130, 234): ["skinny<3, true>"],
    (319, 131, 4517): ["skinny<4, true>"],
    (141, 2835, 821): ["skinny<1, true>", "skinny_reduce<true>"],
    (299, 5038, 393): ["skinny<2, true>", "skinny_reduce<true>"],
    (1096, 5022, 202): ["skinny<3, true>", "skinny_reduce<true>"],
    (1473, 7142, 150): ["skinny<4, true>", "skinny_reduce<true>"],
    (815, 1658, 4146): ["gemm<1, false, 4>"],
    (1633, 980, 2390): ["gemm<1, false, 5>"],
    (533, 669, 4030): ["gemm<1, false, 6>"],
    (1559, 850, 1325): ["gemm<1, false, 7>"],
    (1157, 111, 1987): ["gemm<1, false, 8>"],
    (1293, 900, 6406): ["gemm<1, false, 8>", "gemm<4, false, 8>",
                        "gated_reduce"],
    (284, 4274, 6136): ["gemm<4, false, 5>", "gated_reduce"],
    (328, 5020, 5894): ["gemm<4, false, 6>", "gated_reduce"],
    (1029, 4946, 1869): ["gemm<4, false, 8>", "gated_reduce"],
}
OUT = 130  # columns of the gated block's second product


@pytest.mark.parametrize("m,k,n", PRODUCTS)
def test_product(gpu, plain, m, k, n):  # noqa: F811
    p = Product(m, k, n)
    got, act = p.run(gpu), p.run(gpu, act=True)
    y, bound = io.product(*p.sides(), p.b)
    ro.check(got, y, io.rounded(y, bound))
    # as io.product has it
    bound = 1.13 * bound + 2.0 ** -20 * np.abs(y)
    y = ro.gelu(y)
    ro.check(act, y, io.rounded(y, bound), "GELU")
    assert np.array_equal(got, p.run(plain))
    assert np.array_equal(p.run(gpu, bias=False, room=3),
                          p.run(plain, bias=False))
    assert np.array_equal(act, p.run(plain, act=True))


@pytest.mark.parametrize("m,k,h", GATED)
def test_gated_block(gpu, m, k, h):
    rng = np.random.default_rng((m, k, h))
    x, w1 = rand_bf16(rng, m * k), rand_bf16(rng, 2 * h * k, 1.5 * k ** -0.5)
    w2 = rand_bf16(rng, OUT * h, h ** -0.5)
    sides = [quantize(gpu, x, m, k), quantize(gpu, w1, 2 * h, k),
             quantize(gpu, w2, OUT, h)]

    def run():
        y = gpu.bf16(np.full(m * OUT + 512, MARK, np.uint16))
        gpu.run("h3_hip_mlp_int8_bf16", y, *sides, m, k, h, OUT)
        return gpu.read_bf16(y)
    got = run()
    assert (got[m * OUT:] == MARK).all(), "wrote behind the last row"
    assert np.array_equal(got, run()), "other bits the second time"
    want, bound = io.mlp(io.rows_of(ro.wide(x, m, k)),
                         io.rows_of(ro.wide(w1, 2 * h, k)),
                         io.rows_of(ro.wide(w2, OUT, h)))
    ro.check(got[:m * OUT].reshape(m, OUT), want, io.rounded(want, bound))


@pytest.mark.parametrize("m,k,n", [(106, 104, 129), (510, 129, 5517),
                                   (327, 5013, 1905), (1517, 104, 3021),
                                   (293, 4031, 12329)])
def test_a_bad_row_stays_alone(gpu, m, k, n):
    """Infinities and NaN of one row or channel reach no other."""
    p = Product(m, k, n)
    want = p.run(gpu)
    x, w = p.x.reshape(m, k), p.w.reshape(n, k)
    x[7, 3], x[m - 1, k - 1], w[40, 0] = 0x7f80, 0x7fc0, 0xff80
    got = p.run(gpu)
    bad = np.zeros((m, n), bool)
    bad[[7, m - 1]] = True
    bad[:, 40] = True
    assert np.isnan(ro.wide(got[bad], -1)).all()
    assert np.array_equal(got[~bad], want[~bad])


@pytest.mark.parametrize("m,k,h,n", [(1, 300, 777, 130), (37, 300, 777, 130),
                                     (1517, 104, 3021, 257)])
def test_ungated_block(gpu, m, k, h, n):
    """A product with GELU, whose rows, in bf16 there, are those of a second
    one in 8 bits."""
    rng = np.random.default_rng((m, k, h))
    x, w1 = rand_bf16(rng, m * k), rand_bf16(rng, h * k, k ** -0.5)
    w2, b = rand_bf16(rng, n * h, h ** -0.5), rand_bf16(rng, h, 0.3)
    x8, a8 = quantize(gpu, x, m, k), quantize(gpu, w1, h, k)
    b8, h8 = quantize(gpu, w2, n, h), gpu.int8(m, h)
    hidden, y, bias = gpu.new_bf16(m * h), gpu.new_bf16(m * n), gpu.bf16(b)
    gpu.begin()
    for name, *args in (
            ("linear_gelu_int8_bf16", hidden, x8, a8, bias, m, k, h),
            ("quantize_int8", h8, hidden, m, h),
            ("linear_int8_bf16", y, h8, b8, None, m, h, n)):
        gpu.check(getattr(gpu.L, "h3_hip_" + name)(gpu.h, *args), name)
    gpu.submit()
    got = gpu.read_bf16(hidden).reshape(m, h)
    want, bound = io.product(io.rows_of(ro.wide(x, m, k)),
                             io.rows_of(ro.wide(w1, h, k)), b, True)
    ro.check(got, want, io.rounded(want, bound))
    want, bound = io.product(io.rows_of(ro.wide(got, m, h)),
                             io.rows_of(ro.wide(w2, n, h)))
    ro.check(gpu.read_bf16(y).reshape(m, n), want, io.rounded(want, bound))
