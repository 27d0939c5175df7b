"""An adapter whose padded B has more elements than one launch has threads."""
import numpy as np
import pytest

import requests_oracle as ro
from conftest import rand_bf16, to_f32

pytestmark = pytest.mark.gpu

RANK, K, N = 1024, 64, 1_100_000


def test_the_last_columns_of_a_large_adapter(gpu):
    """They are copied, and looked at for values that are not finite."""
    assert RANK * N > (1 << 22) * 256
    rng = np.random.default_rng(61)
    x, d = rand_bf16(rng, 2 * K), rand_bf16(rng, RANK * K, 0.05)
    w, u = rand_bf16(rng, 4 * K, 0.05), rand_bf16(rng, 4 * RANK, 0.05)

    def put(t, at, bits):
        gpu.run("h3_gpu_copy_bf16", t, at, gpu.bf16(bits), 0, bits.size)

    weight, up, y = (gpu.new_bf16(s) for s in (N * K, N * RANK, 2 * N))
    for t, size in ((weight, N * K), (up, N * RANK)):
        gpu.check(gpu.L.h3_gpu_fill_normal_bf16(gpu.h, t, 0, size, 1, 0.0,
                                                0.02))
    put(weight, (N - 4) * K, w)
    down = gpu.bf16(d)
    bad = u.copy()
    bad[-1] = 0x7F80
    put(up, (N - 4) * RANK, bad)
    with pytest.raises(RuntimeError, match="adapter 0 holds values"):
        gpu.lora_table([down], [up], [RANK], [0.5], K, N)
    put(up, (N - 4) * RANK, u)
    table = gpu.lora_table([down], [up], [RANK], [0.5], K, N)
    gpu.run("h3_hip_linear_lora_bf16", y, gpu.bf16(x), weight, None, table,
            gpu.u32([0, 1]), 2, K, N)
    got = gpu.read_bf16(y).reshape(2, N)
    want, bound = ro.lora(x, w, None, [d], [u], [RANK], [0.5],
                          np.array([0, 1], np.uint32), K, 4)
    ro.check(got[:, -4:].copy(), want, bound)
    assert np.isfinite(to_f32(got)).all()
    for t in (weight, up, y, table):
        gpu.free(t)
