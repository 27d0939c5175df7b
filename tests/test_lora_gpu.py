"""Projections with low-rank adapters against the same in 64 bits, at the
bounds of requests_oracle."""
import os
import subprocess
import sys

import numpy as np
import pytest

import requests_oracle as ro
from conftest import ROOT, rand_bf16, to_f32

pytestmark = pytest.mark.gpu
NONE = ro.NONE


def make(seed, ids, ranks, k, n, bias=True, scale=0.05):
    rng = np.random.default_rng(seed)
    return dict(
        x=rand_bf16(rng, len(ids) * k), w=rand_bf16(rng, n * k, scale),
        b=rand_bf16(rng, n) if bias else None,
        down=[rand_bf16(rng, r * k, scale) for r in ranks],
        up=[rand_bf16(rng, n * r, 0.2) for r in ranks], ranks=list(ranks),
        scales=[float(s) for s in rng.uniform(0.5, 2, len(ranks))],
        ids=np.asarray(ids, np.uint32), k=k, n=n)


def table_of(gpu, a):
    return gpu.lora_table(
        [gpu.bf16(d) if len(d) else None for d in a["down"]],
        [gpu.bf16(u) if len(u) else None for u in a["up"]], a["ranks"],
        a["scales"], a["k"], a["n"])


def run(gpu, a, act=False, table=None, extra=0):
    """The output and `extra` elements behind it."""
    rows, n = len(a["ids"]), a["n"]
    table = table or table_of(gpu, a)
    y = gpu.bf16(np.full(rows * n + extra, 0x4141, np.uint16))
    gpu.run("h3_hip_linear_lora_gelu_bf16" if act else
            "h3_hip_linear_lora_bf16", y, gpu.bf16(a["x"]), gpu.bf16(a["w"]),
            None if a["b"] is None else gpu.bf16(a["b"]), table,
            gpu.u32(a["ids"]), rows, a["k"], n)
    return gpu.read_bf16(y)


def check(gpu, a, act=False, what=""):
    rows, n = len(a["ids"]), a["n"]
    got = run(gpu, a, act, extra=64)
    assert (got[rows * n:] == 0x4141).all(), "wrote behind the last row"
    want, bound = ro.lora(act=act, **a)
    ro.check(got[:rows * n], want, bound, what)
    return got[:rows * n]


def spread(rows, adapters, seed):
    """Each row its own adapter, some of them none, in any order."""
    return np.random.default_rng(seed).choice(
        [*range(adapters), adapters, NONE], rows)


def blocks(*sizes):
    """sizes: (rows, adapter) one after the other."""
    return np.concatenate([np.full(r, a, np.uint32) for r, a in sizes])


# rows around the 32-, 128- and 256-row steps of the tiles; one request
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 96, 97,
                                  127, 128, 129, 160, 161, 255, 256, 257, 300,
                                  513])
def test_rows(gpu, rows):
    check(gpu, make(rows, np.zeros(rows), [16], 256, 320))


@pytest.mark.parametrize("rank", [0, 1, 7, 8, 9, 16, 17, 24, 31, 32, 33, 40, 63,
                                  64, 65, 96, 128, 129, 200, 320])
@pytest.mark.parametrize("rows", [5, 200])
def test_ranks(gpu, rank, rows):
    check(gpu, make(rank, blocks((rows // 2, 1), (rows - rows // 2, 0)),
                    [rank, 8], 192, 260))


@pytest.mark.parametrize("rows", [1, 40, 128, 129, 300])
@pytest.mark.parametrize("act", [False, True])
@pytest.mark.parametrize("bias", [False, True])
def test_rows_of_every_adapter_in_any_order(gpu, rows, act, bias):
    check(gpu, make(rows, spread(rows, 7, rows), [4, 16, 0, 33, 64, 8, 128],
                    320, 516, bias=bias), act)


# K and N that the matrix-core kernels take and that they do not
@pytest.mark.parametrize("k,n", [(64, 4), (64, 256), (128, 260), (448, 1000),
                                 (512, 33), (100, 64), (1, 1), (63, 250),
                                 (65, 132), (2688, 388), (1024, 2308)])
@pytest.mark.parametrize("rows", [3, 150])
def test_widths(gpu, k, n, rows):
    check(gpu, make(k * n, blocks((rows - 1, 0), (1, 1)), [12, 20], k, n))


@pytest.mark.parametrize("rows,k,n", [
    (129, 5120, 5120), (512, 5120, 1536), (778, 7168, 640),
    (1100, 5376, 2052), (40, 5376, 33000), (128, 512, 36000),
    (700, 192, 20480), (2000, 320, 13824)])
def test_long_and_wide(gpu, rows, k, n):
    """Split sums, whole tiles and both, several rounds of tiles."""
    third = rows // 3
    check(gpu, make(rows + k, blocks((third, 0), (third, NONE),
                                     (rows - 2 * third, 1)), [16, 64], k, n,
                    scale=0.02))


@pytest.mark.parametrize("rows,k,n", [
    (129, 64, 132), (200, 64, 4), (300, 192, 4100), (417, 448, 1004),
    (545, 2688, 260), (641, 320, 5120), (1800, 512, 388), (259, 1280, 12900),
    (130, 5120, 13700), (161, 5120, 13824), (224, 5120, 13600),
    (150, 1024, 34000)])
def test_groups_of_rows(gpu, rows, k, n):
    """Over 128 rows of few steps of K or many columns: groups of 96 and 128
    rows, a last one of few, one of 160, 192 and 224, whole sums and pieces,
    one round of workgroups and more."""
    check(gpu, make(rows + n, blocks((rows // 2, 1), (rows // 4, NONE),
                                     (rows - rows // 2 - rows // 4, 0)),
                    [64, 16], k, n))
    check(gpu, make(rows + k, spread(rows, 4, 2), [16, 40, 8, 100], k, n,
                    bias=False), True)


def test_no_row_has_an_adapter(gpu):
    """The same as the projection alone, to its own rounding."""
    for rows in (7, 128, 300):
        a = make(3, np.full(rows, 2), [16, 8], 256, 512)
        got = check(gpu, a)
        y = gpu.new_bf16(rows * 512)
        gpu.run("h3_gpu_linear_bf16", y, gpu.bf16(a["x"]), gpu.bf16(a["w"]),
                gpu.bf16(a["b"]), rows, 256, 512)
        assert (np.abs(to_f32(got) - to_f32(gpu.read_bf16(y))) <=
                2.0 ** -7 * np.abs(to_f32(got)) + 1e-5).all()


@pytest.mark.parametrize("rows", [60, 300])
def test_a_row_reaches_no_other(gpu, rows):
    """NaN and infinities in rows of one request stay there."""
    ids = spread(rows, 3, 1)
    a = make(5, ids, [16, 33, 8], 256, 320)
    x = a["x"].reshape(rows, 256).copy()
    x[::7, 3] = 0x7FC0
    x[3::7, 200] = 0xFF80
    bad = np.zeros(rows, bool)
    bad[::7] = bad[3::7] = True
    want, bound = ro.lora(**a)
    a["x"] = x.reshape(-1)
    got = run(gpu, a).reshape(rows, 320)
    ro.check(got[~bad], want[~bad], bound[~bad])
    assert not np.isfinite(to_f32(got[bad])).any()


@pytest.mark.parametrize("rows", [9, 200])
def test_products_past_the_types_range_are_infinite(gpu, rows):
    """x . down^T past the largest bf16 value: the row is infinite, not NaN."""
    a = make(6, np.zeros(rows), [8], 64, 64)
    a["x"] = ro_bits(np.full(rows * 64, 3e38))
    a["down"] = [ro_bits(np.full(8 * 64, 1.0))]
    a["up"] = [ro_bits(np.full(8 * 64, 1.0))]
    a["w"] = ro_bits(np.zeros(64 * 64))
    got = to_f32(run(gpu, a))
    assert (got == np.inf).all()


@pytest.mark.parametrize("rows", [9, 200])
@pytest.mark.parametrize("rank", [1, 4, 20, 40])
def test_an_infinity_against_positive_adapters_is_one(gpu, rows, rank):
    """It meets the ranks there are, not their padding (0 times it is NaN)."""
    a = make(16, np.zeros(rows), [rank], 64, 64)
    x = np.ones((rows, 64))
    x[::3, 5] = np.inf
    a.update(x=ro_bits(x.reshape(-1)), w=ro_bits(np.ones(64 * 64)),
             down=[ro_bits(np.ones(rank * 64))],
             up=[ro_bits(np.ones(rank * 64))])
    got = to_f32(run(gpu, a)).reshape(rows, 64)
    assert (got[::3] == np.inf).all()
    assert np.isfinite(np.delete(got, np.s_[::3], 0)).all()


@pytest.mark.parametrize("rows", [12, 300])
def test_gelu_of_the_sum_itself(gpu, rows):
    """One rounding.  From -2 up F32 leaves an error under 2^-16 of the result,
    so that under one result in 2^7 lies so near a border between two bf16
    values that it may fall to the other; rounded twice, many would."""
    a = make(17, np.zeros(rows), [16], 256, 512)
    got = to_f32(run(gpu, a, True)).astype(np.float64)
    sums, _ = ro.lora(**a)
    nearest = to_f32(ro_bits(ro.gelu(sums))).reshape(-1)
    up = sums.reshape(-1) > -2
    assert up.sum() > 1000 and (got != nearest)[up].mean() < 2.0 ** -7


def ro_bits(values):
    import oracle
    return oracle.bf16(np.asarray(values, np.float32))


@pytest.mark.parametrize("which", ["down", "up"])
@pytest.mark.parametrize("value", [0x7F80, 0xFF80, 0x7FC1])
def test_adapters_that_are_not_finite_are_refused(gpu, which, value):
    a = make(7, [0], [4, 12], 64, 100)
    a[which][1] = a[which][1].copy()
    a[which][1][-1] = value
    with pytest.raises(RuntimeError, match="adapter 1 holds values"):
        table_of(gpu, a)


def test_the_table_keeps_its_own_copy(gpu):
    a = make(8, np.zeros(70), [20], 128, 256)
    down, up = gpu.bf16(a["down"][0]), gpu.bf16(a["up"][0])
    table = gpu.lora_table([down], [up], a["ranks"], a["scales"], 128, 256)
    for t, n in ((down, 20 * 128), (up, 20 * 256)):
        z = np.zeros(n, np.uint16)
        import h3hip
        assert gpu.L.h3_gpu_tensor_write_bf16(t, h3hip.ptr(z), n)
        gpu.free(t)
    want, bound = ro.lora(**a)
    ro.check(run(gpu, a, table=table), want, bound)


@pytest.mark.parametrize("rows", [8, 300])
def test_the_same_call_gives_the_same_bits(gpu, rows):
    a = make(9, spread(rows, 4, 2), [16, 8, 33, 64], 1024, 512)
    table = table_of(gpu, a)
    first = run(gpu, a, table=table)
    other = make(10, spread(rows, 2, 3), [128, 4], 1024, 512)
    run(gpu, other)
    assert (run(gpu, a, table=table) == first).all()


def test_calls_queued_one_after_the_other(gpu):
    """Two sizes and two tables in one batch share the context's scratch."""
    calls = [make(11, spread(20, 3, 4), [16, 8, 40], 512, 768),
             make(12, np.zeros(400), [128], 512, 768),
             make(13, np.zeros(1), [4], 512, 768)]
    made = []
    for a in calls * 2:
        made.append((a, gpu.new_bf16(len(a["ids"]) * a["n"]),
                     gpu.bf16(a["x"]), gpu.bf16(a["w"]), gpu.bf16(a["b"]),
                     table_of(gpu, a), gpu.u32(a["ids"])))
    gpu.begin()
    for a, y, x, w, b, t, ids in made:
        assert gpu.L.h3_hip_linear_lora_bf16(
            gpu.h, y, x, w, b, t, ids, len(a["ids"]), a["k"], a["n"])
    gpu.submit()
    for a, y, *_ in made:
        want, bound = ro.lora(**a)
        ro.check(gpu.read_bf16(y), want, bound)


@pytest.mark.parametrize("rows,adapters,k,n", [
    (100, 100, 256, 320), (128, 70, 64, 132), (300, 280, 192, 260),
    (2000, 300, 320, 5120)])
def test_more_adapters_than_lanes_or_rows_of_a_tile(gpu, rows, adapters, k, n):
    check(gpu, make(20, np.arange(rows) * 7 % adapters, [2] * adapters, k, n))


def test_two_contexts_at_once(gpu):
    """Each with its own scratch; a table serves both."""
    import h3hip
    with h3hip.Gpu() as other:
        a = make(21, spread(500, 3, 1), [16, 8, 40], 512, 768)
        b = make(22, spread(90, 3, 2), [64, 4, 20], 1024, 512)
        shared = table_of(gpu, a)
        made = []
        for g, c, table in ((gpu, a, shared), (other, a, shared),
                            (gpu, b, None), (other, b, None)):
            made.append((g, c, table or table_of(g, c),
                         [g.new_bf16(len(c["ids"]) * c["n"]) for _ in "123"],
                         g.bf16(c["x"]), g.bf16(c["w"]), g.bf16(c["b"]),
                         g.u32(c["ids"])))
        gpu.begin()
        other.begin()
        for turn in range(3):
            for g, c, table, y, x, w, bias, ids in made:
                g.check(g.L.h3_hip_linear_lora_bf16(
                    g.h, y[turn], x, w, bias, table, ids, len(c["ids"]),
                    c["k"], c["n"]))
        other.submit()
        gpu.submit()
        for g, c, table, y, *_ in made:
            want, bound = ro.lora(**c)
            for t in y:
                ro.check(g.read_bf16(t), want, bound)


def test_simple_kernels(gpu):
    """H3_HIP_REFERENCE=1 takes the sequential kernels, at the same bounds."""
    code = """
import sys
sys.path[:0] = sys.argv[1:]
import h3hip, test_lora_gpu as t, numpy as np
gpu = h3hip.Gpu()
for act in (False, True):
    t.check(gpu, t.make(1, t.spread(50, 3, 1), [4, 16, 33], 256, 300), act)
print("fine")
"""
    done = subprocess.run(
        [sys.executable, "-c", code] + [os.path.join(ROOT, d) for d in (
            "h3.c_amd", "oracle", "tests")], capture_output=True, text=True,
        env={**os.environ, "H3_HIP_REFERENCE": "1"}, timeout=100)
    assert done.returncode == 0 and "fine" in done.stdout, done.stderr[-2000:]
