"""The 8-bit operators as a server of several requests runs them: a block of a
packed forward (adaLN in 8 bits, products, attention over the 8-bit cache of
the requests' texts, the gated block behind its norm), then single rows whose
keys and values join the cache.  Each stage is held against the same in 64 bits
of what the device has as its input."""
import threading

import numpy as np
import pytest

import int8_oracle as io
import requests_oracle as ro
from conftest import rand_bf16
from test_int8_gpu import ctx, plain, quantize  # noqa: F401 (fixtures)
from test_kv8_gpu import Case, Kv, blocks

pytestmark = pytest.mark.gpu

EPS = 1e-6


def product_of(v, bound, w, bias=None):
    """(y, bound) of F32 rows v, known to `bound`, in 8 bits, times (codes,
    scales) w."""
    c, s, doubtful, off = io.quantized(v, bound)
    y, out = io.product((c, s), w, bias)
    t = np.abs(w[1].astype(np.float64))
    return y, out + (doubtful @ np.abs(w[0]).T) * s[:, None] * t + \
        np.abs(c @ w[0].T) * t * off[:, None]


@pytest.mark.parametrize("rows,texts", [
    ([70, 1, 33], [130, 0, 77]), ([1, 1, 1, 1], [33, 64, 1, 200]),
    ([300], [65])])
def test_packed_block(ctx, rows, texts):  # noqa: F811
    rng = np.random.default_rng((len(rows), rows[0]))
    heads, kv_heads, dim, width, text_dim, hidden, slots = \
        4, 2, 64, 320, 200, 500, 6
    m, t, inner = sum(rows), sum(texts), heads * dim
    kv_width = 2 * kv_heads * dim
    weight = {name: rand_bf16(rng, n * k, k ** -0.5) for name, n, k in (
        ("q", inner, width), ("kv", kv_width, text_dim), ("out", width, inner),
        ("fc1", 2 * hidden, width), ("fc2", width, hidden))}
    shape = {"q": (inner, width), "kv": (kv_width, text_dim),
             "out": (width, inner), "fc1": (2 * hidden, width),
             "fc2": (width, hidden)}
    bias = {name: rand_bf16(rng, shape[name][0], 0.1)
            for name in ("q", "kv", "out")}
    w8 = {name: quantize(ctx, weight[name], *shape[name]) for name in weight}
    w64 = {name: io.rows_of(ro.wide(weight[name], *shape[name]))
           for name in weight}
    b8 = {name: ctx.bf16(b) for name, b in bias.items()}
    x, text = rand_bf16(rng, m * width), rand_bf16(rng, t * text_dim)
    norms = [rand_bf16(rng, width) for _ in range(2)]
    mod = rand_bf16(rng, len(rows) * slots * width, 0.3)
    at = np.repeat(np.arange(len(rows), dtype=np.uint32), rows)
    q_first = [int(v) for v in np.cumsum([0, *rows])[:-1]]
    t_first = [int(v) for v in np.cumsum([0, *texts])[:-1]]
    kv_first = [64 * int(v) for v in np.cumsum(
        [0] + [blocks(n) for n in texts])[:-1]]
    cache = ctx.kv_int8(max(64, 64 * sum(map(blocks, texts))), kv_heads, dim)
    plan = ctx.sdpa_packed_plan(q_first, rows, kv_first, texts, heads,
                                kv_heads, dim)
    x_d, text_d, mod_d, at_d = (ctx.bf16(x), ctx.bf16(text), ctx.bf16(mod),
                                ctx.u32(at))
    norm_d = [ctx.bf16(n) for n in norms]
    x8, t8 = ctx.int8(m, width), ctx.int8(t, text_dim)
    o8, y8 = ctx.int8(m, inner), ctx.int8(m, width)
    q, o, y, z = (ctx.new_bf16(m * n) for n in (inner, inner, width, width))
    kv = ctx.new_bf16(t * kv_width)
    scale, L, h = float(np.float32(dim ** -0.5)), ctx.L, ctx.h

    def call(name, *args):
        ctx.check(getattr(L, "h3_hip_" + name)(h, *args), name)

    for _ in range(2):  # the second time into what the first has left
        ctx.begin()
        call("adaln_int8", x8, x_d, norm_d[0], mod_d, at_d, m, width, slots, 1,
             4, EPS)
        call("linear_int8_bf16", q, x8, w8["q"], b8["q"], m, width, inner)
        call("quantize_int8", t8, text_d, t, text_dim)
        call("linear_int8_bf16", kv, t8, w8["kv"], b8["kv"], t, text_dim,
             kv_width)
        ctx.kv_int8_store(cache, kv_first, t_first, texts, kv, 0, kv,
                          kv_heads * dim, kv_width)
        call("sdpa_packed_int8_bf16", o, q, 0, inner, cache, plan, scale)
        call("quantize_int8", o8, o, m, inner)
        call("linear_int8_bf16", y, o8, w8["out"], b8["out"], m, inner, width)
        call("layer_adaln_int8", y8, y, norm_d[1], None, mod_d, at_d, m, width,
             slots, 2, 5, EPS)
        call("mlp_int8_bf16", z, y8, w8["fc1"], w8["fc2"], m, width, hidden,
             width)
        ctx.submit()

    got = {name: ctx.read_bf16(d).reshape(n, -1) for name, d, n in (
        ("q", q, m), ("kv", kv, t), ("o", o, m), ("y", y, m), ("z", z, m))}

    def wide(name):
        return ro.wide(got[name], *got[name].shape)

    mods = ro.wide(mod, len(rows), slots, width)
    eps = float(np.float32(EPS))
    want, bound = product_of(*io.norm(
        ro.wide(x, m, width), ro.wide(norms[0], width), None, mods, at, 1, 4,
        eps, False), w64["q"], bias["q"])
    ro.check(got["q"], want, io.rounded(want, bound), what="q")
    want, bound = io.product(io.rows_of(ro.wide(text, t, text_dim)),
                             w64["kv"], bias["kv"])
    ro.check(got["kv"], want, io.rounded(want, bound), what="kv")
    wide_cache = io.Cache(max(64, 64 * sum(map(blocks, texts))), kv_heads, dim)
    rows64 = wide("kv").reshape(t, 2, kv_heads, dim)
    for first, source, n in zip(kv_first, t_first, texts):
        if n:
            wide_cache.store(first, rows64[source:source + n])
    want, bound, _ = io.attention(
        wide("q").reshape(m, heads, dim), wide_cache,
        list(zip(q_first, rows, kv_first, texts)), heads, kv_heads, dim, scale)
    ro.check(got["o"].reshape(m, heads, dim), want, bound, what="o")
    want, bound = io.product(io.rows_of(wide("o")), w64["out"], bias["out"])
    ro.check(got["y"], want, io.rounded(want, bound), what="y")
    c, s, doubtful, off = io.quantized(*io.norm(
        wide("y"), ro.wide(norms[1], width), None, mods, at, 2, 5, eps, True))
    # the gated block of codes that are one off where doubtful: each may move
    # the hidden values, whose slope by gate and up is within 1.1 of each
    g, u = np.split(c @ w64["fc1"][0].T * s[:, None] * w64["fc1"][1], 2, 1)
    moved = (doubtful @ np.abs(w64["fc1"][0]).T) * s[:, None] * \
        w64["fc1"][1] + np.abs(c @ w64["fc1"][0].T) * w64["fc1"][1] * \
        off[:, None]
    mg, mu = np.split(moved, 2, 1)
    more = 1.1 * mg * np.abs(u) + np.abs(g) * mu + 1.1 * mg * mu
    v = g / (1 + np.exp(-g)) * u
    # as io.mlp, of values known to `more` beside what F32 does there
    og, ou = np.split(5 * io.HALF * np.abs(np.hstack([g, u])) + 2.0 ** -149,
                      2, 1)
    bound = more + 1.1 * og * np.abs(u) + np.abs(g) * ou + og * ou + \
        np.abs(v) * (np.abs(g) + 6) * 2.0 ** -22
    want, bound = product_of(v, bound, w64["fc2"])
    ro.check(got["z"], want, io.rounded(want, bound), what="z")


@pytest.mark.parametrize("heads,kv_heads,dim,has", [
    (8, 2, 128, [0, 63, 64, 130]), (6, 6, 64, [5, 500, 127]),
    (4, 1, 96, [1, 1000])])
def test_rows_join_the_cache(gpu, heads, kv_heads, dim, has):
    """Each step, a new row of each request is stored, then attends to all."""
    room = [64 * blocks(n + 3) for n in has]
    first = [int(v) for v in np.cumsum([0, *room])[:-1]]
    kv = Kv(gpu, sum(room), kv_heads, dim)
    kv.store(first, has)
    rng = np.random.default_rng(3)
    n, width = len(has), heads * dim
    scale = float(np.float32(dim ** -0.5))
    for step in range(3):
        length = [v + step for v in has]
        kv.store([f + v for f, v in zip(first, length)], [1] * n,
                 std=1.0 + step)
        length = [v + 1 for v in length]
        q = rand_bf16(rng, n * width)
        plan = gpu.sdpa_packed_plan(list(range(n)), [1] * n, first, length,
                                    heads, kv_heads, dim)
        y = gpu.new_bf16(n * width)
        gpu.run("h3_hip_sdpa_packed_int8_bf16", y, gpu.bf16(q), 0, width, kv.t,
                plan, scale)
        want, bound, _ = io.attention(
            ro.wide(q, n, heads, dim), kv.wide,
            list(zip(range(n), [1] * n, first, length)), heads, kv_heads, dim,
            scale)
        ro.check(gpu.read_bf16(y).reshape(n, heads, dim), want, bound)


def test_few_and_many_rows_in_one_plan(gpu):
    """Spans that both kinds of items read, and that requests share."""
    a = Case(gpu, [1, 200, 8, 129, 40], [300, 300, 65, 1000, 64], 4, 2, 128)
    a.kf = [0, 0, 320, 448, 320]
    a.kn = [300, 280, 65, 700, 64]
    a.check()


def test_two_contexts_at_once(gpu):
    """Each has scratch of its own, whichever thread calls."""
    import h3hip
    other = h3hip.Gpu()
    try:
        cases = [Case(gpu, [70, 1], [513, 3000], 8, 2, 128, seed=1),
                 Case(other, [70, 1], [600, 2000], 8, 2, 128, seed=2)]
        single = [c.run() for c in cases]
        got = [[], []]

        def work(i):
            for _ in range(8):
                got[i].append(cases[i].run())

        threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        for i in (0, 1):
            assert len(got[i]) == 8
            assert all(np.array_equal(single[i], g) for g in got[i])
    finally:
        other.close()


def test_calls_of_two_contexts_in_turn(gpu):
    import h3hip
    other = h3hip.Gpu()
    try:
        rng = np.random.default_rng(5)
        m, k, n = 300, 2675, 1001
        sides = []
        for g in (gpu, other):
            x, w = rand_bf16(rng, m * k), rand_bf16(rng, n * k)
            sides.append((g, x, w, quantize(g, x, m, k), quantize(g, w, n, k),
                          g.new_bf16(m * n)))
        for g, *_ in sides:
            g.begin()
        for _ in range(3):
            for g, _, _, x8, w8, y in sides:
                g.check(g.L.h3_hip_linear_int8_bf16(g.h, y, x8, w8, None, m, k,
                                                    n), "product")
        for g, *_ in sides:
            g.submit()
        for g, x, w, _, _, y in sides:
            want, bound = io.product(io.rows_of(ro.wide(x, m, k)),
                                     io.rows_of(ro.wide(w, n, k)))
            ro.check(g.read_bf16(y).reshape(m, n), want,
                     io.rounded(want, bound))
    finally:
        other.close()
