"""A packed forward's attention part as a server of several requests runs it:
QKV projection with each request's adapter, self-attention of each request's
rows, cross-attention to each request's text (its keys and values projected
with the adapters too), output projection with the adapters, all in one batch.
Each stage is held against the same in 64 bits of what the device has as its
input."""
import numpy as np
import pytest

import requests_oracle as ro
from conftest import rand_bf16

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,texts,use", [
    ([300, 77, 1], [64, 20, 5], [0, ro.NONE, 1]),
    ([1, 1, 1, 1], [33, 0, 64, 1], [1, 0, 1, 0]),
    ([129], [100], [0])])
def test_packed_forward(gpu, rows, texts, use):
    rng = np.random.default_rng(len(rows))
    heads, kv_heads, dim, width, text_dim = 4, 2, 128, 512, 320
    m, t = sum(rows), sum(texts)
    inner, fused = heads * dim, (heads + 2 * kv_heads) * dim
    ids = np.repeat(np.asarray(use, np.uint32), rows)
    text_ids = np.repeat(np.asarray(use, np.uint32), texts)
    first = [int(v) for v in np.cumsum([0, *rows])[:-1]]
    text_first = [int(v) for v in np.cumsum([0, *texts])[:-1]]
    ranks, scales = [16, 9], [1.0, 0.7]

    def projection(k, n):
        w, b = rand_bf16(rng, n * k, k ** -0.5), rand_bf16(rng, n, 0.1)
        down = [rand_bf16(rng, r * k, k ** -0.5) for r in ranks]
        up = [rand_bf16(rng, n * r, 0.2) for r in ranks]
        return dict(w=w, b=b, down=down, up=up, ranks=ranks, scales=scales,
                    k=k, n=n)

    sizes = {"qkv": (width, fused), "cq": (inner, inner),
             "ckv": (text_dim, 2 * kv_heads * dim), "out": (inner, width)}
    p = {name: projection(*size) for name, size in sizes.items()}
    dev = {name: (gpu.bf16(a["w"]), gpu.bf16(a["b"]), gpu.lora_table(
        [gpu.bf16(d) for d in a["down"]], [gpu.bf16(u) for u in a["up"]],
        ranks, scales, a["k"], a["n"])) for name, a in p.items()}
    x, text = rand_bf16(rng, m * width), rand_bf16(rng, t * text_dim)
    x_d, text_d = gpu.bf16(x), gpu.bf16(text)
    ids_d, text_ids_d = gpu.u32(ids), gpu.u32(text_ids)
    self_plan = gpu.sdpa_packed_plan(first, rows, first, rows, heads, kv_heads,
                                     dim)
    cross_plan = gpu.sdpa_packed_plan(first, rows, text_first, texts, heads,
                                      kv_heads, dim)
    qkv, cq, out = (gpu.new_bf16(m * p[n]["n"]) for n in ("qkv", "cq", "out"))
    ckv = gpu.new_bf16(t * p["ckv"]["n"])
    o1, o2 = gpu.new_bf16(m * inner), gpu.new_bf16(m * inner)
    scale = float(np.float32(dim ** -0.5))
    L, h = gpu.L, gpu.h

    def linear(name, y, source, n, at):
        w, b, table = dev[name]
        gpu.check(L.h3_hip_linear_lora_bf16(
            h, y, source, w, b, table, at, n, p[name]["k"], p[name]["n"]))

    gpu.begin()
    linear("qkv", qkv, x_d, m, ids_d)
    gpu.check(L.h3_hip_sdpa_packed_bf16(
        h, o1, qkv, 0, fused, qkv, inner, qkv, inner + kv_heads * dim, fused,
        self_plan, scale))
    linear("cq", cq, o1, m, ids_d)
    linear("ckv", ckv, text_d, t, text_ids_d)
    gpu.check(L.h3_hip_sdpa_packed_bf16(
        h, o2, cq, 0, inner, ckv, 0, ckv, kv_heads * dim, 2 * kv_heads * dim,
        cross_plan, scale))
    linear("out", out, o2, m, ids_d)
    gpu.submit()

    got = {n: gpu.read_bf16(y) for n, y in dict(
        qkv=qkv, o1=o1, cq=cq, ckv=ckv, o2=o2, out=out).items()}
    for name, source, at in (("qkv", x, ids), ("cq", got["o1"], ids),
                             ("ckv", text, text_ids),
                             ("out", got["o2"], ids)):
        want, bound = ro.lora(x=source, ids=at, **p[name])
        ro.check(got[name], want, bound, name)
    a = ro.wide(got["qkv"], m, heads + 2 * kv_heads, dim)
    want, bound, _ = ro.packed(
        a[:, :heads], a[:, heads:heads + kv_heads], a[:, heads + kv_heads:],
        list(zip(first, rows, first, rows)), heads, kv_heads, dim, scale)
    ro.check(got["o1"], want, bound, "self")
    b = ro.wide(got["ckv"], t, 2, kv_heads, dim)
    want, bound, _ = ro.packed(
        ro.wide(got["cq"], m, heads, dim), b[:, 0], b[:, 1],
        list(zip(first, rows, text_first, texts)), heads, kv_heads, dim,
        scale)
    ro.check(got["o2"], want, bound, "cross")
