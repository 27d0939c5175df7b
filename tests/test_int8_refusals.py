"""What the 8-bit operators refuse, with the message, without a GPU
(requests_oracle.on_fake)."""
import pytest

from requests_oracle import on_fake

PRODUCT = """
m, k, n, h = 5, 200, 32, 48
x, w = gpu.int8(m, k), gpu.int8(n, k)
y, b, f = gpu.new_bf16(m * n), gpu.new_bf16(n), gpu.new_f32(10000)
i8 = gpu.L.h3_gpu_tensor_new_i8(gpu.h, 100000)
cache = gpu.kv_int8(64, 1, 64)
def said(ok):
    return ["" if ok else gpu.error(), len(launches())]
def linear(**more):
    a = dict(y=y, x=x, w=w, b=b, m=m, k=k, n=n)
    a.update(more)
    return said(gpu.L.h3_hip_linear_int8_bf16(gpu.h, *a.values()))
def mlp(**more):
    a = dict(y=y, x=x, w1=gpu.int8(2 * h, k), w2=gpu.int8(n, h), m=m, k=k, h=h,
             n=n)
    a.update(more)
    return said(gpu.L.h3_hip_mlp_int8_bf16(gpu.h, *a.values()))
def rows(**more):
    a = dict(out=x, x=gpu.new_bf16(m * k), m=m, k=k)
    a.update(more)
    return said(gpu.L.h3_hip_quantize_int8(gpu.h, *a.values()))
def values(**more):
    a = dict(y=gpu.new_bf16(m * k), x=x, m=m, k=k)
    a.update(more)
    return said(gpu.L.h3_hip_dequantize_int8(gpu.h, *a.values()))
def rms(**more):
    a = dict(out=x, x=gpu.new_bf16(m * k), w=gpu.new_bf16(k),
             mod=gpu.new_bf16(6 * k), at=gpu.u32([0] * m), m=m, k=k, slots=6,
             shift=3, scale=4, eps=1e-5)
    a.update(more)
    return said(gpu.L.h3_hip_adaln_int8(gpu.h, *a.values()))
def layer(**more):
    a = dict(out=x, x=gpu.new_bf16(m * k), w=gpu.new_bf16(k),
             b=gpu.new_bf16(k), mod=gpu.new_bf16(6 * k), at=gpu.u32([0] * m),
             m=m, k=k, slots=6, shift=3, scale=4, eps=1e-5)
    a.update(more)
    return said(gpu.L.h3_hip_layer_adaln_int8(gpu.h, *a.values()))
"""


@pytest.mark.parametrize("rows,columns", [(0, 5), (5, 0), (5, 131073)])
def test_matrices_refused(rows, columns):
    made, error = on_fake(
        f"out = [bool(gpu.L.h3_hip_int8_new(gpu.h, {rows}, {columns})), "
        "gpu.error()]")
    assert not made and "1 to 131072 columns" in error


NOT_MADE = "not made by h3_hip_int8_new"


@pytest.mark.parametrize("call,message", [
    ("linear(x=None)", NOT_MADE), ("linear(x=i8)", NOT_MADE),
    ("linear(x=y)", NOT_MADE), ("linear(w=cache)", NOT_MADE),
    ("linear(k=199)", "has 200 columns, not 199"),
    ("linear(w=gpu.int8(n, k + 1))", "has 201 columns, not 200"),
    ("linear(m=6, y=gpu.new_bf16(6 * n))", "has 5 rows, under 6"),
    ("linear(n=33, y=gpu.new_bf16(m * 33), b=gpu.new_bf16(33))",
     "has 32 rows, under 33"),
    ("linear(y=gpu.new_bf16(m * n - 1))", "output tensor is too small"),
    ("linear(y=f)", "output tensor has the wrong dtype"),
    ("linear(b=gpu.new_bf16(n - 1))", "bias tensor is too small"),
    ("linear(b=f)", "bias tensor has the wrong dtype"),
    ("linear(b=y)", "a tensor of its own"),
    ("mlp(x=i8)", NOT_MADE), ("mlp(w1=gpu.int8(2 * h - 1, k))", "under 96"),
    ("mlp(w2=gpu.int8(n, h + 1))", "has 49 columns, not 48"),
    ("mlp(w2=w)", "has 200 columns, not 48"),
    ("mlp(h=0)", "0 hidden columns"), ("mlp(h=131073)", "131073 hidden"),
    ("mlp(h=2**31 + h)", "hidden columns"),
    ("mlp(y=f)", "output tensor has the wrong dtype"),
    ("mlp(m=6, y=gpu.new_bf16(6 * n))", "has 5 rows"),
    ("rows(out=i8)", NOT_MADE), ("rows(k=100)", "has 200 columns, not 100"),
    ("rows(m=6, x=gpu.new_bf16(6 * k))", "has 5 rows, under 6"),
    ("rows(x=gpu.new_bf16(m * k - 1))", "input tensor is too small"),
    ("rows(x=f)", "input tensor has the wrong dtype"),
    ("values(x=i8)", NOT_MADE), ("values(y=f)", "wrong dtype"),
    ("values(y=gpu.new_bf16(m * k - 1))", "output tensor is too small"),
    ("rms(w=None)", "weight tensor is too small"),
    ("rms(mod=None)", "modulation tensor is too small"),
    ("rms(at=None)", "row map tensor is too small"),
    ("rms(at=gpu.u32([0] * 4))", "row map tensor is too small"),
    ("rms(at=f)", "row map tensor has the wrong dtype"),
    ("rms(mod=gpu.new_bf16(6 * k - 1))", "modulation tensor is too small"),
    ("rms(shift=6)", "slot out of range"),
    ("rms(scale=6)", "slot out of range"),
    ("rms(x=f)", "wrong dtype"), ("rms(out=i8)", NOT_MADE),
    ("layer(b=gpu.new_bf16(k - 1))", "bias tensor is too small"),
    ("layer(at=None)", "row map tensor is too small"),
    ("layer(scale=7)", "slot out of range"),
])
def test_refused(call, message):
    (error, launched), = on_fake(
        PRODUCT + f"gpu.begin(); fake.fake_clear(); out = [{call}]")
    assert message in error and not launched


@pytest.mark.parametrize("call", ["linear()", "mlp()", "rows()", "values()",
                                  "rms()", "layer()"])
def test_needs_a_batch(call):
    (error, _), = on_fake(PRODUCT + f"out = [{call}]")
    assert "no active command buffer" in error


@pytest.mark.parametrize("call", [
    "linear()", "linear(b=None)", "mlp()", "rows()", "rows(m=2)", "values()",
    "rms()", "layer()", "layer(w=None, b=None, mod=None, at=None, slots=0)",
    "linear(m=2)", "linear(n=7)"])
def test_taken(call):
    (error, launched), = on_fake(
        PRODUCT + f"gpu.begin(); fake.fake_clear(); out = [{call}]")
    assert not error and launched


@pytest.mark.parametrize("call", [
    "linear(m=0)", "linear(n=0)", "mlp(m=0)", "mlp(n=0)", "rows(m=0)",
    "values(m=0)", "rms(m=0)", "layer(m=0)"])
def test_nothing_to_do(call):
    (error, launched), = on_fake(
        PRODUCT + f"gpu.begin(); fake.fake_clear(); out = [{call}]")
    assert not error and not launched


CACHE = """
heads, dim = 2, 64
cache = gpu.kv_int8(200, heads, dim)
k, v = gpu.new_bf16(300 * 128), gpu.new_bf16(300 * 128)
q, y, f = gpu.new_bf16(20 * 256), gpu.new_bf16(20 * 256), gpu.new_f32(100000)
i8 = gpu.int8(64, 128)
def said(ok):
    return ["" if ok else gpu.error(), len(launches())]
def store(first=[0, 64], source=[0, 50], rows=[50, 100], n=2, **more):
    a = dict(k=k, ko=0, v=v, vo=0, stride=128)
    cache_ = more.pop("cache", cache)
    a.update(more)
    lists = [None if r is None else (C.c_uint32 * len(r))(*r)
             for r in (first, source, rows)]
    return said(gpu.L.h3_hip_kv_int8_store(gpu.h, cache_, *lists, n,
                                           *a.values()))
def read(**more):
    a = dict(k=k, v=v, cache=cache, first=0, rows=256)
    a.update(more)
    return said(gpu.L.h3_hip_kv_int8_read(gpu.h, *a.values()))
def plan(qf=[0, 12], qn=[12, 8], kf=[0, 64], kn=[20, 100], heads=4, kv=2,
         dim=64):
    return gpu.sdpa_packed_plan(qf, qn, kf, kn, heads, kv, dim)
def attend(**more):
    a = dict(y=y, q=q, qo=0, qs=256, cache=cache, plan=plan(), scale=0.125)
    a.update(more)
    return said(gpu.L.h3_hip_sdpa_packed_int8_bf16(gpu.h, *a.values()))
"""


@pytest.mark.parametrize("rows,heads,dim", [
    (0, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1, 257), (1, 65536, 1),
    (2**32 - 64, 1, 1)])
def test_caches_refused(rows, heads, dim):
    made, error = on_fake(
        f"out = [bool(gpu.L.h3_hip_kv_int8_new(gpu.h, {rows}, {heads}, {dim}))"
        ", gpu.error()]")
    assert not made and "heads of 1 to 256" in error


KV = "not made by h3_hip_kv_int8_new"


@pytest.mark.parametrize("call,message", [
    ("store(cache=None)", KV), ("store(cache=i8)", KV), ("store(cache=k)", KV),
    ("store(first=None)", "no ranges"), ("store(rows=None)", "no ranges"),
    ("store(stride=127)", "under the rows' 128"),
    ("store(rows=[50, 193])", "range 1 ends behind the cache's 4 blocks"),
    ("store(first=[0, 2**32 - 1])", "ends behind"),
    ("store(first=[0, 40])", "two ranges write rows of block 0"),
    ("store(first=[100, 0])", "two ranges write rows of block 1"),
    ("store(first=[0, 0], rows=[1, 1])", "rows of block 0"),
    ("store(source=[0, 201])", "key tensor is too small"),
    ("store(source=[0, 2**32 - 1])", "key tensor is too small"),
    ("store(ko=150 * 128 + 1, k=gpu.new_bf16(300 * 128))", "key tensor"),
    ("store(vo=150 * 128 + 1)", "value tensor is too small"),
    ("store(vo=2**64 - 8)", "value tensor is too small"),
    ("store(stride=300)", "key tensor is too small"),
    ("store(k=f)", "key tensor has the wrong dtype"),
    ("store(v=f)", "value tensor has the wrong dtype"),
    ("read(cache=i8)", KV), ("read(rows=257)", "end behind the cache's 4"),
    ("read(first=2**32 - 1)", "end behind"), ("read(v=k)", "a tensor each"),
    ("read(k=gpu.new_bf16(256 * 128 - 1))", "key tensor is too small"),
    ("read(v=f)", "value tensor has the wrong dtype"),
    ("attend(cache=i8)", KV), ("attend(cache=None)", KV),
    ("attend(plan=None)", "not built by"), ("attend(plan=q)", "not built by"),
    ("attend(plan=plan(kv=4))", "4 key heads of 64 in the plan, 2 of 64"),
    ("attend(plan=plan(dim=32))", "2 key heads of 32 in the plan"),
    ("attend(plan=plan(kf=[0, 65]))", "begin at a multiple of 64"),
    ("attend(plan=plan(kf=[0, 192]))", "the plan's 292 key rows end behind"),
    ("attend(plan=plan(qn=[20000, 20000], qf=[0, 20000], kf=[0, 64], "
     "kn=[2**31, 2**31 + 640]))", "over 2^32 rows of the cache to unpack"),
    ("attend(plan=plan(qn=[20000, 20000], qf=[0, 20000], kf=[0, 64], "
     "kn=[2**31, 2**31 - 640]))", "2147483648 key rows end behind"),
    ("attend(qs=255)", "under the rows'"), ("attend(scale=-1.0)", "finite"),
    ("attend(scale=float('nan'))", "finite"),
    ("attend(scale=float('inf'))", "finite"),
    ("attend(q=f)", "query tensor has the wrong dtype"),
    ("attend(qo=1)", "query tensor is too small"),
    ("attend(qs=257)", "query tensor is too small"),
    ("attend(y=f)", "output tensor has the wrong dtype"),
    ("attend(y=q)", "a tensor of its own"),
    ("attend(y=gpu.new_bf16(20 * 256 - 1))", "output tensor is too small"),
])
def test_cache_refused(call, message):
    (error, launched), = on_fake(
        CACHE + f"gpu.begin(); fake.fake_clear(); out = [{call}]")
    assert message in error and not launched


@pytest.mark.parametrize("call", ["store()", "read()", "attend()"])
def test_cache_needs_a_batch(call):
    (error, _), = on_fake(CACHE + f"out = [{call}]")
    assert "no active command buffer" in error


@pytest.mark.parametrize("call", [
    "store()", "store(first=[0, 64], rows=[64, 192])", "read()",
    "read(first=255, rows=1)", "attend()", "attend(plan=plan(kf=[0, 0]))",
    "attend(plan=plan(kf=[0, 65], kn=[20, 0]))", "store(vo=150 * 128)"])
def test_cache_taken(call):
    (error, launched), = on_fake(
        CACHE + f"gpu.begin(); fake.fake_clear(); out = [{call}]")
    assert not error and launched


@pytest.mark.parametrize("call", [
    "store(n=0)", "store(n=0, first=None, source=None, rows=None)",
    "store(rows=[0, 0])", "read(rows=0)",
    "attend(plan=plan(qn=[0, 0]))"])
def test_cache_nothing_to_do(call):
    (error, launched), = on_fake(
        CACHE + f"gpu.begin(); fake.fake_clear(); out = [{call}]")
    assert not error and not launched


def test_launches_stay_within_a_grid():
    """Threads below 2^32 and second dimensions below 2^16, whatever the
    rows."""
    made = on_fake("""
made = 9_000_000
x, w = gpu.int8(made, 8), gpu.int8(70000, 8)
src, y = gpu.new_bf16(made * 8), gpu.new_bf16(made * 8)
out8 = gpu.new_bf16(made * 8)
cache = gpu.kv_int8(20_000_000, 300, 1)
kv = gpu.L.h3_gpu_tensor_new_bf16(gpu.h, 20_000_000 * 300)
kv2 = gpu.L.h3_gpu_tensor_new_bf16(gpu.h, 20_000_000 * 300)
gpu.begin(); fake.fake_clear()
L = gpu.L
assert L.h3_hip_quantize_int8(gpu.h, x, src, made, 8)
assert L.h3_hip_dequantize_int8(gpu.h, y, x, made, 8)
assert L.h3_hip_linear_int8_bf16(gpu.h, y, x, w, None, made, 8, 4)
gpu.kv_int8_store(cache, [3], [0], [19_999_000], kv, 0, kv2, 0, 300)
assert L.h3_hip_kv_int8_read(gpu.h, kv, kv2, cache, 5, 19_999_000)
out = launches()
""")
    assert len(made) > 8
    for kernel, x, y, z, threads, _ in made:
        assert x * threads < 1 << 32 and y < 1 << 16 and z < 1 << 16, kernel
        assert x * y * threads < 1 << 32, kernel
