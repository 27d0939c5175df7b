"""What the operators of packed requests refuse, with the message, and what
they take, without a GPU (requests_oracle.on_fake)."""
import pytest

from requests_oracle import on_fake

LORA = """
k, n, rows = 64, 32, 5
x, w, b = gpu.new_bf16(rows * k), gpu.new_bf16(n * k), gpu.new_bf16(n)
y, f = gpu.new_bf16(rows * n), gpu.new_f32(10000)
ids = gpu.u32([0] * rows)
def table(down=4 * 64, up=4 * 32, rank=4, scale=1.0, count=1, k=64, n=32,
          none=False):
    d, u = gpu.new_bf16(down), gpu.new_bf16(up)
    one = (C.c_void_p * 1)(None if none else d), (C.c_void_p * 1)(u)
    h = gpu.L.h3_hip_lora_table(gpu.h, *one, (C.c_uint32 * 1)(rank),
                                (C.c_float * 1)(scale), count, k, n)
    return h
def call(**more):
    a = dict(y=y, x=x, w=w, b=b, table=table(), ids=ids, rows=rows, k=k, n=n)
    a.update(more)
    ok = gpu.L.h3_hip_linear_lora_bf16(gpu.h, *a.values())
    made = [l for l in launches() if not l[0].startswith("hk_lora_pack")]
    return ["" if ok else gpu.error(), len(made)]
"""


@pytest.mark.parametrize("make,message", [
    ("table(rank=1025, down=1025 * 64, up=1025 * 32)", "over 1024"),
    ("table(scale=float('inf'))", "not finite"),
    ("table(scale=float('nan'))", "not finite"),
    ("table(count=0)", "at least one"), ("table(k=0)", "at least one"),
    ("table(down=4 * 64 - 1)", "down tensor is too small"),
    ("table(up=4 * 32 - 1)", "up tensor is too small"),
    ("table(none=True)", "down tensor is too small"),
])
def test_adapter_tables_refused(make, message):
    made, error = on_fake(LORA + f"h = {make}; out = [bool(h), gpu.error()]")
    assert not made and message in error


def test_rank_zero_needs_no_adapter():
    assert on_fake(LORA + "out = bool(table(rank=0, none=True))")


@pytest.mark.parametrize("change,message", [
    ("table=None", "not built by h3_hip_lora_table"),
    ("table=ids", "not built by h3_hip_lora_table"),
    ("table=gpu.sdpa_packed_plan([0], [1], [0], [1], 1, 1, 64)",
     "not built by h3_hip_lora_table"),
    ("table=table(k=32, down=4 * 32)", "64 to 32 differs from the table's 32"),
    ("table=table(n=31)", "differs from the table's 64 to 31"),
    ("ids=None", "map tensor is too small"),
    ("ids=gpu.u32([0] * 4)", "map tensor is too small"),
    ("ids=f", "map tensor has the wrong dtype"),
    ("x=f", "input tensor has the wrong dtype"),
    ("rows=6", "input tensor is too small"),
    ("b=gpu.new_bf16(31)", "bias tensor is too small"),
    ("y=gpu.new_bf16(5 * 32 - 1)", "output tensor is too small"),
    ("y=x", "a tensor of its own"), ("y=w", "a tensor of its own"),
    ("y=b", "output tensor is too small"),
])
def test_linear_with_adapters_refused(change, message):
    (error, launched), = on_fake(
        LORA + f"gpu.begin(); fake.fake_clear(); out = [call({change})]")
    assert message in error and not launched


def test_linear_with_adapters_needs_a_batch():
    (error, _), = on_fake(LORA + "out = [call()]")
    assert "no active command buffer" in error


def test_no_rows_launch_nothing():
    out = on_fake(LORA + """
t = table()
gpu.begin(); fake.fake_clear()
out = [call(table=t, rows=0), call(table=t)]
""")
    assert out[0] == ["", 0] and out[1][0] == "" and out[1][1] > 0


PACKED = """
heads, kv, dim = 4, 2, 64
q, k = gpu.new_bf16(20 * 4 * 64), gpu.new_bf16(30 * 2 * 64)
v, y = gpu.new_bf16(30 * 2 * 64), gpu.new_bf16(20 * 4 * 64)
f = gpu.new_f32(10000)
def plan(qf=[0, 12], qn=[12, 8], kf=[0, 20], kn=[20, 10], n=2, heads=4, kv=2,
         dim=64):
    a = [None if r is None else (C.c_uint32 * 2)(*r) for r in (qf, qn, kf, kn)]
    return gpu.L.h3_hip_sdpa_packed_plan(gpu.h, *a, n, heads, kv, dim)
def call(**more):
    a = dict(y=y, q=q, qo=0, qs=256, k=k, ko=0, v=v, vo=0, ks=128,
             plan=plan(), scale=0.125)
    a.update(more)
    ok = gpu.L.h3_hip_sdpa_packed_bf16(gpu.h, *a.values())
    return ["" if ok else gpu.error(), len(launches())]
"""


@pytest.mark.parametrize("change,message", [
    ("n=0", "at least one request"), ("qf=None", "at least one request"),
    ("kn=None", "at least one request"), ("kv=3", "multiple of key heads"),
    ("kv=0", "multiple of key heads"), ("heads=0", "multiple of key heads"),
    ("dim=0", "head_dim 1 to 256"), ("dim=257", "head_dim 1 to 256"),
    ("qf=[0, 11]", "overlap at row 11"), ("qf=[9, 0], qn=[1, 10]", "overlap"),
    ("qf=[5, 5], qn=[1, 1]", "overlap at row 5"),
    ("qf=[0, 0xffffffff]", "pass 2^32"), ("kf=[0, 0xfffffff6]", "pass 2^32"),
    ("qn=[12, 0xf0000000]", "too many query rows"),
])
def test_attention_plans_refused(change, message):
    made, error = on_fake(
        PACKED + f"h = plan({change}); out = [bool(h), gpu.error()]")
    assert not made and message in error


@pytest.mark.parametrize("change,message", [
    ("plan=None", "not built by"), ("plan=f", "not built by"),
    ("plan=q", "not built by"), ("qs=255", "under the rows'"),
    ("ks=127", "under the rows'"), ("scale=-1.0", "not negative"),
    ("scale=float('nan')", "must be finite"),
    ("scale=float('inf')", "must be finite"), ("q=f", "query tensor"),
    ("k=f", "key tensor"), ("v=f", "value tensor"), ("y=f", "output tensor"),
    ("q=None", "query tensor"), ("qo=1", "query tensor is too small"),
    ("ko=1", "key tensor is too small"), ("vo=1", "value tensor is too small"),
    ("qs=257", "query tensor is too small"),
    ("ks=129", "key tensor is too small"),
    ("qo=2**64 - 8", "query tensor is too small"),
    ("vo=2**64 - 8", "value tensor is too small"),
    ("y=q", "a tensor of its own"),
    ("y=gpu.new_bf16(20 * 256 - 1)", "output tensor is too small"),
])
def test_packed_attention_refused(change, message):
    (error, launched), = on_fake(
        PACKED + f"gpu.begin(); out = [call({change})]")
    assert message in error and not launched


def test_packed_attention_needs_a_batch():
    (error, _), = on_fake(PACKED + "out = [call()]")
    assert "no active command buffer" in error


def test_packed_attention_takes():
    """Shared keys, empty requests on either side, rows of no request, the
    last rows of the tensors."""
    out = on_fake(PACKED + """
gpu.begin()
for p in (dict(), dict(kf=[0, 0], kn=[30, 30]), dict(kn=[0, 0]),
          dict(qn=[0, 8]), dict(qf=[0, 19], qn=[1, 1], kf=[29, 0], kn=[1, 1]),
          dict(qf=[12, 0], qn=[8, 12])):
    fake.fake_clear()
    t = plan(**p)
    out = (out or []) + [call(plan=t)]
fake.fake_clear()
out.append(call(plan=plan(qn=[0, 0])))
""")
    assert all(not error and launched for error, launched in out[:-1]), out
    assert out[-1] == ["", 0]


@pytest.mark.parametrize("m,k,n", [(8_400_000, 64, 4), (129, 64, 1 << 22),
                                   (70_000, 64, 4096), (128, 64, 1 << 22)])
def test_adapter_launches_stay_within_a_grid(m, k, n):
    """Threads of a launch below 2^32 and its second dimension below 2^16, for
    the most rows and columns too."""
    made = on_fake("""
x, w = gpu.new_bf16(m * k), gpu.new_bf16(n * k)
y, ids = gpu.new_bf16(m * n), gpu.L.h3_gpu_tensor_from_u32(gpu.h, None, m)
tables = []
for rank in (4, 64):
    d, u = gpu.new_bf16(rank * k), gpu.new_bf16(rank * n)
    tables.append(gpu.lora_table([d] * 3, [u] * 3, [rank] * 3, [1.0] * 3, k, n))
gpu.begin(); fake.fake_clear()
for t in tables:
    assert gpu.L.h3_hip_linear_lora_bf16(gpu.h, y, x, w, None, t, ids, m, k, n)
out = launches()
""", m=m, k=k, n=n)
    assert made
    for kernel, x, y, z, threads, _ in made:
        assert x * threads < 1 << 32 and y < 1 << 16 and z < 1 << 16, kernel
