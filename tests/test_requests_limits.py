"""The operators of packed requests at the ends of their ranges, without a GPU
(requests_oracle.on_fake)."""
import pytest

from requests_oracle import on_fake

PLAN = """
def plan(qn, kn, heads=1, kv=1, dim=8, kf=None):
    n, u32 = len(qn), C.c_uint32
    qf = [sum(qn[:i]) for i in range(n)]
    return gpu.L.h3_hip_sdpa_packed_plan(
        gpu.h, (u32 * n)(*qf), (u32 * n)(*qn), (u32 * n)(*(kf or [0] * n)),
        (u32 * n)(*kn), n, heads, kv, dim)
"""


@pytest.mark.parametrize("kn", [0xFFFFFFFF, 0xFFFFFFFF - 31, 0xFFFFFFFF - 63,
                                0xFFFFFF01])
@pytest.mark.parametrize("qn", [[1], [0], [3, 200]])
def test_more_keys_than_the_kernels_count(qn, kn):
    """Their 32-bit key numbers would wrap in the last tile: a loop that never
    ends, or rows of zeros."""
    made, error = on_fake(
        PLAN + "h = plan(qn, kn); out = [bool(h), gpu.error()]", qn=qn,
        kn=[5] * (len(qn) - 1) + [kn])
    assert not made and "key rows, over 4294967040" in error


def test_the_most_keys_that_they_count():
    assert on_fake(PLAN + "out = bool(plan([1], [0xFFFFFF00]))")


@pytest.mark.parametrize("rows,heads", [(6000, 3000), (8000, 4)])
def test_launches_of_many_items_stay_within_a_grid(rows, heads):
    """A single row's key heads are an item each; a launch has fewer than 2^32
    threads, and the launches together every item once."""
    made = on_fake(PLAN + """
h = plan([1] * rows, [64] * rows, heads, heads)
y, q = gpu.new_bf16(rows * heads * 8), gpu.new_bf16(rows * heads * 8)
k = gpu.new_bf16(64 * heads * 8)
gpu.begin(); fake.fake_clear()
assert gpu.L.h3_hip_sdpa_packed_bf16(gpu.h, y, q, 0, heads * 8, k, 0, k, 0,
                                     heads * 8, h, 1.0), gpu.error()
out = launches()
""", rows=rows, heads=heads)
    assert all(kernel == "hk_packed_flash<64>" for kernel, *_ in made)
    assert all(x * threads < 1 << 32 for _, x, _, _, threads, _ in made)
    assert sum(x for _, x, *_ in made) == rows * heads


@pytest.mark.parametrize("qn,kn,heads,kv,dim", [
    ([1] * 8, [6144] * 8, 64, 8, 128), ([128, 40], [9720, 9000], 32, 32, 64),
    ([300], [3000], 12, 4, 96)])
def test_packed_attention_without_scratch(qn, kn, heads, kv, dim):
    """It is taken, with no joins."""
    made = on_fake(PLAN + """
h = plan(qn, kn, heads, kv, dim)
y, q = (gpu.new_bf16(sum(qn) * heads * dim) for _ in "yq")
k = gpu.new_bf16(max(kn) * kv * dim)
gpu.begin()
out = []
for size in (0, -1):
    fake.fake_largest_block(C.c_size_t(size)); fake.fake_clear()
    assert gpu.L.h3_hip_sdpa_packed_bf16(
        gpu.h, y, q, 0, heads * dim, k, 0, k, 0, kv * dim, h, 1.0), gpu.error()
    out.append([l[0] for l in launches()])
""", qn=qn, kn=kn, heads=heads, kv=kv, dim=dim)
    flash = f"hk_packed_flash<{dim}>"
    joined = f"hk_packed_joined<{64 if dim <= 64 else 128}>"
    assert made == [[flash], [flash, joined]]


@pytest.mark.parametrize("gelu", [False, True])
@pytest.mark.parametrize("rows,k,n", [(39, 2688, 96768), (128, 64, 36000),
                                      (5, 128, 140000), (300, 320, 20480),
                                      (1000, 320, 5120)])
def test_adapters_without_scratch(rows, k, n, gelu):
    """They go over tiles, which need no sums of the whole output."""
    made = on_fake("""
d, u = gpu.new_bf16(16 * k), gpu.new_bf16(16 * n)
t = gpu.lora_table([d], [u], [16], [1.0], k, n)
x, w, y = gpu.new_bf16(rows * k), gpu.new_bf16(n * k), gpu.new_bf16(rows * n)
ids = gpu.u32([0] * rows)
call = (gpu.L.h3_hip_linear_lora_gelu_bf16 if gelu else
        gpu.L.h3_hip_linear_lora_bf16)
gpu.begin()
out = []
for size in (8 << 20, -1):
    fake.fake_largest_block(C.c_size_t(size)); fake.fake_clear()
    assert call(gpu.h, y, x, w, None, t, ids, rows, k, n), gpu.error()
    out.append([l[0].split("<")[0] for l in launches()])
""", rows=rows, k=k, n=n, gelu=gelu)
    assert made == [["hk_lora_low", "hk_lora_halves", "hk_gemm_lora"],
                    ["hk_lora_skinny", "hk_lora_join"]]


@pytest.mark.parametrize("rank,k,n", [(1024, 64, 4_300_000),
                                      (1024, 4_300_000, 64), (4, 64, 32)])
def test_launches_of_large_adapters_stay_within_a_grid(rank, k, n):
    """B padded and A may have over 2^32 elements."""
    made = on_fake("""
d, u = gpu.new_bf16(rank * k), gpu.new_bf16(rank * n)
fake.fake_clear()
gpu.lora_table([d], [u], [rank], [1.0], k, n)
out = launches()
""", rank=rank, k=k, n=n)
    assert [kernel for kernel, *_ in made] == [
        "hk_lora_pack", "hk_lora_pack", "hk_lora_pack_fragments"]
    assert all(x * threads < 1 << 32 for _, x, _, _, threads, _ in made)
