"""Which kernels a projection with adapters runs, found without a GPU
(requests_oracle.on_fake)."""
import pytest

from requests_oracle import on_fake
from test_lora_tiles_gpu import CUT, MANY, SEVERAL, SHAPES, SMALL

RUN = """
out = []
for rows, k, n, ranks, gelu in cases:
    down = [gpu.new_bf16(r * k) for r in ranks]
    up = [gpu.new_bf16(r * n) for r in ranks]
    t = gpu.lora_table(down, up, ranks, [1.0] * len(ranks), k, n)
    x, w = gpu.new_bf16(rows * k), gpu.new_bf16(n * k)
    y, ids = gpu.new_bf16(rows * n), gpu.u32([0] * rows)
    gpu.begin(); fake.fake_clear()
    call = (gpu.L.h3_hip_linear_lora_gelu_bf16 if gelu else
            gpu.L.h3_hip_linear_lora_bf16)
    assert call(gpu.h, y, x, w, None, t, ids, rows, k, n), gpu.error()
    gpu.submit()
    out.append([l[0] for l in launches()])
    for h in down + up + [t, x, w, y, ids]:
        gpu.free(h)
"""


def kernels(cases):
    return on_fake(RUN, cases=[[*c[:3], list(c[3]), c[4]] for c in cases])


def over_tiles(low, gemm, gelu):
    """Full names of SHAPES' short ones."""
    epilogue, blocks = gemm[len("gemm<"):-1].split(", ")
    act = "5" if gelu else "0"
    cut = epilogue == "3"
    return ["hk_lora_" + low, "hk_lora_halves",
            f"hk_gemm_lora<{'3' if cut else act}, false, {blocks}>"] + (
                [f"hk_splitk_reduce<{act}>"] if cut else [])


@pytest.mark.parametrize("gelu", [False, True])
def test_kernels_over_tiles(gelu):
    made = kernels([(*s, gelu) for s in SHAPES])
    for shape, names, found in zip(SHAPES, SHAPES.values(), made):
        assert found == over_tiles(*names, gelu), shape


def test_every_first_product_and_tile_height_is_among_them():
    assert {low for low, _ in SHAPES.values()} == {
        f"low<{rb}, {j}>" for rb in (1, 2, 4) for j in (2, 4)}
    assert {gemm for _, gemm in SHAPES.values()} == {
        *(f"gemm<0, {b}>" for b in (4, 5, 6, 7, 8)),
        *(f"gemm<3, {b}>" for b in (5, 6, 8))}


def test_shapes_of_other_tables():
    """The other tests' of test_lora_tiles_gpu.py."""
    cut = (284, 5120, 6428)
    cases = [*SEVERAL.items(), *((s, (2,) * 281) for s in MANY),
             *((SMALL, (r, 8)) for r in (1, 64, 320)),
             *((CUT, (r, 8)) for r in (4, 33, 64, 1024)),
             *((s, (16, 33, 8)) for s in (SMALL, (386, 512, 21528), cut)),
             *((s, r) for s in (SMALL, cut) for r in ((16,), (16, 8, 33, 64)))]
    for (shape, ranks), found in zip(cases, kernels(
            [(*s, r, False) for s, r in cases])):
        assert found[1] == "hk_lora_halves", (shape, ranks[:4], found)
        assert found[2].startswith("hk_gemm_lora<")
        assert found[2].startswith("hk_gemm_lora<3") == (
            shape in (cut, CUT, (562, 2560, 9664), (2725, 2560, 1432)))


# us over groups of rows and over tiles, adapters in the order of the rows
@pytest.mark.parametrize("rows,k,n,ranks,groups", [
    (400, 5120, 13824, (16,), False),         # 107, 95
    (400, 5120, 13824, (64, 16), False),      # 114, 101
    (400, 5120, 13824, (128,) * 16, True),    # 134, 172
    (400, 5120, 13824, (512,) * 16, True),    # 251, 366
    (400, 5120, 13824, (16,) * 64, True),     # 112, 196
    (400, 5120, 13824, (128,) * 64, True),    # 182, 356
    (1000, 5120, 5120, (16,), False),         # 88, 72
    (1000, 5120, 5120, (128,) * 64, True),    # 131, 200
    (1000, 5120, 5120, (16,) * 64, True),     # 96, 118
    (1000, 5120, 13824, (128,) * 64, False),  # 298, 258
    (1000, 5120, 13824, (16,) * 64, False),   # 217, 168
    (2000, 2688, 10752, (128,) * 64, False),  # 267, 207
    (597, 5120, 5120, (128,) * 64, True)])    # 104, 254
def test_many_adapters_go_the_faster_way(rows, k, n, ranks, groups):
    made, = kernels([(rows, k, n, ranks, False)])
    assert (made[-1] == "hk_lora_join") == groups


@pytest.mark.parametrize("rows,k,n,kernel", [
    (1, 5120, 5120, "<1, 1, false>"), (16, 256, 320, "<1, 1, false>"),
    (17, 256, 320, "<1, 2, false>"), (39, 2688, 96768, "<2, 2, false>"),
    (96, 256, 320, "<3, 2, false>"), (128, 512, 36000, "<4, 2, false>"),
    (130, 5120, 13700, "<5, 2, false>"), (161, 5120, 13824, "<6, 2, false>"),
    (224, 5120, 13600, "<7, 2, false>"), (161, 256, 320, "<3, 2, true>"),
    (300, 192, 4100, "<4, 2, true>")])
def test_kernels_over_groups_of_rows(rows, k, n, kernel):
    made, = kernels([(rows, k, n, (16,), False)])
    assert made == ["hk_lora_skinny" + kernel, "hk_lora_join"]
