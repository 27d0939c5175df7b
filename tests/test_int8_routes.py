"""Which kernels the 8-bit operators run at the shapes of their tests, found
without a GPU (requests_oracle.on_fake), so that a change of the choice between
them leaves none without a test."""
import os
import re

import pytest

from conftest import ROOT
from requests_oracle import on_fake
from test_int8_kernels_gpu import GATED, OUT, PRODUCTS
from test_int8_no_room_gpu import BLOCKS, ROOM, WHOLE
from test_kv8_many_gpu import FEW, MANY, ROWS

RUN = """
out = []
for case in cases:
    *shape, gelu, room = case
    calls, made = gpu.L, []
    def new(f, *a):
        made.append(f(*a))
        return made[-1]
    m, k, h = shape[:3]
    x = new(gpu.int8, m, k)
    if len(shape) == 4:
        args = [new(gpu.new_bf16, m * shape[3]), x, new(gpu.int8, 2 * h, k),
                new(gpu.int8, shape[3], h), *shape]
        call = calls.h3_hip_mlp_int8_bf16
    else:
        args = [new(gpu.new_bf16, m * h), x, new(gpu.int8, h, k), None, *shape]
        call = (calls.h3_hip_linear_gelu_int8_bf16 if gelu else
                calls.h3_hip_linear_int8_bf16)
    gpu.begin(); fake.fake_clear()
    fake.fake_largest_block(C.c_size_t(2 ** 64 - 1 if room is None else room))
    assert call(gpu.h, *args), gpu.error()
    fake.fake_largest_block(C.c_size_t(2 ** 64 - 1))
    gpu.submit()
    out.append([l[0].removeprefix("hk_int8_") for l in launches()])
    for t in made:
        gpu.free(t)
"""


def kernels(cases):
    """Of [rows, input, output columns (, or hidden and output), GELU, the
    largest block that may be allocated]."""
    return on_fake(RUN, cases=cases)


def with_gelu(names):
    return [n.replace("gemm<0", "gemm<5") for n in names]


def test_products():
    made = kernels([[*s, False, None] for s in PRODUCTS])
    for (shape, names), found in zip(PRODUCTS.items(), made):
        assert found == names, shape
    made = kernels([[*s, True, None] for s in PRODUCTS])
    for (shape, names), found in zip(PRODUCTS.items(), made):
        assert found == with_gelu(names), shape


def test_gated_blocks():
    made = kernels([[*s, OUT, False, None] for s in GATED])
    for (shape, names), found in zip(GATED.items(), made):
        assert found[:len(names)] == names, shape
        assert found[len(names)].startswith("rows_vec<3,"), shape


BARE = """
fake.fake_largest_block(C.c_size_t(0))
gpu = h3hip.Gpu()
fake.fake_largest_block(C.c_size_t(2 ** 64 - 1))
"""


@pytest.mark.parametrize("shape", WHOLE)
def test_products_without_scratch(shape):
    (found,), = on_fake(BARE + RUN, cases=[[*shape, False, 0]])
    assert found == WHOLE[shape] and len(PRODUCTS[shape]) == 2


@pytest.mark.parametrize("shape", BLOCKS)
def test_gated_blocks_without_scratch(shape):
    made, = on_fake(BARE + RUN, cases=[[*shape, OUT, False, ROOM[shape]]])
    assert made[0] == BLOCKS[shape] and made[1].startswith("rows_vec<3,")
    assert len(GATED[shape]) == 2


def test_every_kernel_is_among_them():
    names = {n for shapes in (PRODUCTS, GATED) for k in shapes.values()
             for n in k}
    names |= {n for k in PRODUCTS.values() for n in with_gelu(k)}
    assert names == {
        "dot<1, false>", "dot<2, false>", "dot<2, true>", "tile_reduce",
        "gated_reduce",
        *(f"skinny_reduce<{g}>" for g in ("false", "true")),
        *(f"narrow<{w}, {g}>" for w in (1, 2) for g in ("false", "true")),
        *(f"skinny<{mb}, {g}>" for mb in (1, 2, 3, 4)
          for g in ("false", "true")),
        *(f"gemm<{e}, false, {jb}>" for e in (0, 1, 5)
          for jb in (4, 5, 6, 7, 8)),
        # few tiles of 128 and of 224 rows are never left over
        *(f"gemm<{e}, false, {jb}>" for e in (3, 4) for jb in (5, 6, 8))}
    # and no other product kernel is in the source
    text = open(os.path.join(ROOT, "h3.c_amd", "csrc", "hk_int8.hip")).read()
    found = set(re.findall(r"\bhk_int8_(\w+)\(hk_(?:skinny|gemm)_args",
                           text)) | {"gemm"}
    assert {n.split("<")[0] for n in names} == found


ATTEND = """
out = []
for qn, kf, kn, heads, kv, dim in cases:
    qf = [int(v) for v in np.cumsum([0] + qn)[:-1]]
    if kf is None:
        kf = [64 * int(v) for v in np.cumsum([0] + [
            (n + 63) // 64 for n in kn])[:-1]]
    width = heads * dim
    made = [gpu.new_bf16(sum(qn) * width), gpu.new_bf16(sum(qn) * width),
            gpu.kv_int8(max(f + n for f, n in zip(kf, kn)), kv, dim),
            gpu.sdpa_packed_plan(qf, qn, kf, kn, heads, kv, dim)]
    y, q, cache, plan = made
    gpu.begin(); fake.fake_clear()
    assert gpu.L.h3_hip_sdpa_packed_int8_bf16(gpu.h, y, q, 0, width, cache,
                                              plan, 0.125), gpu.error()
    gpu.submit()
    out.append([l[0] for l in launches()])
    for t in made:
        gpu.free(t)
"""


def of_attention(names):
    at = {"codes": "hk_packed_codes", "joined": "hk_packed_joined",
          "few": "hk_kv8_few", "simple": "hk_kv8_simple"}
    full = [n.replace(n.split("<")[0], at[n.split("<")[0]]) for n in names]
    return ["hk_kv8_unpack"] * names[0].startswith("codes") + full


def test_attention_of_many_rows():
    made = on_fake(ATTEND, cases=[list(c[:-1]) for c in MANY])
    for case, found in zip(MANY, made):
        assert found == of_attention(case[-1]), case
    assert {k for c in MANY for k in c[-1]} == {
        "simple", "joined<64>", "joined<128>",
        *(f"few<{d}>" for d in (32, 64, 96, 128)),
        *(f"codes<{d}>" for d in (64, 96, 128))}


@pytest.mark.parametrize("dim,padded", [(64, 64), (80, 96), (96, 96),
                                        (128, 128)])
def test_attention_of_the_other_cases_of_many_rows(dim, padded):
    few, codes = f"few<{padded}>", f"codes<{padded}>"
    cases = [([FEW], [70], [few]), ([FEW], [100], [few]),
             ([FEW, 1], [100, 128], [few]), ([FEW] * 20, [110] * 20, [few]),
             ([ROWS], [70], [codes, few]), ([ROWS], [100], [codes, few]),
             ([ROWS, 1], [100, 128], [codes, few]),
             ([ROWS] * 3, [110] * 3, [codes, few])]
    made = on_fake(ATTEND, cases=[[q, None, k, 2, 2, dim]
                                  for q, k, _ in cases])
    for case, found in zip(cases, made):
        assert found == of_attention(case[-1]), case


def test_attention_of_many_requests_and_long_ones():
    for count in (63, 64, 65, 150):
        made = on_fake(ATTEND, cases=[
            [[33 + i % 3 for i in range(count)], None,
             [1 + 37 * i % 128 for i in range(count)], 5, 5, 64],
            [[40] * count, [64 * (i % 7) for i in range(count)],
             [1 + 23 * i % 250 for i in range(count)], 5, 5, 64]])
        assert all(m == of_attention(["codes<64>"]) for m in made), count
    made, = on_fake(ATTEND, cases=[[[4096], None, [1475], 8, 8, 64]])
    assert made == of_attention(["codes<64>"])


def test_attention_without_scratch():
    """As test_int8_no_room_gpu.py has it: room from a call of whole items."""
    cases = [[[16384], None, [9720], 8, 8, 128], [[128], None, [9720], 8, 8, 128]]
    text = ATTEND.replace("gpu.begin();", "gpu.begin(); fake.fake_largest_block("
                          "C.c_size_t(0 if qn == [128] else 2 ** 64 - 1));")
    assert on_fake(BARE + text, cases=cases) == [
        of_attention(["codes<128>"])] * 2
