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
