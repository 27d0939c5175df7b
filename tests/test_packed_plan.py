"""The work list of a packed attention's plan, and the kernels as compiled,
without a GPU."""
import os
import random
import shutil
import subprocess
import tempfile

import numpy as np
import pytest

from conftest import ROOT
from requests_oracle import on_fake
from test_attn_isa import HIPCC, _offenders

PLAN = """
out = []
for qn, kn, heads, kv, dim in cases:
    qf = [int(v) for v in np.cumsum([0] + qn)[:-1]]
    kf = [int(v) for v in np.cumsum([0] + kn)[:-1]]
    q, k = gpu.new_bf16(sum(qn) * heads * dim), gpu.new_bf16(
        max(1, sum(kn)) * kv * dim)
    y = gpu.new_bf16(sum(qn) * heads * dim)
    plan = gpu.sdpa_packed_plan(qf, qn, kf, kn, heads, kv, dim)
    gpu.begin(); fake.fake_clear()
    ok = gpu.L.h3_hip_sdpa_packed_bf16(
        gpu.h, y, q, 0, heads * dim, k, 0, k, 0, kv * dim, plan, 1.0)
    assert ok, gpu.error()
    n = gpu.L.h3_gpu_tensor_elements(plan)
    out.append([launches(), contents(plan, n).tolist()])
    for t in (q, k, y, plan):
        gpu.free(t)
    gpu.submit()
"""
QB, WHOLE = 128, 0xFFFFFFFF


def lists(case):
    qn, kn, heads, kv, dim = case
    (made, words), = on_fake(PLAN, cases=[case])
    requests = sum(n > 0 for n in qn)
    items = made[0][1]
    joins = made[1][1] if len(made) > 1 else 0
    words = np.array(words, np.int64)
    at = requests * 5
    assert len(words) == at + items * 9 + joins * 6
    return (made, words[at:at + items * 9].reshape(items, 9),
            words[at + items * 9:].reshape(joins, 6))


def cover(case):
    """Every key tile of every row block and key head is in one item, pieces
    lie side by side, and their joins name them all."""
    qn, kn, heads, kv, dim = case
    made, items, joins = lists(case)
    group = heads // kv
    seen, ends = {}, {}
    for qf, rows, row, head, kf, kr, t0, t1, part in items.tolist():
        if rows == 0:
            continue
        seen.setdefault((qf, row, head), []).append((t0, t1, part))
        i = next(i for i in range(len(qn)) if sum(qn[:i]) == qf and qn[i])
        assert row < rows <= qn[i] * group and kr == kn[i]
        assert kf == sum(kn[:i]) and ends.setdefault((qf, row, head),
                                                     rows) == rows
    # rows in blocks of one size, 128 or 32, whole but for a request's last
    qb = 32 if any(row % QB for _, row, _ in seen) else QB
    want = {(sum(qn[:i]), b, h): min(b + qb, qn[i] * group)
            for i in range(len(qn))
            for b in range(0, qn[i] * group, qb) for h in range(kv)}
    assert ends == want
    joined = {(qf, row, head): (part, pieces)
              for qf, _, row, head, part, pieces in joins.tolist()}
    used = []
    for (qf, row, head), pieces in seen.items():
        i = next(i for i in range(len(qn)) if sum(qn[:i]) == qf and qn[i])
        tiles = -(-kn[i] // 64)
        pieces.sort()
        assert pieces[0][0] == 0 and pieces[-1][1] == tiles
        assert all(a[1] == b[0] for a, b in zip(pieces, pieces[1:]))
        if len(pieces) == 1:
            assert pieces[0][2] == WHOLE and (qf, row, head) not in joined
            continue
        assert all(a < b for a, b, _ in pieces), "an empty piece"
        first, count = joined.pop((qf, row, head))
        assert [p for _, _, p in pieces] == list(range(first, first + count))
        used += [p for _, _, p in pieces]
    assert not joined and sorted(used) == list(range(len(used)))
    return made, items, joins


@pytest.mark.parametrize("case", [
    ([1], [1], 1, 1, 64), ([1], [0], 4, 2, 128), ([0, 5, 0], [9, 0, 3], 4, 4, 128),
    ([1] * 16, [20, 33, 512, 77, 126, 1, 300, 64, 65, 63, 200, 411, 90, 18, 256,
                150], 40, 40, 128),
    ([1] * 8, [9720, 6144, 8191, 4096, 5000, 9001, 7777, 6145], 64, 8, 128),
    ([1536, 778], [512, 126], 40, 40, 128), ([6144] * 4, [512, 77, 300, 0], 40,
                                             40, 128),
    ([778, 1536, 2378], [778, 1536, 2378], 56, 56, 128),
    ([1], [33240], 1, 1, 128), ([33240], [33240], 1, 1, 64),
    ([3, 200], [20000, 1], 128, 1, 64)])
def test_every_tile_once(case):
    cover(case)


def test_every_tile_once_at_random():
    rng = random.Random(5)
    for _ in range(12):
        n = rng.randint(1, 20)
        group, kv = rng.choice([1, 2, 5, 8]), rng.choice([1, 3, 8])
        cover(([rng.choice([0, 1, 2, 65, 300]) for _ in range(n)] + [1],
               [rng.choice([0, 1, 64, 700, 9000]) for _ in range(n + 1)],
               group * kv, kv, rng.choice([64, 128])))


def test_long_items_are_cut():
    made, items, joins = cover(([1] * 8, [6144] * 8, 64, 8, 128))
    # 64 long items on 512 places: cut, each place at most one, and joined
    assert len(joins) == 64 and len(made) == 2 and len(items) == 512
    assert made[1][2] == 2  # 8 rows each, four a workgroup
    assert made[0][0] == "hk_packed_flash<128>"
    made, items, joins = cover(([6144] * 2, [512] * 2, 40, 40, 128))
    assert not len(joins) and len(made) == 1


@pytest.mark.parametrize("dim,kernel", [
    (1, "hk_packed_simple"), (8, "hk_packed_flash<64>"),
    (64, "hk_packed_flash<64>"), (72, "hk_packed_flash<96>"),
    (96, "hk_packed_flash<96>"), (104, "hk_packed_flash<128>"),
    (100, "hk_packed_simple"), (128, "hk_packed_flash<128>"),
    (136, "hk_packed_simple"), (256, "hk_packed_simple")])
def test_kernel_by_head_size(dim, kernel):
    (made, _), = on_fake(PLAN, cases=[([5], [70], 2, 1, dim)])
    assert made[0][0] == kernel


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not installed")
def test_flash_kernels_wait_for_their_transposed_reads():
    """As test_attn_isa.py, for the packed kernel with its own flags."""
    work = tempfile.mkdtemp(prefix="hk_packed_isa_")
    try:
        subprocess.run(
            [HIPCC, "-O3", "-std=c++17", "-fPIC", "--offload-arch=gfx950",
             "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
             "-mllvm", "-amdgpu-mfma-vgpr-form", "-fno-signed-zeros",
             "-fno-trapping-math", "-fassociative-math",
             "-freciprocal-math", "--save-temps", "-c",
             os.path.join(ROOT, "h3.c_amd", "csrc", "hk_packed.hip"), "-o",
             os.path.join(work, "x.o")], cwd=work, check=True,
            capture_output=True)
        asm, = (f for f in os.listdir(work)
                if f.endswith(".s") and "amdgcn" in f)
        text = open(os.path.join(work, asm)).read().splitlines()
    finally:
        shutil.rmtree(work, ignore_errors=True)
    found, name = {}, None
    for line in text:
        if line.startswith("_Z15hk_packed_flashI") and ":" in line:
            name = line.split(":")[0]
            found[name] = []
        elif name and line.startswith(".Lfunc_end"):
            name = None
        elif name:
            found[name].append(line)
    assert len(found) == 3
    for name, body in found.items():
        assert any("ds_read_b64_tr_b16" in l for l in body), name
        assert not _offenders(body), (name, _offenders(body)[:3])


def test_items_behind_the_last_full_round_are_cut():
    # 1064 items on 256 CUs: the last 40 in pieces, the others whole
    made, items, joins = cover(([2378], [2378], 56, 56, 128))
    assert len(joins) == 40 and len(made) == 2
    assert sum(items[:, 8] == WHOLE) == 1024
    made, items, joins = cover(([77, 1200], [77, 1200], 56, 56, 128))
    assert len(joins) and len(made) == 2
    # five rounds, and 2.8
    for rows in (4096, 2185):
        made, items, joins = cover(([rows], [rows], 40, 40, 128))
        assert not len(joins) and len(made) == 1


def test_few_items_are_of_few_rows():
    # 48 items of 128 rows; 102 of which the small ones would be 400
    for qn, heads, small in (([700], 8, 176), ([300], 40, 0), ([1], 8, 0)):
        made, items, joins = cover((qn, qn, heads, heads, 128))
        sizes = items[items[:, 1] > 0]
        assert not len(joins)
        assert (sizes[:, 1] - sizes[:, 2]).max() <= (32 if small else 128)
        assert not small or len(sizes) == small
    # long contexts are cut instead
    made, items, joins = cover(([128], [9720], 8, 8, 128))
    assert len(joins) == 8
