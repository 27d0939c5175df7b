"""What a packed attention's plan holds for a cache in 8 bits, without a GPU
(requests_oracle.on_fake)."""
import pytest

from requests_oracle import on_fake

PLAN = """
qn, kf, kn, heads, kv, dim = case
qf = [int(v) for v in np.cumsum([0] + qn)[:-1]]
plan = gpu.sdpa_packed_plan(qf, qn, kf, kn, heads, kv, dim)
held = C.c_size_t.from_address(plan + 16).value // 4  # h3_gpu_tensor.bytes
lists = gpu.L.h3_gpu_tensor_elements(plan)
out = [lists, contents(plan, held)[lists:].tolist()]
"""


@pytest.mark.parametrize("qn,kf,kn,heads,kv,dim,spans", [
    ([6144] * 4, [0, 512, 640, 0], [512, 77, 300, 0], 40, 40, 128,
     [(0, 0, 8), (8, 8, 2), (10, 10, 5)]),
    # a text that requests share, whole and in part
    ([4096] * 4, [0, 0, 0, 64], [128, 65, 256, 1], 8, 8, 64,
     [(0, 0, 2), (0, 2, 4), (1, 6, 1)]),
    # a request of few rows has no part in it, nor has a row behind 128
    ([129, 1, 32, 33], [0, 128, 192, 256], [70, 64, 60, 128], 2, 2, 64,
     [(0, 0, 2), (4, 2, 2)]),
    # items of 32 rows; keys that do not begin at whole blocks; none
    ([700], [0], [700], 8, 8, 128, []), ([6144], [3], [512], 40, 40, 128, []),
    ([6144], [0], [0], 40, 40, 128, [])])
def test_spans_of_blocks(qn, kf, kn, heads, kv, dim, spans):
    """Three words for each range of blocks that requests of many rows read, and
    nothing for each of the plan's items."""
    _, words = on_fake(PLAN, case=[qn, kf, kn, heads, kv, dim])
    assert words == [w for s in spans for w in s]
