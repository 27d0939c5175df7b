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
