"""The mask of h3_gpu_sdpa_set_sparse and packed attention."""
import numpy as np
import pytest

from test_packed_gpu import Case
from test_sparse_gpu import clear, random_mask, register

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qn", [[700], [300, 400], [699, 1]])
def test_a_registered_mask_is_not_applied(gpu, qn):
    """Also to as many rows as it was registered for, in one request."""
    a = Case(51, qn, qn, 2, 2, 128)
    want = a.check(gpu)
    ptr, idx = random_mask(np.random.default_rng(1), 700)
    assert register(gpu, ptr, idx, 700), gpu.error()
    try:
        assert (a.run(gpu) == want).all()
    finally:
        clear(gpu)
