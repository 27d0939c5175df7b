"""What the Python binding of the 8-bit operators refuses by itself, without a
GPU (requests_oracle.on_fake)."""
import pytest

from requests_oracle import on_fake


@pytest.mark.parametrize("first,source,rows,taken", [
    ([0, 64], [0, 5], [5, 7], True), ([0], [0, 5], [5, 7], False),
    ([0, 64], [5], [5, 7], False), ([0, 64], [0, 5], [5], False)])
def test_store_of_uneven_lists(first, source, rows, taken):
    """A row number that is missing is no 0, which would be a row."""
    said, launched = on_fake("""
cache, kv = gpu.kv_int8(128, 1, 64), gpu.new_bf16(12 * 64)
gpu.begin(); fake.fake_clear()
try:
    gpu.kv_int8_store(cache, *lists, kv, 0, kv, 0, 64)
    out = ""
except ValueError as e:
    out = str(e)
out = [out, len(launches())]
""", lists=[first, source, rows])
    assert (not said and launched) if taken else (said and not launched)
