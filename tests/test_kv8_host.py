"""What of the 8-bit K/V entries needs no GPU: a state's size and its refusals, and calls without a handle."""
import pytest

from kv8_util import state_bytes
from straydog_b200 import _lib


@pytest.mark.parametrize("context,kv_heads,dim", [(32, 1, 64), (64, 3, 128), (32768, 2, 256), (1 << 24, 8, 128)])
def test_the_size_of_a_state(context, kv_heads, dim):
    assert _lib.load().sdx_kv8_bytes(context, kv_heads, dim) == state_bytes(context, kv_heads, dim)


@pytest.mark.parametrize("context,kv_heads,dim", [(0, 1, 64), (33, 1, 64), (1 << 25, 1, 64), (32, 0, 64), (32, 1025, 64), (32, 1, 96), (32, 1, 0)])
def test_sizes_that_are_none(context, kv_heads, dim):
    lib = _lib.load()
    assert lib.sdx_kv8_bytes(context, kv_heads, dim) == 0
    assert lib.sd_error()


def test_a_null_handle_is_an_error():
    lib = _lib.load()
    assert lib.sdx_kv8_write(None, None, None, None, None, 1, 1, 64, 0, None, None, 0, 0) == -1
    assert lib.sdx_kv8_attention(None, None, None, None, None, 1, 1, 1, 64, 0, 1.0, 0.0, None, 0, None, None, 0, None, None, 0, 1) == -1
    assert lib.sdx_masked_attention(None, None, 0, None, 0, None, 0, None, None, 1, 1, 1, 64, 1, 1.0, 0.0, None, 0, None, None, 0) == -1
    assert lib.sdx_kv8_evict(None, None, None, None, None, 1, 1, 0, 0, 1, 64, 0, None, None, None, None) == -1
    assert b"handle" in lib.sd_error()
