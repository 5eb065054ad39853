"""Attention calls whose workgroups a launch does not hold, or whose rows pass 32 bits within the last tile, are refused
before a device is touched."""
import ctypes

import pytest

from phptensors import _abi
from test_operator_refusals import LIB, P, desc, refused

PACKED = dict(q_starts=4096, q_lengths=4096, k_starts=4096, k_lengths=4096)
# 2^24 workgroups of 256 threads are one too many
FORWARD = [dict(sequences=1 << 23, queries=1, keys=1), dict(sequences=1 << 22, queries=65, keys=1, heads=8, kv_heads=4),
           dict(sequences=(1 << 21) + 1, kv_heads=1, queries=64, keys=1),   # a tile a sequence, and the places of 8
           dict(sequences=1, heads=1, kv_heads=1, queries=2 ** 31 - 255, keys=1), dict(sequences=1, queries=1, keys=2 ** 31 - 255)]
BACKWARD = [dict(sequences=1 << 21, queries=1, keys=1, heads=8, kv_heads=8), dict(sequences=1 << 14, queries=1, keys=1 << 16),
            dict(sequences=(1 << 21) + 1, kv_heads=1, queries=1, keys=128)]


@pytest.mark.parametrize("change", FORWARD + BACKWARD, ids=str)
def test_too_many_tiles(change):
    d = ctypes.byref(desc(**change))
    if change in FORWARD:
        refused(LIB.pt_attention(d, P, P, P, P, P, P, None))
    refused(LIB.pt_attention_backward(d, P, P, P, P, P, P, P, _abi.BFLOAT16, P, P, P, None))


def test_bounds_are_cut_before_they_are_counted():
    """Bounds past the tensors' rows are not work: what is refused here is the missing output."""
    change = dict(PACKED, queries=2 ** 31 - 1, keys=2 ** 31 - 1, q_rows=1000, k_rows=1000)
    assert LIB.pt_attention(ctypes.byref(desc(**change)), P, P, P, None, P, P, None) == _abi.PT_ERR_INVALID
    assert "output is missing" in _abi.last_error()
