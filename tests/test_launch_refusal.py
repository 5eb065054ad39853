"""pt_launch refuses 2^32 threads and more, of which HIP would keep the low 32 bits, before it touches a device."""
import ctypes

import pytest

from phptensors import _abi


@pytest.mark.parametrize("blocks,threads", [(1 << 24, 256), ((1 << 32) - 1, 2), (1 << 22, 1024), (1 << 31, 64)])
def test_threads_past_32_bits(blocks, threads):
    never_read = ctypes.c_void_p(4096)
    assert _abi.load().pt_launch(never_read, blocks, threads, None, None) == _abi.PT_ERR_INVALID
    assert "2^32" in _abi.last_error()


def test_no_blocks():
    assert _abi.load().pt_launch(ctypes.c_void_p(4096), 0, 256, None, None) == _abi.PT_OK
