"""CPU: the most rows that the adapter entry points take.  A workgroup of 512 threads has 16 rows, and a launch has fewer than 2^32 threads."""
import ctypes

import pytest

from triton_grouped_gemm_amd import _native

MOST = (1 << 27) - 16


@pytest.mark.parametrize("backward", [0, 1])
@pytest.mark.parametrize("rank", [8, 64, 128])
def test_most_rows(backward, rank):
    assert -(-MOST // 16) * 512 < 1 << 32 <= -(-(MOST + 1) // 16) * 512
    need = ctypes.c_int64(-1)
    call = lambda m: _native.load().tgg_lora_workspace_bytes(backward, m, 8, 8, rank, 1, ctypes.addressof(need))
    assert call(MOST) == 0 and need.value > 0
    for m in (MOST + 1, (1 << 27) - 1, 1 << 27):
        assert call(m) == 1 and f"M={m}" in _native.last_error()


def test_calls_of_too_many_rows():
    """(Their workspace is too small as well, so that none of them gets as far as a launch.)"""
    buf = ctypes.create_string_buffer(4096)
    p = ctypes.addressof(buf)
    p += -p % 256
    lib = _native.load()
    assert lib.tgg_lora_linear(p, p, p, p, p, 0, None, p, None, MOST + 1, 8, 8, 8, 1, 0, p, 0, None) == 1 and "M=" in _native.last_error()
    assert lib.tgg_lora_linear_bwd(p, p, p, p, p, p, 0, None, p, p, p, p, MOST + 1, 8, 8, 8, 1, 0, p, 0, None) == 1 and "M=" in _native.last_error()
