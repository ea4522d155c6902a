"""CPU: sizes that the kernels take as 32-bit numbers are refused where they do not fit, not cut off.  (Expanded tensors: sizes without
memory.)"""
import pytest
import torch

from triton_grouped_gemm_amd.gemm.gated import gated_backward, m_grouped_gated_gemm, m_grouped_gated_gemm_projections
from triton_grouped_gemm_amd.gemm.INT4.m_grouped_gemm_int4 import m_grouped_gemm_int4

BEYOND = (1 << 32) + 128  # 128 in 32 bits


def wide(*shape, dtype=torch.bfloat16):
    return torch.zeros((1,) * len(shape), dtype=dtype).expand(shape)


def test_scale_groups_of_the_4_bit_product():
    """One scale for all of K by its shape; cut off to 128 there would be 16 of them to read."""
    x, codes, scales = wide(4, 2048), wide(2, 4, 16, 64, 16, dtype=torch.uint8), wide(2, 1, 64)
    for group_size in (BEYOND, 1 << 31):
        with pytest.raises(ValueError, match="group_size"):
            m_grouped_gemm_int4(x, codes, scales, torch.tensor([2, 2]), group_size)
    with pytest.raises(AssertionError, match="GPU"):
        m_grouped_gemm_int4(x, codes, scales, torch.tensor([2, 2]), (1 << 31) - 128)


def test_lengths_and_columns():
    sizes = torch.tensor([1])
    with pytest.raises(AssertionError, match="32 bits"):
        m_grouped_gemm_int4(wide(1, BEYOND), wide(1, 1, BEYOND // 128, 64, 16, dtype=torch.uint8), wide(1, BEYOND // 128, 16), sizes)
    with pytest.raises(AssertionError, match="32 bits"):
        m_grouped_gemm_int4(wide(1, 128), wide(1, BEYOND // 16, 1, 64, 16, dtype=torch.uint8), wide(1, 1, BEYOND), sizes)
    for call in (m_grouped_gated_gemm, m_grouped_gated_gemm_projections):
        with pytest.raises(AssertionError, match="32 bits"):
            call(wide(1, BEYOND), wide(1, 32, BEYOND), sizes, True)
        with pytest.raises(AssertionError, match="32 bits"):
            call(wide(1, 64), wide(1, 64, BEYOND), sizes, False)
    with pytest.raises(AssertionError, match="32 bits"):
        gated_backward(wide(1, BEYOND), wide(1, 2 * BEYOND, dtype=torch.float32))
