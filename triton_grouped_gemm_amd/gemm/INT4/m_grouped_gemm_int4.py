"""M-grouped products with 4-bit weights and group scales: the experts' projections of a decode step.

``m_grouped_gemm_int4`` computes, for every row r of group g(r),

    y[r] = A[r] @ W[g(r)]^T,    W[g][n, k] = (q[n, k] - z[n, k // group_size]) * s[n, k // group_size],    q in 0..15

(z = 8 unless ``zeros`` is given, whose bytes are 0..15 like the codes) and returns ``y``, or with ``activation`` the gated block
``act(y[:F]) * y[F:]`` of N = 2 F columns, as ``m_grouped_gated_gemm`` does.  Sums are fp32, the weights are not rounded, the result is
rounded once.  ``quant.int4_cast`` makes the operands: ``per_group_cast_to_int4`` from 16-bit weights, ``pack_int4`` from 4-bit values.

Two limits, because bfloat16 operands are biased codes, 128 + q or 144 + q - z, whose bias is taken back in the fp32 sums: zero points lie on the
device and are not checked, and one above 15 gives wrong weights; and a row of A with infinities, or with magnitudes that add up to more than
2e36 within 128 values of K, gives NaN or infinity.

It stands beside ``m_grouped_gemm`` (gemm/BF16/m_grouped_gemm_TMA.py:297-462 of the reference, which has no 4-bit weights) and
is meant for few rows a group: the codes are read once for up to 64 rows of a group.
"""
from typing import Optional

import torch
from torch import Tensor
from torch.compiler import is_compiling

from ... import _native
from ..BF16.m_grouped_gemm import _sizes_on_device


@torch.library.custom_op("moe::m_grouped_gemm_int4", mutates_args=())
def m_grouped_gemm_int4(A: Tensor, codes: Tensor, scales: Tensor, size_per_group: Tensor, group_size: int = 128,
                        zeros: Optional[Tensor] = None, activation: Optional[str] = None, numSM: int = -1) -> Tensor:
    if activation is not None and activation not in _native.ACTIVATION_CODE:
        raise ValueError(f"activation must be None or one of {sorted(_native.ACTIVATION_CODE)}, got {activation!r}")
    if group_size not in (32, 64) and (not 128 <= group_size < 1 << 31 or group_size % 128):
        raise ValueError(f"group_size must be 32, 64 or a multiple of 128 below 2^31, got {group_size}")
    assert A.dim() == 2, "A must be [M, K]"
    assert A.dtype in _native.DTYPE_CODE, f"data type {A.dtype} not supported"
    assert scales.dim() == 3 and scales.dtype == A.dtype, "scales must be [G, ceil(K / group_size), N] in A's type"
    M, K = A.shape
    num_groups, scale_groups, N = scales.shape
    assert K % 8 == 0 and K > 0 and N % 8 == 0 and N > 0, "K and N must be multiples of 8 (16-byte rows)"
    assert K < 1 << 31 and N < 1 << 31, "K and N must fit 32 bits"
    assert scale_groups == -(-K // group_size), "scales must hold one row per group of group_size values of K"
    assert codes.dtype == torch.uint8 and codes.shape == (num_groups, -(-N // 16), -(-K // 128), 64, 16), \
        "codes must be what pack_int4 returns for [G, N, K] values"
    assert zeros is None or (zeros.dtype == torch.uint8 and zeros.shape == scales.shape), "zeros must be uint8 of the scales' shape"
    assert activation is None or N % 32 == 0, "a gated block needs gate and up columns in multiples of 16"
    assert size_per_group.dim() == 1 and size_per_group.shape[0] == num_groups, \
        "size_per_group must hold one entry per group of codes"
    assert 1 <= num_groups <= _native.MAX_GROUPS, f"at most {_native.MAX_GROUPS} groups are supported"
    _native.require_gpu(A, codes, scales, zeros)
    assert codes.device == A.device and scales.device == A.device and (zeros is None or zeros.device == A.device), \
        "all operands must live on one GPU"
    A, codes, scales = A.contiguous(), codes.contiguous(), scales.contiguous()
    zeros = None if zeros is None else zeros.contiguous()
    out = A.new_empty(M, N if activation is None else N // 2)
    if M == 0:
        return out
    with torch.cuda.device(A.device):
        sizes, is64 = _sizes_on_device(size_per_group, A.device)
        _native.call("tgg_m_grouped_gemm_int4", A.data_ptr(), codes.data_ptr(), scales.data_ptr(), _native.ptr(zeros), out.data_ptr(),
                     sizes.data_ptr(), is64, num_groups, M, N, K, group_size,
                     -1 if activation is None else _native.ACTIVATION_CODE[activation], _native.DTYPE_CODE[A.dtype], int(numSM),
                     _native.stream_of(A))
    return out


@m_grouped_gemm_int4.register_fake
def _(A, codes, scales, size_per_group, group_size=128, zeros=None, activation=None, numSM=-1):
    return A.new_empty(A.shape[0], scales.shape[2] if activation is None else scales.shape[2] // 2)


class _MGroupedGemmInt4(_native.EagerOp):
    """The operator ``moe::m_grouped_gemm_int4``: ``zeros`` are bytes 0..15 (not looked at: others give wrong weights in bfloat16); rows past ``sum(size_per_group)`` are left uninitialised, as in
    ``m_grouped_gemm``.  An ordinary eager call goes to the kernel directly."""
    __name__ = "m_grouped_gemm_int4"

    def __call__(self, A: Tensor, codes: Tensor, scales: Tensor, size_per_group: Tensor, group_size: int = 128,
                 zeros: Optional[Tensor] = None, activation: Optional[str] = None, numSM: int = -1) -> Tensor:
        if not (self.replaced or is_compiling()):
            out = (_native._host or _native.host()).m_grouped_gemm_int4(A, codes, scales, size_per_group, group_size, zeros,
                                                                        activation, numSM)
            if out is not None:
                return out
        return super().__call__(A, codes, scales, size_per_group, group_size, zeros, activation, numSM)


m_grouped_gemm_int4.__class__ = _MGroupedGemmInt4
