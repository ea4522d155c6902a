"""Gated feed-forward block over expert-contiguous rows: both projections, the activation and the product in one kernel.

``m_grouped_gated_gemm`` computes, for every row r of group g(r) and with ``h = A[r] @ B[g(r)]^T`` (``trans_b``, B is
``[G, 2 F, K]``) or ``A[r] @ B[g(r)]`` (B is ``[G, K, 2 F]``),

    out[r] = act(h[:F]) * h[F:]            act: "silu" x sigma(x), "gelu_tanh" x sigma(2 sqrt(2/pi) (x + 0.044715 x^3))

in fp32 from the product's accumulators to the one rounding at the end.  It stands beside ``m_grouped_gemm`` and takes its
arguments; the layers of the reference run the grouped product (gemm/BF16/m_grouped_gemm_TMA.py:297-462) and the activation
as separate operators.  ``ops.gated_gmm`` is the differentiable form.
"""
from typing import Tuple

import torch
from torch import Tensor
from torch.compiler import is_compiling

from .. import _native
from .BF16.m_grouped_gemm import _sizes_on_device


def _activation_code(activation: str) -> int:
    if activation not in _native.ACTIVATION_CODE:
        raise ValueError(f"activation must be one of {sorted(_native.ACTIVATION_CODE)}, got {activation!r}")
    return _native.ACTIVATION_CODE[activation]


def _gated_launch(A: Tensor, B: Tensor, size_per_group: Tensor, trans_b: bool, activation: str, numSM: int, projections: bool):
    code = _activation_code(activation)
    assert A.dim() == 2 and B.dim() == 3, "A must be [M, K] and B [G, 2 F, K] or [G, K, 2 F]"
    M, K = A.shape
    num_groups, N = B.shape[0], B.shape[1] if trans_b else B.shape[2]
    assert (B.shape[2] if trans_b else B.shape[1]) == K, "K of A should be equal to K of B"
    assert A.dtype in _native.DTYPE_CODE, f"data type {A.dtype} not supported"
    assert A.dtype == B.dtype, "A and B must share one data type"
    assert N % 16 == 0 and N > 0, "B must hold F gate and F up columns, F a multiple of 8 (16-byte rows)"
    assert K % 8 == 0, "K must be a multiple of 8 (16-byte rows)"
    assert K < 1 << 31 and N < 1 << 31, "K and 2 F must fit 32 bits"
    assert size_per_group.dim() == 1 and size_per_group.shape[0] == num_groups, \
        "size_per_group must hold one entry per group of B"
    assert 1 <= num_groups <= _native.MAX_GROUPS, f"at most {_native.MAX_GROUPS} groups are supported"
    _native.require_gpu(A, B)
    assert A.device == B.device, "A and B must live on one GPU"
    A, B = A.contiguous(), B.contiguous()
    out = A.new_empty(M, N // 2)
    h = A.new_empty(M, N, dtype=torch.float32) if projections else None
    if M == 0:
        return out, h
    with torch.cuda.device(A.device):
        sizes, is64 = _sizes_on_device(size_per_group, A.device)
        _native.call("tgg_m_grouped_gated_gemm", A.data_ptr(), B.data_ptr(), out.data_ptr(), _native.ptr(h), sizes.data_ptr(),
                     is64, num_groups, M, N // 2, K, int(bool(trans_b)), code, _native.DTYPE_CODE[A.dtype], int(numSM),
                     _native.stream_of(A))
    return out, h


@torch.library.custom_op("moe::m_grouped_gated_gemm", mutates_args=())
def m_grouped_gated_gemm(A: Tensor, B: Tensor, size_per_group: Tensor, trans_b: bool = False, activation: str = "silu",
                         numSM: int = -1) -> Tensor:
    return _gated_launch(A, B, size_per_group, trans_b, activation, numSM, False)[0]


@m_grouped_gated_gemm.register_fake
def _(A, B, size_per_group, trans_b=False, activation="silu", numSM=-1):
    return A.new_empty(A.shape[0], (B.shape[1] if trans_b else B.shape[2]) // 2)


@torch.library.custom_op("moe::m_grouped_gated_gemm_projections", mutates_args=())
def m_grouped_gated_gemm_projections(A: Tensor, B: Tensor, size_per_group: Tensor, trans_b: bool = False,
                                     activation: str = "silu", numSM: int = -1) -> Tuple[Tensor, Tensor]:
    return _gated_launch(A, B, size_per_group, trans_b, activation, numSM, True)


@m_grouped_gated_gemm_projections.register_fake
def _(A, B, size_per_group, trans_b=False, activation="silu", numSM=-1):
    N = B.shape[1] if trans_b else B.shape[2]
    return A.new_empty(A.shape[0], N // 2), A.new_empty(A.shape[0], N, dtype=torch.float32)


@torch.library.custom_op("moe::gated_backward", mutates_args=())
def gated_backward(grad: Tensor, h: Tensor, activation: str = "silu") -> Tensor:
    code = _activation_code(activation)
    assert grad.dim() == 2 and h.dim() == 2 and h.shape == (grad.shape[0], 2 * grad.shape[1]), \
        "grad must be [M, F] and h [M, 2 F]"
    assert grad.dtype in _native.DTYPE_CODE and h.dtype == torch.float32, f"data types {grad.dtype} and {h.dtype} not supported"
    assert grad.shape[1] % 8 == 0 and grad.shape[1] > 0, "F must be a multiple of 8 (16-byte rows)"
    assert grad.shape[1] < 1 << 30, "2 F must fit 32 bits"
    _native.require_gpu(grad, h)
    assert grad.device == h.device, "grad and h must live on one GPU"
    grad, h = grad.contiguous(), h.contiguous()
    dh = grad.new_empty(h.shape)
    if not h.shape[0]:
        return dh
    with torch.cuda.device(h.device):
        _native.call("tgg_gated_backward", grad.data_ptr(), h.data_ptr(), dh.data_ptr(), grad.shape[0], grad.shape[1], code,
                     _native.DTYPE_CODE[grad.dtype], _native.stream_of(h))
    return dh


@gated_backward.register_fake
def _(grad, h, activation="silu"):
    return grad.new_empty(h.shape)


class _Gated(_native.EagerOp):
    """The operator ``moe::m_grouped_gated_gemm``: ``out [M, F]``; rows past ``sum(size_per_group)`` are left uninitialised,
    as in ``m_grouped_gemm``.  An ordinary eager call goes to the kernel directly."""
    __name__ = "m_grouped_gated_gemm"

    def __call__(self, A: Tensor, B: Tensor, size_per_group: Tensor, trans_b: bool = False, activation: str = "silu",
                 numSM: int = -1) -> Tensor:
        if not (self.replaced or is_compiling()):
            out = (_native._host or _native.host()).m_grouped_gated_gemm(A, B, size_per_group, trans_b, activation, numSM, False)
            if out is not None:
                return out
        return super().__call__(A, B, size_per_group, trans_b, activation, numSM)


class _GatedProjections(_native.EagerOp):
    """The operator ``moe::m_grouped_gated_gemm_projections``: ``(out [M, F], h [M, 2 F])``, h the projections in fp32,
    which ``gated_backward`` takes."""
    __name__ = "m_grouped_gated_gemm_projections"

    def __call__(self, A: Tensor, B: Tensor, size_per_group: Tensor, trans_b: bool = False, activation: str = "silu",
                 numSM: int = -1) -> Tuple[Tensor, Tensor]:
        if not (self.replaced or is_compiling()):
            both = (_native._host or _native.host()).m_grouped_gated_gemm(A, B, size_per_group, trans_b, activation, numSM, True)
            if both is not None:
                return both
        return super().__call__(A, B, size_per_group, trans_b, activation, numSM)


class _GatedBackward(_native.EagerOp):
    """The operator ``moe::gated_backward``: the gradient of ``h`` from that of ``out = act(h[:, :F]) * h[:, F:]``, every row."""
    __name__ = "gated_backward"

    def __call__(self, grad: Tensor, h: Tensor, activation: str = "silu") -> Tensor:
        if not (self.replaced or is_compiling()):
            dh = (_native._host or _native.host()).gated_backward(grad, h, activation)
            if dh is not None:
                return dh
        return super().__call__(grad, h, activation)


m_grouped_gated_gemm.__class__ = _Gated
m_grouped_gated_gemm_projections.__class__ = _GatedProjections
gated_backward.__class__ = _GatedBackward
