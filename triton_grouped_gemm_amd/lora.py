"""Low-rank adapters of many requests beside a shared projection, differentiable.

    out[m] = weight x[m] + scales[l] lora_b[l] (lora_a[l] x[m])        l = adapters[m]

The adapters are the groups of a grouped product whose rows stand in any order and whose sums go on into the shared product's: one
rounding.  The reference leaves adapters to its callers, who would sort rows for two grouped products (gemm/BF16/m_grouped_gemm_TMA.py:435) and add.
"""
import ctypes
import functools
from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _native
from ._native import require_gpu
from .gemm.BF16.k_grouped_gemm import k_grouped_gemm

MAX_RANK, MAX_SIDE = 128, 1 << 16


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(backward: int, m: int, n: int, k: int, r: int, count: int, device: int) -> int:
    need = ctypes.c_int64(0)
    _native.call("tgg_lora_workspace_bytes", backward, m, n, k, r, count, ctypes.addressof(need))
    return need.value


def _check(x: Tensor, weight: Tensor, lora_a: Tensor, lora_b: Tensor, adapters: Tensor, scales: Optional[Tensor]) -> None:
    if x.dim() != 2 or weight.dim() != 2 or lora_a.dim() != 3 or lora_b.dim() != 3:
        raise ValueError("x must be [M, K], weight [N, K], lora_a [L, R, K] and lora_b [L, N, R], got "
                         f"{tuple(x.shape)}, {tuple(weight.shape)}, {tuple(lora_a.shape)} and {tuple(lora_b.shape)}")
    (m, k), n, (count, r) = x.shape, weight.shape[0], lora_a.shape[:2]
    if weight.shape[1] != k or lora_a.shape[2] != k or lora_b.shape != (count, n, r):
        raise ValueError("x must be [M, K], weight [N, K], lora_a [L, R, K] and lora_b [L, N, R], got "
                         f"{tuple(x.shape)}, {tuple(weight.shape)}, {tuple(lora_a.shape)} and {tuple(lora_b.shape)}")
    if x.dtype not in _native.DTYPE_CODE:
        raise ValueError(f"data type {x.dtype} not supported: bf16 and fp16 are")
    if not x.dtype == weight.dtype == lora_a.dtype == lora_b.dtype:
        raise ValueError("x, weight, lora_a and lora_b must share one data type")
    if n % 8 or k % 8 or not (8 <= n <= MAX_SIDE and 8 <= k <= MAX_SIDE):
        raise ValueError(f"N and K must be multiples of 8 up to {MAX_SIDE} (16-byte rows), got {n} and {k}")
    if r % 8 or not 8 <= r <= MAX_RANK:
        raise ValueError(f"the rank must be a multiple of 8 up to {MAX_RANK} (fill lora_a and lora_b with zeros), got {r}")
    if not 1 <= count <= _native.MAX_GROUPS:
        raise ValueError(f"the number of adapters must be in [1, {_native.MAX_GROUPS}], got {count}")
    if adapters.shape != (m,) or adapters.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"adapters must be an int32 or int64 tensor with one entry per row of x, got {tuple(adapters.shape)} {adapters.dtype}")
    if scales is not None and (scales.shape != (count,) or scales.dtype != torch.float32):
        raise ValueError(f"scales must be an fp32 tensor with one entry per adapter, got {tuple(scales.shape)} {scales.dtype}")
    if not all(t.device == x.device for t in (weight, lora_a, lora_b, adapters) + (() if scales is None else (scales,))):
        raise ValueError("all operands must live on one GPU")


def _aligned(t: Tensor) -> Tensor:
    """``t`` as the kernels take it, contiguous and from a multiple of 16 bytes on: a slice of a flat buffer is copied, and so is a gradient that autograd hands back as one."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _launch(x, weight, lora_a, lora_b, adapters, scales, keep_h: bool):
    _check(x, weight, lora_a, lora_b, adapters, scales)
    require_gpu(x)
    (m, k), n, (count, r) = x.shape, weight.shape[0], lora_a.shape[:2]
    x, weight, lora_a, lora_b = (_aligned(t) for t in (x, weight, lora_a, lora_b))
    adapters = adapters.contiguous()
    scales = None if scales is None else scales.contiguous()
    out = x.new_empty(m, n)
    h = x.new_empty(m, r, dtype=torch.float32) if keep_h else None
    if m:
        with torch.cuda.device(x.device):
            need = _workspace_bytes(0, m, n, k, r, count, x.device.index)
            ws = torch.empty(need, dtype=torch.uint8, device=x.device)
            _native.call("tgg_lora_linear", x.data_ptr(), weight.data_ptr(), lora_a.data_ptr(), lora_b.data_ptr(), adapters.data_ptr(),
                         int(adapters.dtype == torch.int64), _native.ptr(scales), out.data_ptr(), _native.ptr(h), m, n, k, r, count,
                         _native.DTYPE_CODE[x.dtype], ws.data_ptr(), need, _native.stream_of(x))
    return out, h


@torch.library.custom_op("moe::lora_linear", mutates_args=())
def _lora_linear(x: Tensor, weight: Tensor, lora_a: Tensor, lora_b: Tensor, adapters: Tensor, scales: Optional[Tensor]) -> Tensor:
    return _launch(x, weight, lora_a, lora_b, adapters, scales, False)[0]


@_lora_linear.register_fake
def _(x, weight, lora_a, lora_b, adapters, scales):
    return x.new_empty(x.shape[0], weight.shape[0])


@torch.library.custom_op("moe::lora_linear_hidden", mutates_args=())
def _lora_linear_hidden(x: Tensor, weight: Tensor, lora_a: Tensor, lora_b: Tensor, adapters: Tensor, scales: Optional[Tensor]) -> Tuple[Tensor, Tensor]:
    """Also ``scales[l] lora_a[l] x[m]``, ``[M, R]`` in fp32, which the backward pass takes."""
    return _launch(x, weight, lora_a, lora_b, adapters, scales, True)


@_lora_linear_hidden.register_fake
def _(x, weight, lora_a, lora_b, adapters, scales):
    return x.new_empty(x.shape[0], weight.shape[0]), x.new_empty(x.shape[0], lora_a.shape[1], dtype=torch.float32)


@torch.library.custom_op("moe::lora_linear_backward", mutates_args=())
def _lora_linear_backward(grad: Tensor, x: Tensor, weight: Tensor, lora_a: Tensor, lora_b: Tensor, adapters: Tensor, scales: Optional[Tensor],
                          h: Tensor, want_x: bool, want_a: bool, want_b: bool) -> Tuple[Tensor, Tensor, Tensor]:
    """The gradients of ``x``, ``lora_a`` and ``lora_b``; an empty tensor for one that is not wanted."""
    _check(x, weight, lora_a, lora_b, adapters, scales)
    (m, k), n, (count, r) = x.shape, weight.shape[0], lora_a.shape[:2]
    if grad.shape != (m, n) or grad.dtype != x.dtype:
        raise ValueError(f"grad must be the output's gradient in x's type, got {tuple(grad.shape)} {grad.dtype}")
    if h.shape != (m, r) or h.dtype != torch.float32:
        raise ValueError(f"h must be the [M, R] fp32 tensor of the forward call, got {tuple(h.shape)} {h.dtype}")
    if not grad.device == h.device == x.device:
        raise ValueError("all operands must live on one GPU")
    require_gpu(x)
    grad, x, weight, lora_a, lora_b, h = (_aligned(t) for t in (grad, x, weight, lora_a, lora_b, h))
    adapters = adapters.contiguous()
    scales = None if scales is None else scales.contiguous()
    dx = torch.empty_like(x) if want_x else x.new_empty(0)
    make = torch.empty_like if m else torch.zeros_like
    da = make(lora_a) if want_a else x.new_empty(0)
    db = make(lora_b) if want_b else x.new_empty(0)
    if m and (want_x or want_a or want_b):
        with torch.cuda.device(x.device):
            need = _workspace_bytes(1, m, n, k, r, count, x.device.index)
            ws = torch.empty(need, dtype=torch.uint8, device=x.device)
            _native.call("tgg_lora_linear_bwd", grad.data_ptr(), x.data_ptr(), weight.data_ptr(), lora_a.data_ptr(), lora_b.data_ptr(), adapters.data_ptr(),
                         int(adapters.dtype == torch.int64), _native.ptr(scales), h.data_ptr(), dx.data_ptr() if want_x else 0,
                         da.data_ptr() if want_a else 0, db.data_ptr() if want_b else 0, m, n, k, r, count, _native.DTYPE_CODE[x.dtype],
                         ws.data_ptr(), need, _native.stream_of(x))
    return dx, da, db


@_lora_linear_backward.register_fake
def _(grad, x, weight, lora_a, lora_b, adapters, scales, h, want_x, want_a, want_b):
    return tuple(t.new_empty(t.shape if want else (0,)) for t, want in ((x, want_x), (lora_a, want_a), (lora_b, want_b)))


# (what is registered for them runs in ``lora_linear`` too: see EagerOp)
_lora_linear.__class__ = _lora_linear_hidden.__class__ = _lora_linear_backward.__class__ = _native.EagerOp


class LoraLinear(torch.autograd.Function):
    """``lora_linear`` with the gradients of activations, adapters and, where it is asked for, of the shared weights (the K-grouped product of all
    rows).  ``scales`` has none."""

    @staticmethod
    def forward(ctx, x, weight, lora_a, lora_b, adapters, scales):
        result = None
        if not (_lora_linear_hidden.replaced or torch.compiler.is_compiling()):
            result = (_native._host or _native.host()).lora_linear(x, weight, lora_a, lora_b, adapters, scales, True)
        out, h = result if result is not None else _lora_linear_hidden(x, weight, lora_a, lora_b, adapters, scales)
        ctx.save_for_backward(x, weight, lora_a, lora_b, adapters, scales, h)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, weight, lora_a, lora_b, adapters, scales, h = ctx.saved_tensors
        want = [ctx.needs_input_grad[0], ctx.needs_input_grad[2], ctx.needs_input_grad[3]]
        grads = None
        if any(want) and not (_lora_linear_backward.replaced or torch.compiler.is_compiling()):
            grads = (_native._host or _native.host()).lora_linear_backward(x, weight, lora_a, lora_b, adapters, scales, grad.contiguous(), h, *want)
        if grads is None:
            if not torch.compiler.is_compiling() and _native.has_tangent(grad):
                raise RuntimeError("the gradients of lora_linear have no forward-mode derivative (no jvp): detach what they are multiplied with")
            grads = _lora_linear_backward(grad, x, weight, lora_a, lora_b, adapters, scales, h, *want)
        dx, da, db = (g if w else None for g, w in zip(grads, want))
        dw = None
        if ctx.needs_input_grad[1]:
            if x.shape[0]:
                rows = torch.full((1,), x.shape[0], dtype=torch.int32, device=x.device)
                dw = k_grouped_gemm(_aligned(grad), _aligned(x), rows)[0]
            else:
                dw = torch.zeros_like(weight)
        return dx, dw, da, db, None, None


def lora_linear(x: Tensor, weight: Tensor, lora_a: Tensor, lora_b: Tensor, adapters: Tensor, scales: Optional[Tensor] = None) -> Tensor:
    """``out[m] = weight x[m] + scales[l] lora_b[l] (lora_a[l] x[m])`` with ``l = adapters[m]``, ``[M, N]``.

    ``x`` ``[M, K]``, ``weight`` ``[N, K]``, ``lora_a`` ``[L, R, K]`` and ``lora_b`` ``[L, N, R]`` in bf16 or fp16 (N and K multiples of 8 up to 65536, R one of
    8 up to 128, L up to 1024, M up to 2^27 - 16; operands that are not contiguous, or do not begin at a multiple of 16 bytes, are copied); ``adapters`` ``[M]`` int32 or int64 on the GPU, in any order: a row whose entry is outside ``[0, L)``
    (-1, say) has no adapter; ``scales`` ``[L]`` fp32, 1 unless given.  fp32 sums and one rounding of the result.  The hidden values ``scales[l] lora_a[l] x[m]``
    (in the gradients those of the output's gradient too) are fp32; beyond 128 rows, and in the gradients, they enter the second product in two bfloat16 parts, which leave out at most 2^-17 of each (in ``lora_a``'s and
    ``lora_b``'s gradients two parts of the operands' type).  Differentiable in ``x``, ``weight``,
    ``lora_a`` and ``lora_b``, once and backwards (forward-mode tangents are refused); adapters without rows get zero gradients."""
    if not (_lora_linear.replaced or torch.compiler.is_compiling()):
        out = (_native._host or _native.host()).lora_linear(x, weight, lora_a, lora_b, adapters, scales, False)
        if out is not None:
            return out
    _check(x, weight, lora_a, lora_b, adapters, scales)
    if scales is not None and scales.requires_grad and torch.is_grad_enabled():
        raise ValueError("scales is not differentiable: detach it")
    require_gpu(x)
    if (torch.is_grad_enabled() and any(t.requires_grad for t in (x, weight, lora_a, lora_b))) or torch.compiler.is_compiling() \
            or _native.has_tangent(x, weight, lora_a, lora_b, scales):  # (the function refuses a tangent)
        return LoraLinear.apply(x, weight, lora_a, lora_b, adapters, scales)
    return _lora_linear(x, weight, lora_a, lora_b, adapters, scales)
