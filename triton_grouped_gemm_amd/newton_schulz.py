"""Newton-Schulz orthogonalisation of stacks of matrices, and the optimiser's step that uses it.

``gmm``'s weight gradients are stacks ``[G, K, N]`` or ``[G, N, K]``, those of adapters ``[L, R, K]`` and ``[L, N, R]``: every matrix of such a
stack is brought near the orthogonal one of its singular vectors by ``steps`` products

    X = x / (|x|_F + eps),    X <- a X + (b X X^T + c (X X^T)^2) X

which raise its singular values towards 1.  The reference has no optimiser.
"""
import ctypes
import functools
import math
from typing import Optional, Sequence, Tuple

import torch
from torch import Tensor

from . import _native
from ._native import require_gpu

_TYPE_CODE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
MAX_STEPS, MAX_SIDE = 100, 1 << 16


@functools.lru_cache(maxsize=256)
def _workspace_bytes(batch: int, rows: int, cols: int, device: int) -> int:
    need = ctypes.c_int64(0)
    _native.call("tgg_newton_schulz_workspace_bytes", batch, rows, cols, ctypes.addressof(need))
    return need.value


def _check(name: str, x: Tensor, steps: int, coefficients: Sequence[float], eps: float) -> Tuple[int, int, int]:
    """``(matrices, rows, columns)`` of a stack."""
    if x.dim() < 2 or x.dtype not in _TYPE_CODE:
        raise ValueError(f"{name} must be a [..., rows, columns] tensor in bf16, fp16 or fp32, got {tuple(x.shape)} {x.dtype}")
    rows, cols = x.shape[-2:]
    if not (1 <= rows <= MAX_SIDE and 1 <= cols <= MAX_SIDE):
        raise ValueError(f"{name}'s matrices must have between 1 and {MAX_SIDE} rows and columns, got {rows} x {cols}")
    if not 0 <= steps <= MAX_STEPS:
        raise ValueError(f"steps must be in [0, {MAX_STEPS}], got {steps}")
    if len(coefficients) != 3 or not all(math.isfinite(c) for c in coefficients):
        raise ValueError(f"coefficients must be three finite numbers, got {tuple(coefficients)}")
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    return math.prod(x.shape[:-2]), rows, cols


def _refuse_tangents(name: str, *tensors: Tensor) -> None:
    if not torch.compiler.is_compiling() and _native.has_tangent(*tensors):
        raise RuntimeError(f"{name} has no forward-mode derivative (no jvp): detach its operands")


def _workspace(batch: int, rows: int, cols: int, device: torch.device):
    need = _workspace_bytes(batch, rows, cols, device.index)
    return torch.empty(need, dtype=torch.uint8, device=device), need


@torch.library.custom_op("moe::orthogonalize", mutates_args=())
def _orthogonalize(x: Tensor, steps: int, a: float, b: float, c: float, eps: float) -> Tensor:
    batch, rows, cols = _check("x", x, steps, (a, b, c), eps)
    require_gpu(x)
    x = x.contiguous()
    out = torch.empty_like(x)
    if batch:
        with torch.cuda.device(x.device):
            workspace, need = _workspace(batch, rows, cols, x.device)
            _native.call("tgg_newton_schulz", x.data_ptr(), out.data_ptr(), batch, rows, cols, steps, a, b, c, eps, _TYPE_CODE[x.dtype],
                         workspace.data_ptr(), need, _native.stream_of(x))
    return out


@_orthogonalize.register_fake
def _(x, steps, a, b, c, eps):
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def orthogonalize(x: Tensor, steps: int = 5, coefficients: Sequence[float] = COEFFICIENTS, eps: float = 1e-7) -> Tensor:
    """Every matrix of ``x`` ``[..., rows, columns]`` (bf16, fp16 or fp32, any sizes up to 65536) after ``steps`` Newton-Schulz products, in its type.

    Multiplied and carried from step to step in 22 bits with fp32 sums, whatever the type, and rounded once at the end.  (What that leaves out grows in weak directions as they do, by up to
    3.4445 a step, and entries below 2^-13 of the norm have fewer bits.)  The workspace is 8 bytes times the shorter side times the sum of both sides a matrix: 7 times a bf16 stack of 1536 x 2048.  A matrix of zeros stays one (unless ``eps`` is 0); one with a NaN or an infinity becomes
    NaN, and no other of the stack is touched by it.  ``coefficients`` have to keep singular values near 1 (entries below 64).  Not differentiable, in either mode."""
    coefficients = tuple(float(v) for v in coefficients)
    steps, eps = int(steps), float(eps)
    _check("x", x, steps, coefficients, eps)
    _refuse_tangents("orthogonalize", x)
    require_gpu(x)
    return _orthogonalize(x, steps, *coefficients, eps)


@torch.library.custom_op("moe::muon_update", mutates_args=("weight", "momentum"))
def _muon_update(weight: Tensor, grad: Tensor, momentum: Tensor, keep: float, step: float, beta: float, nesterov: bool, steps: int,
                 a: float, b: float, c: float, eps: float) -> None:
    batch, rows, cols = _check_muon(weight, grad, momentum, steps, (a, b, c), eps)
    require_gpu(weight, grad, momentum)
    grad = grad.contiguous()
    if any(_overlap(p, q) for p, q in ((weight, momentum), (grad, momentum), (weight, grad))):
        raise ValueError("weight, grad and momentum must not share memory")
    if batch:
        with torch.cuda.device(weight.device):
            workspace, need = _workspace(batch, rows, cols, weight.device)
            _native.call("tgg_muon_update", weight.data_ptr(), _TYPE_CODE[weight.dtype], grad.data_ptr(), _TYPE_CODE[grad.dtype], momentum.data_ptr(),
                         batch, rows, cols, keep, step, beta, int(nesterov), steps, a, b, c, eps, workspace.data_ptr(), need,
                         _native.stream_of(weight))


@_muon_update.register_fake
def _(weight, grad, momentum, keep, step, beta, nesterov, steps, a, b, c, eps):
    return None


def _overlap(p: Tensor, q: Tensor) -> bool:
    """Whether two contiguous tensors share memory."""
    return p.data_ptr() < q.data_ptr() + q.numel() * q.element_size() and q.data_ptr() < p.data_ptr() + p.numel() * p.element_size()


def _check_muon(weight: Tensor, grad: Tensor, momentum: Tensor, steps: int, coefficients: Sequence[float], eps: float) -> Tuple[int, int, int]:
    shape = _check("weight", weight, steps, coefficients, eps)
    if grad.shape != weight.shape or grad.dtype not in _TYPE_CODE:
        raise ValueError(f"grad must be a bf16, fp16 or fp32 tensor of weight's shape, got {tuple(grad.shape)} {grad.dtype}")
    if momentum.shape != weight.shape or momentum.dtype != torch.float32:
        raise ValueError(f"momentum must be an fp32 tensor of weight's shape, got {tuple(momentum.shape)} {momentum.dtype}")
    if not (weight.is_contiguous() and momentum.is_contiguous()):
        raise ValueError("weight and momentum are updated in place and must be contiguous")
    if not weight.device == grad.device == momentum.device:
        raise ValueError("all operands must live on one GPU")
    return shape


@torch.no_grad()
def muon_update(weight: Tensor, grad: Tensor, momentum: Tensor, lr: float, beta: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
                scale: Optional[float] = None, steps: int = 5, coefficients: Sequence[float] = COEFFICIENTS, eps: float = 1e-7) -> None:
    """One optimiser step of a stack of matrices ``[..., rows, columns]``, in place:

        momentum = beta momentum + (1 - beta) grad
        u        = beta momentum + (1 - beta) grad   with ``nesterov``, else momentum
        weight   = (1 - lr weight_decay) weight - lr scale orthogonalize(u)

    ``momentum`` is fp32; ``weight`` and ``grad`` are bf16, fp16 or fp32 each.  ``scale`` is ``sqrt(max(1, rows / columns))`` unless given.  ``momentum``, ``weight`` and ``grad`` do not share memory.  The
    direction is multiplied as ``orthogonalize`` does it and the weights are rounded once."""
    coefficients = tuple(float(v) for v in coefficients)
    steps, eps, beta = int(steps), float(eps), float(beta)
    _, rows, cols = _check_muon(weight, grad, momentum, steps, coefficients, eps)
    scale = math.sqrt(max(1.0, rows / cols)) if scale is None else float(scale)
    lr, weight_decay = float(lr), float(weight_decay)
    if not all(math.isfinite(v) for v in (lr, beta, weight_decay, scale)):
        raise ValueError(f"lr, beta, weight_decay and scale must be finite, got {lr}, {beta}, {weight_decay} and {scale}")
    _refuse_tangents("muon_update", weight, grad, momentum)
    require_gpu(weight, grad, momentum)
    _muon_update(weight, grad, momentum, 1.0 - lr * weight_decay, lr * scale, beta, bool(nesterov), steps, *coefficients, eps)
