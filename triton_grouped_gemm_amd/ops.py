"""Differentiable grouped GEMM: forward, activation gradient and weight gradient on the three native kernels.

Mirrors the autograd wrapper of the reference's baseline extension (grouped_gemm/grouped_gemm/ops.py:12-42):
``gmm(a, b, batch_sizes, trans_b=False, num_sm=-1)`` with

    forward   out = a[rows of g] @ b[g]      (or @ b[g].T with trans_b)        M-grouped, layout NN / NT
    d a       grad @ b[g].T                  (or grad @ b[g])                  M-grouped with trans_b flipped
    d b       a_g.T @ grad_g   ([K, N])      (or grad_g.T @ a_g, [N, K])       K-grouped over the group's rows

``batch_sizes`` may live on the host (as the reference's extension requires) or on the device; a device tensor
is used as is, with no host synchronisation.
"""
from typing import Tuple

import torch
from torch import Tensor

from . import _native
from ._native import require_gpu
from .gemm.BF16.k_grouped_gemm import k_grouped_gemm
from .gemm.BF16.m_grouped_gemm import m_grouped_gemm
from .gemm.gated import gated_backward, m_grouped_gated_gemm, m_grouped_gated_gemm_projections


def _device_sizes(batch_sizes: torch.Tensor, device: torch.device) -> torch.Tensor:
    if batch_sizes.dtype not in (torch.int32, torch.int64):
        batch_sizes = batch_sizes.to(torch.int64)
    return batch_sizes.to(device, non_blocking=True)


class GroupedGemm(torch.autograd.Function):
    """grouped_gemm/grouped_gemm/ops.py:12-38."""

    @staticmethod
    def forward(ctx, a, b, batch_sizes, trans_b, num_sm=-1):
        if not batch_sizes.is_cuda:
            # the reference asserts this on its host-side sizes; device-resident sizes are not read back
            assert torch.count_nonzero(batch_sizes) != 0, "Input batch_sizes should not be all zeros!"
        require_gpu(a, b)
        sizes = _device_sizes(batch_sizes, a.device)
        ctx.save_for_backward(a, b, sizes)
        ctx.trans_b = bool(trans_b)
        ctx.num_sm = int(num_sm)
        return m_grouped_gemm(a.contiguous(), b.contiguous(), sizes, ctx.trans_b, ctx.num_sm)

    @staticmethod
    def backward(ctx, grad):
        grad = grad.contiguous()
        a, b, sizes = ctx.saved_tensors
        trans_b = ctx.trans_b
        agrad = None
        if ctx.needs_input_grad[0]:
            agrad = m_grouped_gemm(grad, b.contiguous(), sizes, not trans_b, ctx.num_sm)
        bgrad = None
        if ctx.needs_input_grad[1]:
            lhs, rhs = (grad, a) if trans_b else (a, grad)
            bgrad = k_grouped_gemm(lhs.contiguous(), rhs.contiguous(), sizes, numSM=ctx.num_sm)
        return agrad, bgrad, None, None, None


def _records(*tensors) -> bool:
    """Whether a call on these tensors needs its autograd function: a gradient may be asked for, or the call is traced."""
    return (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)) or torch.compiler.is_compiling()


def gmm(a, b, batch_sizes, trans_b=False, num_sm=-1):
    """grouped_gemm/grouped_gemm/ops.py:41-42."""
    if not _records(a, b) and not m_grouped_gemm.replaced:
        out = (_native._host or _native.host()).m_grouped_gemm(a, b, batch_sizes, bool(trans_b), int(num_sm))
        if out is not None:
            return out
    return GroupedGemm.apply(a, b, batch_sizes, trans_b, num_sm)


class GatedGroupedGemm(torch.autograd.Function):
    """``gated_gmm`` with the gradients of activations and weights: the projections are kept (in fp32: their rounding would be a
    third one in the gradients, beside that of ``dh`` and their own), one pass
    makes their gradient ``dh`` from the output's, and the grouped products of ``dh`` are those of ``gmm``."""

    @staticmethod
    def forward(ctx, a, b, batch_sizes, activation, trans_b, num_sm):
        sizes = _device_sizes(batch_sizes, a.device)
        out, h = m_grouped_gated_gemm_projections(a, b, sizes, bool(trans_b), activation, int(num_sm))
        ctx.save_for_backward(a, b, sizes, h)
        ctx.activation, ctx.trans_b, ctx.num_sm = activation, bool(trans_b), int(num_sm)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        a, b, sizes, h = ctx.saved_tensors
        if not a.shape[0]:  # no rows: nothing to launch
            return torch.zeros_like(a), torch.zeros_like(b), None, None, None, None
        dh = gated_backward(grad.contiguous(), h, ctx.activation)
        agrad = bgrad = None
        if ctx.needs_input_grad[0]:
            agrad = m_grouped_gemm(dh, b.contiguous(), sizes, not ctx.trans_b, ctx.num_sm)
        if ctx.needs_input_grad[1]:
            lhs, rhs = (dh, a.contiguous()) if ctx.trans_b else (a.contiguous(), dh)
            bgrad = k_grouped_gemm(lhs, rhs, sizes, numSM=ctx.num_sm)
        return agrad, bgrad, None, None, None, None


def gated_gmm(a, b, batch_sizes, activation="silu", trans_b=False, num_sm=-1):
    """The gated feed-forward block of every expert: ``act(a_g @ gate_g) * (a_g @ up_g)``, ``[M, F]``, where ``b`` is
    ``[G, K, 2 F]`` (``[G, 2 F, K]`` with ``trans_b``), gate first, and ``activation`` is ``"silu"`` or ``"gelu_tanh"``.  Stands where
    ``gmm``, ``chunk``, the activation and the product would; fp32 from the products to the one rounding of the result."""
    require_gpu(a, b)
    if not _records(a, b):
        return m_grouped_gated_gemm(a, b, _device_sizes(batch_sizes, a.device), bool(trans_b), activation, int(num_sm))
    return GatedGroupedGemm.apply(a, b, batch_sizes, activation, trans_b, num_sm)


# ---------------------------------------------------------------------------------------------------------------
# MoE token permute / unpermute (grouped_gemm/grouped_gemm/ops.py:52-257)
# ---------------------------------------------------------------------------------------------------------------
import ctypes  # noqa: E402
import functools  # noqa: E402
import warnings  # noqa: E402


_ACT_CODE = {torch.bfloat16: 0, torch.float16: 1, torch.float8_e4m3fn: 2, torch.float8_e5m2: 3, torch.float32: 4}
MAX_EXPERTS = 1024


def _act_code(t: torch.Tensor) -> int:
    if t.dtype not in _ACT_CODE:
        raise RuntimeError("Wrong activation tensor type.")  # grouped_gemm/csrc/permute.cu:686
    return _ACT_CODE[t.dtype]


@functools.lru_cache(maxsize=256)
def _sort_workspace_bytes(tokens: int, topk: int, num_experts: int) -> int:
    need = ctypes.c_int64(0)
    _native.call("tgg_moe_sort_workspace_bytes", tokens, topk, num_experts, ctypes.byref(need))
    return need.value


def _sort_workspace(tokens: int, topk: int, num_experts: int, device):
    """``(tensor to keep until the launch, pointer, bytes)`` of the sort's workspace; small sorts need none."""
    need = _sort_workspace_bytes(tokens, topk, num_experts)
    ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    return ws, _native.ptr(ws), need


def permute_map(indices: torch.Tensor, num_out_tokens: int = 0, num_experts: int = MAX_EXPERTS,
                counts_dtype: torch.dtype = torch.int32):
    """Stable expert-major order of a ``[num_tokens, topK]`` int32 expert assignment.

    Returns ``(row_id_map [topK * num_tokens] int32, tokens_per_expert [num_experts])``: ``row_id_map[k * T + t]``
    is the permuted row of assignment ``(t, k)`` (-1 when dropped: expert id -1, or row >= ``num_out_tokens`` > 0),
    exactly the map the reference builds from a radix sort (grouped_gemm/csrc/permute.cu:40-101, :541-548);
    ``tokens_per_expert`` is what the grouped GEMMs take as ``size_per_group`` (counts before capacity dropping).
    """
    if counts_dtype in (torch.int32, torch.int64):
        result = _native.host().permute_map(indices, num_out_tokens, num_experts, counts_dtype == torch.int64)
        if result is not None:
            return result
    require_gpu(indices)
    if indices.dim() == 1:
        indices = indices.view(-1, 1)
    tokens, topk = indices.shape
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError(f"num_experts must be in [1, {MAX_EXPERTS}], got {num_experts}")
    idx = indices.to(torch.int32).contiguous()
    row_id_map = torch.empty(tokens * topk, dtype=torch.int32, device=idx.device)
    counts = torch.empty(num_experts, dtype=counts_dtype, device=idx.device)
    ws, ws_ptr, ws_bytes = _sort_workspace(tokens, topk, num_experts, idx.device)
    _native.call("tgg_moe_permute_map", idx.data_ptr(), tokens, topk, num_experts, int(num_out_tokens),
                 row_id_map.data_ptr(), counts.data_ptr(), int(counts_dtype == torch.int64), ws_ptr, ws_bytes,
                 _native.stream_of(idx))
    return row_id_map, counts


def _unpermute_raw(inp, row_id_map, probs, num_tokens, topk):
    out = torch.empty((num_tokens, inp.size(1)), dtype=inp.dtype, device=inp.device)
    _native.call("tgg_moe_unpermute", inp.data_ptr(), out.data_ptr(), row_id_map.data_ptr(),
                 probs.data_ptr() if probs is not None else 0, num_tokens, topk, inp.size(1), _act_code(inp),
                 _native.stream_of(inp))
    return out


def _operand(op: str, name: str, t, device, dtype=None, recommended: str = ""):
    """One tensor argument of a permute / unpermute call brought into the form the kernels take: on the activations'
    device, of the index / probability type, contiguous.  Each adjustment is announced with the warning the
    reference's wrappers give for it (grouped_gemm/grouped_gemm/ops.py:60-92, :178-214), so callers see the same
    diagnostics; nothing is done to a tensor that already conforms."""
    if t.is_cpu:
        warnings.warn(f"The input `{name}` of {op} op is on the device: CPU!")
        t = t.to(device)
    if dtype is not None and t.dtype != dtype:
        warnings.warn(f"The data type of the input `{name}` of {op} op is {t.dtype}! The recommended type is {recommended}.")
        t = t.to(dtype)
    if not t.is_contiguous():
        warnings.warn(f"The input `{name}` of {op} op is discontiguous!")
        t = t.contiguous()
    return t


def _activations(op: str, t):
    if t.is_cpu:
        raise RuntimeError(f"[Error] The input `input_act` of {op} op is on the device: CPU!")
    return _operand(op, "input_act", t, t.device)


class PermuteMoE_topK(torch.autograd.Function):
    """grouped_gemm/grouped_gemm/ops.py:52-160.  The workspace the reference keeps between calls is not needed."""

    @staticmethod
    def forward(ctx, input_act, indices, num_out_tokens, max_token_num, num_experts=MAX_EXPERTS):
        if not input_act.numel():
            return input_act, None
        result = _native.host().permute(input_act, indices, num_out_tokens, num_experts)
        if result is not None:
            ctx.set_materialize_grads(False)  # no zero gradient is made for the integer map
            ctx.row_id_map = result[1]
            ctx.num_tokens, ctx.num_topK = indices.shape
            ctx.input_form = input_act.shape, input_act.dtype, input_act.device
            return result
        op = "permute_topK"
        input_act = _activations(op, input_act)
        indices = indices.view(-1, 1) if indices.dim() == 1 else indices
        if input_act.size(0) != indices.size(0):
            raise RuntimeError(f"[Error] {op} op input `indices` shape mismatch! "
                               f"Expect {input_act.size(0)}, but got {indices.size(0)}.")
        indices = _operand(op, "indices", indices, input_act.device, torch.int32, "torch.int32")
        tokens, topk = indices.shape
        if not 1 <= num_experts <= MAX_EXPERTS:
            raise ValueError(f"num_experts must be in [1, {MAX_EXPERTS}], got {num_experts}")
        idx = indices.contiguous()
        row_id_map = torch.empty(tokens * topk, dtype=torch.int32, device=idx.device)
        n_out = num_out_tokens if num_out_tokens > 0 else tokens * topk
        permuted = torch.empty((n_out, input_act.size(1)), dtype=input_act.dtype, device=input_act.device)
        ws, ws_ptr, ws_bytes = _sort_workspace(tokens, topk, num_experts, idx.device)
        _native.call("tgg_moe_permute", input_act.data_ptr(), permuted.data_ptr(), idx.data_ptr(), tokens, topk,
                     num_experts, int(num_out_tokens), input_act.size(1), _act_code(input_act), row_id_map.data_ptr(),
                     0, 0, ws_ptr, ws_bytes, _native.stream_of(input_act))
        ctx.set_materialize_grads(False)  # no zero gradient is made for the integer map
        ctx.row_id_map = row_id_map
        ctx.num_tokens = tokens
        ctx.num_topK = topk
        ctx.input_form = input_act.shape, input_act.dtype, input_act.device
        return permuted, row_id_map

    @staticmethod
    def backward(ctx, permuted_act_grad, _):
        if permuted_act_grad is None:  # nothing downstream gave the rows a gradient
            shape, dtype, device = ctx.input_form
            return torch.zeros(shape, dtype=dtype, device=device), None, None, None, None
        if not permuted_act_grad.numel():
            return permuted_act_grad, None, None, None, None
        grad = permuted_act_grad.contiguous()
        return _unpermute_raw(grad, ctx.row_id_map, None, ctx.num_tokens, ctx.num_topK), None, None, None, None


class UnpermuteMoE_topK(torch.autograd.Function):
    """grouped_gemm/grouped_gemm/ops.py:168-249.  Arithmetic is fp32 with one rounding to the activation type (the
    reference multiplies and accumulates in the activation type)."""

    @staticmethod
    def forward(ctx, input_act, row_id_map, probs=None):
        if not input_act.numel():
            ctx.probs = probs
            return input_act
        op = "unpermute_topK"
        input_act = _activations(op, input_act)
        if probs is not None and row_id_map.size(0) != probs.numel():
            raise RuntimeError(f"[Error] {op} op input `probs` shape mismatch! "
                               f"Expect {row_id_map.size(0)}, but got {probs.size(0) * probs.size(1)}.")
        if probs is None and row_id_map.numel() < input_act.size(0):  # one entry per row is read
            raise RuntimeError(f"[Error] {op} op input `row_id_map` shape mismatch! "
                               f"Expect {input_act.size(0)}, but got {row_id_map.numel()}.")
        row_id_map = _operand(op, "row_id_map", row_id_map, input_act.device, torch.int32, "torch.int32")
        if probs is not None:
            probs = _operand(op, "probs", probs, input_act.device, torch.float32, "torch.float32")
        num_tokens, topk = (probs.size(0), probs.size(1)) if probs is not None else (input_act.size(0), 1)
        out = _unpermute_raw(input_act, row_id_map, probs, num_tokens, topk)
        ctx.save_for_backward(input_act, row_id_map, probs)
        ctx.topk = topk
        return out

    @staticmethod
    def backward(ctx, unpermuted_act_grad):
        if not unpermuted_act_grad.numel():
            return unpermuted_act_grad, None, ctx.probs
        grad = unpermuted_act_grad.contiguous()
        input_act, row_id_map, probs = ctx.saved_tensors
        act_grad = prob_grad = None
        if ctx.needs_input_grad[0] or (probs is not None and ctx.needs_input_grad[2]):
            tokens = grad.size(0)
            # rows no kept assignment maps to (possible only after drops) stay unwritten, as in the reference
            act_grad = torch.empty_like(input_act)
            want_pg = probs is not None and ctx.needs_input_grad[2]
            if want_pg:
                prob_grad = torch.empty_like(probs)
            _native.call("tgg_moe_unpermute_bwd", grad.data_ptr(), input_act.data_ptr(), row_id_map.data_ptr(),
                         probs.data_ptr() if probs is not None else 0, act_grad.data_ptr(),
                         prob_grad.data_ptr() if want_pg else 0, tokens, ctx.topk, grad.size(1), _act_code(grad),
                         _native.stream_of(grad))
            if not ctx.needs_input_grad[0]:
                act_grad = None
        return act_grad, None, prob_grad


def permute(input_act, indices, num_out_tokens=None, max_token_num=0, num_experts=MAX_EXPERTS):
    """grouped_gemm/grouped_gemm/ops.py:251-253; ``num_experts`` (optional, <= 1024) sizes the sort's table."""
    num_out_tokens = 0 if num_out_tokens is None else num_out_tokens
    if not _records(input_act):
        result = _native.host().permute(input_act, indices, num_out_tokens, num_experts)
        if result is not None:
            return result
    return PermuteMoE_topK.apply(input_act, indices, num_out_tokens, max_token_num, num_experts)


def unpermute(input_act, row_id_map, probs=None):
    """grouped_gemm/grouped_gemm/ops.py:255-256."""
    if not _records(input_act, probs):
        out = _native.host().unpermute(input_act, row_id_map, probs)
        if out is not None:
            return out
    return UnpermuteMoE_topK.apply(input_act, row_id_map, probs)


# ---------------------------------------------------------------------------------------------------------------
# Top-k router: what permute / unpermute take
# ---------------------------------------------------------------------------------------------------------------
_SCORING_CODE = {"softmax": 0, "sigmoid": 1}  # TGG_SOFTMAX, TGG_SIGMOID
_LOGIT_CODE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
MAX_TOPK = 64


def _check_router(logits: Tensor, topk: int, scoring: int) -> None:
    if logits.dim() != 2 or logits.dtype not in _LOGIT_CODE:
        raise ValueError(f"logits must be a [tokens, experts] tensor in bf16, fp16 or fp32, got {tuple(logits.shape)} {logits.dtype}")
    experts = logits.shape[1]
    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"the number of experts must be in [1, {MAX_EXPERTS}], got {experts}")
    if not 1 <= topk <= min(MAX_TOPK, experts):
        raise ValueError(f"topk must be in [1, {min(MAX_TOPK, experts)}], got {topk}")
    if scoring not in _SCORING_CODE.values():
        raise ValueError(f"scoring code {scoring} not supported")


def _router_rows(logits: Tensor) -> Tensor:
    """``logits`` as the kernels read them: neighbouring experts in neighbouring places, rows any distance apart."""
    strided = logits.stride(1) != 1 and logits.shape[1] > 1 or logits.stride(0) < logits.shape[1]
    return logits.contiguous() if strided else logits


@torch.library.custom_op("moe::topk_router", mutates_args=())
def _router_forward(logits: Tensor, topk: int, scoring: int, renormalize: bool) -> Tuple[Tensor, Tensor]:
    _check_router(logits, topk, scoring)
    require_gpu(logits)
    logits = _router_rows(logits)
    probs = torch.empty((logits.shape[0], topk), dtype=torch.float32, device=logits.device)
    indices = torch.empty((logits.shape[0], topk), dtype=torch.int32, device=logits.device)
    if logits.shape[0]:
        with torch.cuda.device(logits.device):
            _native.call("tgg_moe_router", logits.data_ptr(), logits.stride(0), logits.shape[0], logits.shape[1], topk, scoring,
                         int(renormalize), _LOGIT_CODE[logits.dtype], probs.data_ptr(), indices.data_ptr(),
                         _native.stream_of(logits))
    return probs, indices


@_router_forward.register_fake
def _(logits, topk, scoring, renormalize):
    return (logits.new_empty((logits.shape[0], topk), dtype=torch.float32),
            logits.new_empty((logits.shape[0], topk), dtype=torch.int32))


@torch.library.custom_op("moe::topk_router_backward", mutates_args=())
def _router_backward(logits: Tensor, probs: Tensor, indices: Tensor, grad: Tensor, scoring: int, renormalize: bool) -> Tensor:
    if probs.dim() != 2 or probs.dtype != torch.float32:
        raise ValueError(f"probs must be the [tokens, topk] fp32 tensor of the forward call, got {tuple(probs.shape)} {probs.dtype}")
    _check_router(logits, probs.shape[1], scoring)
    if probs.shape[0] != logits.shape[0]:
        raise ValueError(f"probs must hold one row per token, got {probs.shape[0]} for {logits.shape[0]}")
    if indices.shape != probs.shape or indices.dtype != torch.int32:
        raise ValueError(f"indices must be the int32 tensor of the forward call, got {tuple(indices.shape)} {indices.dtype}")
    if grad.shape != probs.shape or not grad.dtype.is_floating_point:
        raise ValueError(f"grad must be a floating-point tensor of the shape of probs, got {tuple(grad.shape)} {grad.dtype}")
    if not probs.device == indices.device == grad.device == logits.device:
        raise ValueError("all operands must live on one GPU")
    require_gpu(logits)
    logits = _router_rows(logits)
    out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    if logits.shape[0]:
        probs, indices, grad = probs.contiguous(), indices.contiguous(), grad.float().contiguous()
        with torch.cuda.device(logits.device):
            _native.call("tgg_moe_router_bwd", logits.data_ptr(), logits.stride(0), probs.data_ptr(), indices.data_ptr(),
                         grad.data_ptr(), logits.shape[0], logits.shape[1], probs.shape[1], scoring, int(renormalize),
                         _LOGIT_CODE[logits.dtype], out.data_ptr(), _native.stream_of(logits))
    return out


@_router_backward.register_fake
def _(logits, probs, indices, grad, scoring, renormalize):
    return logits.new_empty(logits.shape)


# (what is registered for them runs in ``topk_router`` too: see EagerOp)
_router_forward.__class__ = _router_backward.__class__ = _native.EagerOp


class TopkRouter(torch.autograd.Function):
    """``topk_router`` with the gradient of the logits; the experts' numbers have none.  (An ordinary eager call is recorded by the
    native call path instead, with the same two launches.)"""

    @staticmethod
    def forward(ctx, logits, topk, scoring, renormalize):
        probs, indices = _router_forward(logits, topk, scoring, renormalize)
        ctx.mark_non_differentiable(indices)
        ctx.save_for_backward(logits, probs, indices)
        ctx.scoring, ctx.renormalize = scoring, renormalize
        return probs, indices

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, _):
        logits, probs, indices = ctx.saved_tensors
        return _router_backward(logits, probs, indices, grad, ctx.scoring, ctx.renormalize), None, None, None


def topk_router(logits, topk, scoring="softmax", renormalize=True):
    """The ``topk`` experts of every token and their probabilities: ``(probs [T, topk] fp32, indices [T, topk] int32)``, in the form
    that ``permute`` (``indices``) and ``unpermute`` (``probs``) take.

    ``logits`` ``[T, E]`` bf16, fp16 or fp32 (E <= 1024, topk <= 64).  Larger logits come first, equal ones by index, NaN above
    all.  ``scoring``: ``"softmax"`` over all experts or ``"sigmoid"``; ``renormalize`` divides the chosen probabilities by their
    sum.  A logit of ``-inf`` masks an expert, which is then never chosen: entries left over have index -1, an assignment that ``permute``
    drops, and probability 0.  Arithmetic is fp32; differentiable in ``logits``."""
    if not (_router_forward.replaced or _router_backward.replaced or torch.compiler.is_compiling()):
        result = (_native._host or _native.host()).topk_router(logits, topk, _SCORING_CODE.get(scoring), renormalize)
        if result is not None:
            return result
    if scoring not in _SCORING_CODE:
        raise ValueError(f"scoring must be one of {sorted(_SCORING_CODE)}, got {scoring!r}")
    topk, code, renormalize = int(topk), _SCORING_CODE[scoring], bool(renormalize)
    _check_router(logits, topk, code)
    require_gpu(logits)
    logits = _router_rows(logits)  # recorded, so that a copy's gradient has the logits' strides
    if not _records(logits):
        return _router_forward(logits, topk, code, renormalize)
    return TopkRouter.apply(logits, topk, code, renormalize)
