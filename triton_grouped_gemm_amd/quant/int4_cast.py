"""Weights in 4 bits for ``m_grouped_gemm_int4``: made once, when a model is loaded.

``per_group_cast_to_int4`` quantises 16- or 32-bit weights, ``pack_int4`` lays out 4-bit values that come from elsewhere and
``unpack_int4`` undoes it.  Everything is integer and elementwise torch arithmetic on whatever device the weights are on, one
expert at a time.
"""
from typing import Optional, Tuple

import torch

_NIBBLE_TO_VALUE = (0, 2, 4, 6, 1, 3, 5, 7)  # which of a word's eight values each nibble holds


def pack_int4(values: torch.Tensor) -> torch.Tensor:
    """``[G, N, K]`` integers 0..15 -> uint8 ``[G, ceil(N/16), ceil(K/128), 64, 16]``, the layout the kernel reads: blocks of 16 columns
    x 128 values, in which entry ``16 lg + c`` is column c and its byte ``4 s + m`` holds values ``32 s + 8 lg + e`` of the
    block, e in the order 0 2 4 6 1 3 5 7 from the low nibble of byte 0 on.  Beyond N and K there are zeros."""
    if values.dim() != 3 or values.dtype.is_floating_point or values.dtype == torch.bool:
        raise ValueError(f"values must be a [G, N, K] integer tensor, got {tuple(values.shape)} {values.dtype}")
    G, N, K = values.shape
    if not (G and N and K):
        raise ValueError(f"values must not be empty, got {tuple(values.shape)}")
    nb, kb = -(-N // 16), -(-K // 128)
    out = torch.empty((G, nb, kb, 64, 16), dtype=torch.uint8, device=values.device)
    for g in range(G):
        v = values[g]
        if int(v.min()) < 0 or int(v.max()) > 15:
            raise ValueError("values must lie in 0..15")
        q = torch.zeros((nb * 16, kb * 128), dtype=torch.uint8, device=values.device)
        q[:N, :K] = v
        q = q.view(nb, 16, kb, 4, 4, 8)[..., list(_NIBBLE_TO_VALUE)]  # block, column, block, step s, chunk lg, nibble
        both = q[..., 0::2] | (q[..., 1::2] << 4)
        out[g] = both.permute(0, 2, 4, 1, 3, 5).reshape(nb, kb, 64, 16)
    return out


def unpack_int4(codes: torch.Tensor, N: int, K: int) -> torch.Tensor:
    """What ``pack_int4`` was given: uint8 ``[G, N, K]``."""
    if codes.dim() != 5 or codes.dtype != torch.uint8 or codes.shape[1:] != (-(-N // 16), -(-K // 128), 64, 16):
        raise ValueError(f"codes of {tuple(codes.shape)} {codes.dtype} are not those of {N} x {K} values")
    G, nb, kb = codes.shape[:3]
    c = codes.view(G, nb, kb, 4, 16, 4, 4)
    q = torch.empty((G, nb, kb, 4, 16, 4, 8), dtype=torch.uint8, device=codes.device)
    for nibble, value in enumerate(_NIBBLE_TO_VALUE):
        q[..., value] = (c[..., nibble // 2] >> (4 * (nibble % 2))) & 15
    return q.permute(0, 1, 4, 2, 5, 3, 6).reshape(G, nb * 16, kb * 128)[:, :N, :K].contiguous()


@torch.no_grad()
def per_group_cast_to_int4(w: torch.Tensor, group_size: int = 128, zeros: bool = False,
                           ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """``w`` ``[G, N, K]`` -> ``(codes, scales [G, ceil(K/group_size), N], zeros or None)`` for ``m_grouped_gemm_int4``, scales in the
    weights' type (bf16 or fp16; fp32 weights give bf16 scales).  No gradient is recorded, whether the weights are trained or not.

    Without zero points a group's values are ``(q - 8) s`` with s the largest magnitude over 7; with them the group's range, extended
    to hold 0, is divided into 15 steps.  Codes are rounded to nearest against the rounded scale, so that a value is off by at most half
    a step, except that what lies beyond the last code is cut off."""
    if w.dim() != 3 or w.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError(f"w must be a [G, N, K] tensor in bf16, fp16 or fp32, got {tuple(w.shape)} {w.dtype}")
    if group_size not in (32, 64) and (group_size < 128 or group_size % 128):
        raise ValueError(f"group_size must be 32, 64 or a multiple of 128, got {group_size}")
    G, N, K = w.shape
    if not (G and N and K):
        raise ValueError(f"w must not be empty, got {tuple(w.shape)}")
    dtype = torch.bfloat16 if w.dtype == torch.float32 else w.dtype
    groups = -(-K // group_size)
    codes = torch.empty((G, -(-N // 16), -(-K // 128), 64, 16), dtype=torch.uint8, device=w.device)
    scales = torch.empty((G, groups, N), dtype=dtype, device=w.device)
    points = torch.empty((G, groups, N), dtype=torch.uint8, device=w.device) if zeros else None
    for g in range(G):
        v = torch.zeros((N, groups * group_size), dtype=torch.float32, device=w.device)
        v[:, :K] = w[g]
        v = v.view(N, groups, group_size)
        if zeros:
            low, high = v.amin(-1).clamp_max(0), v.amax(-1).clamp_min(0)
            step = (high - low) / 15
        else:
            step = v.abs().amax(-1) / 7
        scale = step.to(dtype)
        scale = torch.where(scale == 0, torch.ones_like(scale), scale)
        s = scale.float()
        zero = torch.round(-low / s).clamp(0, 15) if zeros else torch.full_like(s, 8)
        q = (torch.round(v / s[..., None]) + zero[..., None]).clamp(0, 15).to(torch.uint8)
        codes[g] = pack_int4(q.view(1, N, -1)[:, :, :K])[0]
        scales[g] = scale.t()
        if zeros:
            points[g] = zero.t().to(torch.uint8)
    return codes, scales, points
