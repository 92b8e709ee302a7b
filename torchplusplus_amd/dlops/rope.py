"""Rotary embedding ops (reference: torchpp/dlops/rope.py:6-54).

rope_apply / qkrope_apply keep the reference signatures and return new
tensors; `rope_apply_` is the in-place variant. The kernels accept fp16 and
bf16 inputs with fp16, bf16 or fp32 cos/sin tables, and qkrope_apply allows
fewer K heads than Q heads (GQA). rope_apply_at rotates every token at a
position of its own (drafted trees, far contexts) from frequencies that
rope_frequencies makes, in either pair layout and over part of a head.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from torchplusplus_amd._native import ext as _ext

_C = _ext()


def rope_apply(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """Rotate-half RoPE of x [B, H, S, D] with tables [S, D] (rope.py:6-21)."""
    return _C.rope_apply_cuda(x, cos, sin)


def rope_apply_(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """In-place rope_apply; returns x."""
    return _C.rope_apply_(x, cos, sin)


def qkrope_apply(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor):
    """RoPE of q [B, Hq, S, D] and k [B, Hk, S, D] in one launch (rope.py:24-41)."""
    return _C.qkrope_apply_cuda(q, k, cos, sin)


def compute_rope_params(head_dim, theta_base, context_length, device="cuda",
                        dtype=torch.float32, out_dtype=torch.float16):
    """cos/sin tables [context_length, head_dim] (rope.py:43-54): angles
    pos * theta^(-2j/D) in `dtype`, duplicated over both halves, cast to
    `out_dtype` (fp16 in the reference)."""
    assert head_dim % 2 == 0, "head dim must be divisible by 2"
    j = torch.arange(0, head_dim, 2, device=device, dtype=dtype)
    inv_freq = 1.0 / (theta_base ** (j / head_dim))
    pos = torch.arange(context_length, device=device, dtype=dtype)
    ang = torch.outer(pos, inv_freq)
    ang = torch.cat([ang, ang], dim=1)
    return ang.cos().to(out_dtype).contiguous(), ang.sin().to(out_dtype).contiguous()


def rope_frequencies(rotary_dim: int, theta_base: float = 10000.0, scaling: Optional[str] = None,
                     factor: float = 1.0, original_context: int = 0, beta_fast: float = 32.0,
                     beta_slow: float = 1.0, device="cuda") -> Tuple[torch.Tensor, float]:
    """(inv_freq fp64 [rotary_dim / 2] in radians a position, attention factor)
    for rope_apply_at. Pair j turns by theta^(-2j / rotary_dim) a position;
    `scaling` stretches that by `factor` for contexts longer than the trained:
      "linear"  every frequency divided by factor (position interpolation)
      "ntk"     theta * factor^(R / (R - 2)): the slowest pair is divided by
                factor, the fastest kept
      "yarn"    pairs that turn more than beta_fast times over original_context
                kept, those that turn less than beta_slow times divided by
                factor, a linear ramp over j between; attention factor
                0.1 ln(factor) + 1
    In fp64: an fp32 frequency is off by 0.06 rad at position 10^6."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"unknown scaling: {scaling}")
    if factor < 1.0:
        raise ValueError(f"factor must be at least 1, got {factor}")
    if scaling == "ntk":
        if rotary_dim < 4:
            raise ValueError("ntk scaling needs a rotary_dim of 4 at least")
        theta_base = theta_base * factor ** (rotary_dim / (rotary_dim - 2))
    j = torch.arange(rotary_dim // 2, dtype=torch.float64)
    freq = float(theta_base) ** (-2.0 * j / rotary_dim)
    attention_factor = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        if original_context < 1:
            raise ValueError("yarn scaling needs original_context, the trained context length")

        def pair(turns):  # the pair that turns so often over the trained context
            return (rotary_dim * math.log(original_context / (turns * 2 * math.pi))
                    / (2 * math.log(theta_base)))

        low = max(math.floor(pair(beta_fast)), 0)
        high = min(math.ceil(pair(beta_slow)), rotary_dim - 1)
        keep = 1.0 - ((j - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
        freq = freq / factor * (1.0 - keep) + freq * keep
        attention_factor = 0.1 * math.log(factor) + 1.0
    return freq.to(device), attention_factor


def rope_apply_at(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor,
                  inv_freq: torch.Tensor, interleaved: bool = False,
                  attention_factor: float = 1.0):
    """Rotary embedding of q [B, S, Hq, D] and k [B, S, Hk, D] (or None) at
    positions [B, S] or [S] (int32 or int64), in one launch; new contiguous
    tensors. The first 2 * len(inv_freq) elements of a head turn, in pairs
    (j, j + R/2) or, interleaved, (2j, 2j + 1); the rest, and tokens at negative
    positions (padding), are copied. inv_freq as from rope_frequencies. q and k
    may be views of a fused projection (any strides, contiguous last dim)."""
    return _C.rope_at(q, k, positions, inv_freq, interleaved, attention_factor, False)


def rope_apply_at_(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor,
                   inv_freq: torch.Tensor, interleaved: bool = False,
                   attention_factor: float = 1.0):
    """rope_apply_at in place; returns (q, k)."""
    return _C.rope_at(q, k, positions, inv_freq, interleaved, attention_factor, True)
