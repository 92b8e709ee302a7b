"""Attention of drafted tokens over a KV cache (no counterpart in the
reference, which decodes one token at a time, torchpp/attention/gqa.py:117-128).
"""
from __future__ import annotations

from typing import Optional

import torch

from torchplusplus_amd._native import ext as _ext

_C = _ext()

TREE_MAX_TOKENS = 64  # drafted tokens a sequence: a bit each in the kernels' masks


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   seqlens: torch.Tensor, parents: Optional[torch.Tensor] = None,
                   k_exps: Optional[torch.Tensor] = None, v_exps: Optional[torch.Tensor] = None,
                   softmax_scale: Optional[float] = None, out: Optional[torch.Tensor] = None
                   ) -> torch.Tensor:
    """q [B, T, Hq, D], T drafted tokens (1 to 64) of each sequence, whose keys
    and values are in the caches [B, Hkv, L, D] at positions seqlens[b] ..
    seqlens[b] + T - 1, behind the context's seqlens[b] (int32 [B]). Token t sees
    the context, itself and its ancestors by `parents` (int32 [B, T]: an earlier
    token, or -1 for the context; any other value is padding and sees nothing,
    nor do its children; None: a chain). Rows that see nothing are 0, as are
    those of tokens past the cache's end; a row whose scores are all -inf is NaN.

    Caches of q's dtype, or of float8_e4m3fn / int8 codes with the exponent
    bytes k_exps, v_exps of a QuantKVCache. T = 1 is a decode step over either.
    softmax_scale is above 0, by default 1/sqrt(D). Returns o [B, T, Hq, D]."""
    if softmax_scale is not None and not 2.0 ** -126 <= softmax_scale < 2.0 ** 126:  # fp32's normal range
        raise ValueError(f"softmax_scale must be above 0 and finite, got {softmax_scale}")
    return _C.tree_attention(q, k_cache, v_cache, seqlens, parents, k_exps, v_exps,
                             0.0 if softmax_scale is None else float(softmax_scale), out)
