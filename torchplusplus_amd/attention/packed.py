"""Attention of a batch of sequences of different lengths: whole prompts packed
one behind the other, and one new token of each over a cache held in pages (no
counterpart in the reference, whose batches are rectangular and whose caches are
one tensor a sequence, torchpp/attention/gqa.py:117-128)."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from torchplusplus_amd._native import ext as _ext

_C = _ext()


def _scale(softmax_scale: Optional[float]) -> float:
    if softmax_scale is None:
        return 0.0
    if not 2.0 ** -126 <= softmax_scale < 2.0 ** 126:  # fp32's normal range
        raise ValueError(f"softmax_scale must be above 0 and finite, got {softmax_scale}")
    return float(softmax_scale)


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                     cu_seqlens_k: Optional[torch.Tensor] = None, softmax_scale: Optional[float] = None,
                     causal: bool = True, window_size: Tuple[int, int] = (-1, -1),
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """flash_attn_func for sequences packed one behind the other: q [Nq, Hq, D],
    k and v [Nk, Hkv, D] (fp16 or bf16; last dim contiguous, other strides free).
    Sequence b has rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1 of q and, by
    cu_seqlens_k (default cu_seqlens, Nk = Nq), of k and v: int32 [B + 1] on the
    device, ascending. They are not read on the host: an end past the tensors is
    cut to them. Lengths of 0 are allowed.

    causal and window_size=(left, right), -1 unbounded, are aligned bottom-right in
    each sequence. A row that sees nothing is 0; one whose scores are all -inf is
    NaN. Rows of no sequence (behind the last one, in a padded batch) stay as they
    were in a given `out`, and are 0 in a new one. softmax_scale is above 0, by
    default 1/sqrt(D). head_dim 64 and 128 with 16-byte rows run on the matrix
    cores, with weights rounded to the type of v (fp16: those below 2^-32 of the
    row's largest may count as 0); others up to 256 on a slow kernel, a wave a row.
    Returns o [Nq, Hq, D]."""
    left, right = window_size
    return _C.packed_attention(q, k, v, cu_seqlens, cu_seqlens_k, _scale(softmax_scale), bool(causal), int(left),
                               int(right), out)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_tables: torch.Tensor,
                    seqlens: torch.Tensor, softmax_scale: Optional[float] = None, window_left: int = -1,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """decode_attention over a cache held in pages: one query per sequence, q [B,
    Hq, D], against the first seqlens[b] positions (int32 [B]) of the sequence,
    position j in row j % page_size of page block_tables[b, j // page_size] (int32
    [B, M]) of k_pages, v_pages [pages, Hkv, page_size, D] (page_size a power of
    two, 16 to 1024). window_left >= 0 keeps positions >= seqlens[b] - 1 -
    window_left.

    Lengths are limited to the table's positions; the positions of a table entry
    that is no page (outside [0, pages), e.g. -1 for one given back) are not seen.
    A row that sees nothing is 0; one whose scores are all -inf is NaN.
    softmax_scale is above 0, by default 1/sqrt(D). head_dim 64 and 128 with
    16-byte rows run on the matrix cores, others up to 256 on a slow kernel.
    Returns o [B, Hq, D]."""
    return _C.paged_attention(q, k_pages, v_pages, block_tables, seqlens, _scale(softmax_scale), int(window_left), out)
