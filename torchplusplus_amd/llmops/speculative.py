"""Verification of drafted tokens (no counterpart in the reference, whose
samplers, torchpp/llmops/llm.py:114-186, draw one token at a time)."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from torchplusplus_amd._native import ext as _ext

_C = _ext()


def verify_draft(draft_tokens: torch.Tensor, target_probs: torch.Tensor, uniforms: torch.Tensor,
                 draft_probs: Optional[torch.Tensor] = None, parents: Optional[torch.Tensor] = None
                 ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Which of the drafted tokens [B, T] (int64, T at most 64; outside [0, V):
    padding) stay, so that the sequence is one drawn from the target's
    probabilities [B, T + 1, V] (fp32, fp16 or bf16; row 0 follows the context,
    row t + 1 drafted token t), from uniform numbers [B, T + 1] (fp32, in
    [0, 1)).

    With draft_probs [B, T, V] the tokens are a chain drawn from them: token i
    stays while u_i q_i < p_i, and the next token is drawn from max(p - q, 0) at
    the first that does not (from p behind the last, or at padding). Without,
    they were chosen without a draw and form a chain or, with parents (int32
    [B, T] as in tree_attention), a tree: at each node the child c stays for
    which u_depth falls into its share of p, and where none does the next token
    is drawn from p without the children. Draws are by inverse CDF with the last
    uniform number, sums in fp64.

    Returns accepted [B] int32, path [B, T] int32 (the accepted tokens' indices,
    then -1) and next_token [B] int64 (-1 where the target's row has no mass)."""
    return _C.verify_draft(draft_tokens, target_probs, uniforms, draft_probs, parents)
