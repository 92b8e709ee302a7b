"""Log probabilities of tokens under a model's logits (no counterpart in the
reference, whose samplers, torchpp/llmops/llm.py:114-186, keep none)."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from torchplusplus_amd._native import ext as _ext

_C = _ext()


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor                # fp32 [...]
    entropy: torch.Tensor                 # fp32 [...], in nats
    top_logprobs: Optional[torch.Tensor]  # fp32 [..., top_k], falling
    top_tokens: Optional[torch.Tensor]    # int64 [..., top_k]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top_k: int = 0) -> TokenLogprobs:
    """Log probabilities of `tokens` [...] (int64) under `logits` [..., V] (fp32,
    fp16 or bf16), the entropy of each row and, for top_k > 0 (at most 32), the top_k
    most probable tokens, the lowest index first among equal logits.

    In one pass over the logits, sums in fp32. A token outside [0, V) is padding: its
    log probability is 0. Logits of -inf have no share. A row with a NaN or +inf, or
    of -inf alone, gives NaN (top_tokens -1 with a NaN or +inf)."""
    if tokens.shape != logits.shape[:-1]:
        raise ValueError(f"tokens {tuple(tokens.shape)} do not fit logits {tuple(logits.shape)}")
    rows = logits.reshape(-1, logits.shape[-1]) if logits.dim() != 2 else logits
    lp, ent, top, ids = _C.token_logprobs(rows, tokens.reshape(-1), int(top_k))
    if logits.dim() == 2:
        return TokenLogprobs(lp, ent, top, ids)
    shape = tokens.shape
    return TokenLogprobs(lp.view(shape), ent.view(shape), None if top is None else top.view(*shape, top_k),
                         None if ids is None else ids.view(*shape, top_k))
