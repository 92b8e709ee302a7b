"""KV cache (reference: torchpp/llmops/kvcache.py:6-116).

Same constructor and update/reset API, with the reference's defects fixed:
  * the cache is [B, n_kv_heads, max_seq_len, head_dim] for any batch B
    (batch was hard-coded to 1 at kvcache.py:40,45);
  * it is allocated once at full length on first use (kvcache.py:66 allocated
    a single position);
  * update() returns the prefix [:cache_len] as views, not one position
    (kvcache.py:79-80) and not `.contiguous()` copies (kvcache.py:106-107);
  * writing past max_seq_len raises instead of corrupting memory.
The attention kernels read and write this layout in place: K/V rows of
sequence b, head h are contiguous along positions.

QuantKVCache holds 8-bit codes instead (no counterpart in the reference, whose
cache is fp16).
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from torchplusplus_amd._native import ext as _ext

_C = _ext()


def _keep(rows: torch.Tensor, start: torch.Tensor, path: torch.Tensor) -> None:
    """rows [B, H, L, ...]: row start[b] + path[b, i] to row start[b] + i for
    each path[b, i] >= 0; other rows keep what they hold. Gathered whole before
    anything is written, each row written once (entries of -1, and those past
    the cache's end, write a row of their own back to itself)."""
    if path.dim() != 2 or path.shape[0] != rows.shape[0] or start.shape != path.shape[:1]:
        raise ValueError(f"start {tuple(start.shape)} and path {tuple(path.shape)} must be [B] and [B, n], "
                         f"for at most the cache's sequences")
    n, length = path.shape[1], rows.shape[2]
    if n > length:
        raise ValueError(f"a path of {n} tokens in a cache of {length} positions")
    first = start.view(-1, 1).long()
    to = first + torch.arange(n, device=path.device)
    src = first + path.long()
    moves = (path >= 0) & (first >= 0) & (to < length) & (src < length)
    to = to % length
    src = torch.where(moves, src, to)
    seq = torch.arange(path.shape[0], device=path.device).view(-1, 1)
    raw = rows.view(torch.uint8) if rows.element_size() == 1 else rows
    raw[seq, :, to] = raw[seq, :, src]


QUANT_CODES = (torch.float8_e4m3fn, torch.int8)  # element types of a cache of 8-bit codes


def kv_quant_append(k: torch.Tensor, v: torch.Tensor, k_codes: torch.Tensor, v_codes: torch.Tensor,
                    k_exps: torch.Tensor, v_exps: torch.Tensor,
                    positions: Union[int, torch.Tensor], counts: Optional[torch.Tensor] = None) -> None:
    """Write k, v [B, S, Hkv, D] (fp16 or bf16, any strides that keep rows
    16-byte aligned) into caches of codes [B, Hkv, L, D] (float8_e4m3fn or int8)
    and exponent bytes [B, Hkv, L] (uint8): a row is codes * 2^(byte - 127), the
    least power of two that holds it, codes rounded to nearest (ties to even); a
    value past the largest below 2^128 that codes hold counts as that.
    Token s of sequence b goes to positions[b] + s (an int: the same for all);
    tokens outside the cache, or past counts[b], are not written. A row with an
    infinity or NaN is kept as NaN. D in {64, 128, 256}."""
    if isinstance(positions, torch.Tensor):
        _C.kv_quant_append(k, v, k_codes, v_codes, k_exps, v_exps, positions, 0, counts)
    else:
        _C.kv_quant_append(k, v, k_codes, v_codes, k_exps, v_exps, None, positions, counts)


def kv_quant_read(k_codes: torch.Tensor, v_codes: torch.Tensor, k_exps: torch.Tensor,
                  v_exps: torch.Tensor, length: int, dtype: torch.dtype = torch.bfloat16
                  ) -> Tuple[torch.Tensor, torch.Tensor]:
    """The first `length` rows of such caches as values: two new tensors
    [B, Hkv, length, D] of `dtype` (exact in bfloat16; one rounding, limited to
    +-65504, in float16)."""
    return _C.kv_quant_read(k_codes, v_codes, k_exps, v_exps, length, dtype)


class KVCache:
    def __init__(self, max_seq_len: int, n_kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.float16, device=torch.device("cuda"),
                 batch_size: Optional[int] = None):
        self.max_seq_len = max_seq_len
        self.n_kv_heads = n_kv_heads
        self.head_dim = head_dim
        self.dtype = dtype
        self.device = device
        self.k_cache: Optional[torch.Tensor] = None
        self.v_cache: Optional[torch.Tensor] = None
        self.cache_len = 0
        if batch_size is not None:
            self.ensure(batch_size, 0)

    @property
    def batch_size(self) -> int:
        return 0 if self.k_cache is None else self.k_cache.shape[0]

    def ensure(self, batch_size: int, length: int) -> None:
        """Allocate (once) for `batch_size` sequences; check `length` fits."""
        if length > self.max_seq_len:
            raise ValueError(f"KV cache overflow: {length} > max_seq_len {self.max_seq_len}")
        if self.k_cache is None or self.k_cache.shape[0] < batch_size:
            shape = (batch_size, self.n_kv_heads, self.max_seq_len, self.head_dim)
            self.k_cache = torch.zeros(shape, dtype=self.dtype, device=self.device)
            self.v_cache = torch.zeros(shape, dtype=self.dtype, device=self.device)
            self.cache_len = 0

    def update(self, k: torch.Tensor, v: torch.Tensor, index: Optional[int] = None
               ) -> Tuple[torch.Tensor, torch.Tensor]:
        """Write k, v [B, n_kv_heads, S, head_dim] at cache_len (index None) or
        at `index`, and return the cached prefix [B, n_kv_heads, cache_len, D]."""
        bsz, _, seq_len, _ = k.shape
        start = self.cache_len if index is None else int(index)
        end = start + seq_len
        self.ensure(bsz, end)
        self.k_cache[:bsz, :, start:end] = k
        self.v_cache[:bsz, :, start:end] = v
        self.cache_len = max(self.cache_len, end) if index is not None else end
        return self.k_cache[:bsz, :, : self.cache_len], self.v_cache[:bsz, :, : self.cache_len]

    def keep(self, start: torch.Tensor, path: torch.Tensor) -> None:
        """After a verification: the rows of the accepted drafted tokens, at
        start[b] + path[b, i] (entries of -1 are none), move to start[b] + i.
        start [B] (where the first drafted token's row is), path [B, n]; cache_len
        is the caller's to advance."""
        for rows in (self.k_cache, self.v_cache):
            _keep(rows[: path.shape[0]], start, path)

    def reset(self) -> None:
        self.cache_len = 0
        if self.k_cache is not None:
            self.k_cache.zero_()
            self.v_cache.zero_()


class QuantKVCache:
    """KVCache whose rows are 8-bit codes with an exponent byte each (see
    kv_quant_append): half the memory, and half the bytes a decode step reads.
    `dtype` is the type of the values that go in and come back, `code_dtype`
    torch.float8_e4m3fn (3 bits after the first of each element) or torch.int8
    (7 bits after the first of the row's largest element).

    head_dim 64 or 128; 256 too, but no attention kernel is fast there (one for any size
    reads a key at a time, over codes as over 16-bit values).

    append() writes tokens, attention.tree_attention reads the codes in place
    (GroupedQueryAttention does both), read() decodes a prefix, update() is
    KVCache.update: append, then the decoded prefix."""

    def __init__(self, max_seq_len: int, n_kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.float16, device=torch.device("cuda"),
                 batch_size: Optional[int] = None, code_dtype: torch.dtype = torch.float8_e4m3fn):
        if code_dtype not in QUANT_CODES:
            raise TypeError(f"code_dtype must be float8_e4m3fn or int8, got {code_dtype}")
        if dtype not in (torch.float16, torch.bfloat16):
            raise TypeError(f"dtype must be float16 or bfloat16, got {dtype}")
        if head_dim not in (64, 128, 256):
            raise ValueError(f"head_dim must be 64, 128 or 256, got {head_dim}")
        self.max_seq_len = max_seq_len
        self.n_kv_heads = n_kv_heads
        self.head_dim = head_dim
        self.dtype = dtype
        self.code_dtype = code_dtype
        self.device = device
        self.k_codes: Optional[torch.Tensor] = None
        self.v_codes: Optional[torch.Tensor] = None
        self.k_exps: Optional[torch.Tensor] = None
        self.v_exps: Optional[torch.Tensor] = None
        self.cache_len = 0
        if batch_size is not None:
            self.ensure(batch_size, 0)

    @property
    def batch_size(self) -> int:
        return 0 if self.k_codes is None else self.k_codes.shape[0]

    def ensure(self, batch_size: int, length: int) -> None:
        """Allocate (once) for `batch_size` sequences; check `length` fits."""
        if length > self.max_seq_len:
            raise ValueError(f"KV cache overflow: {length} > max_seq_len {self.max_seq_len}")
        if self.k_codes is None or self.k_codes.shape[0] < batch_size:
            # whole groups of 16 exponent bytes: the attention reads them so
            room = -(-self.max_seq_len // 16) * 16
            shape = (batch_size, self.n_kv_heads, room, self.head_dim)
            kw = dict(device=self.device)
            self.k_codes = torch.zeros(shape, dtype=torch.int8, **kw).view(self.code_dtype)
            self.v_codes = torch.zeros(shape, dtype=torch.int8, **kw).view(self.code_dtype)
            self.k_exps = torch.full(shape[:3], 127, dtype=torch.uint8, **kw)
            self.v_exps = torch.full(shape[:3], 127, dtype=torch.uint8, **kw)
            self.cache_len = 0

    def rows(self, bsz: int):
        """(k_codes, v_codes, k_exps, v_exps) of the first `bsz` sequences."""
        return self.k_codes[:bsz], self.v_codes[:bsz], self.k_exps[:bsz], self.v_exps[:bsz]

    def append(self, k: torch.Tensor, v: torch.Tensor, positions: Union[int, torch.Tensor],
               counts: Optional[torch.Tensor] = None) -> None:
        """Write k, v [B, S, n_kv_heads, D] from positions[b] on (an int: the
        same for every sequence, and cache_len grows to cover it; a device
        tensor leaves cache_len to the caller). See kv_quant_append."""
        bsz, seq_len = k.shape[0], k.shape[1]
        if isinstance(positions, torch.Tensor):
            self.ensure(bsz, 0)
        else:
            if positions < 0:
                raise ValueError(f"position {positions} is below 0")
            self.ensure(bsz, int(positions) + seq_len)
        kv_quant_append(k, v, *self.rows(bsz), positions, counts)
        if not isinstance(positions, torch.Tensor):
            self.cache_len = max(self.cache_len, int(positions) + seq_len)

    def read(self, length: Optional[int] = None, batch_size: Optional[int] = None
             ) -> Tuple[torch.Tensor, torch.Tensor]:
        """The first `length` (default cache_len) positions of the first
        `batch_size` sequences as values [B, n_kv_heads, length, D]."""
        bsz = self.batch_size if batch_size is None else batch_size
        return kv_quant_read(*self.rows(bsz), self.cache_len if length is None else length, self.dtype)

    def update(self, k: torch.Tensor, v: torch.Tensor, index: Optional[int] = None
               ) -> Tuple[torch.Tensor, torch.Tensor]:
        """KVCache.update: write k, v [B, n_kv_heads, S, D] at cache_len (index
        None) or at `index`; returns the decoded prefix."""
        bsz, _, seq_len, _ = k.shape
        start = self.cache_len if index is None else int(index)
        before = self.cache_len
        self.append(k.transpose(1, 2), v.transpose(1, 2), start)
        self.cache_len = max(before, start + seq_len) if index is not None else start + seq_len
        return self.read(batch_size=bsz)

    def keep(self, start: torch.Tensor, path: torch.Tensor) -> None:
        """KVCache.keep on codes and exponents."""
        for rows in self.rows(path.shape[0]):
            _keep(rows, start, path)

    def reset(self) -> None:
        self.cache_len = 0
        if self.k_codes is not None:
            for c in (self.k_codes, self.v_codes):
                c.view(torch.uint8).zero_()
            for e in (self.k_exps, self.v_exps):
                e.fill_(127)
