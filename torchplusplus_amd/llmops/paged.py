"""A KV cache held in pages, for batches of sequences of different lengths (no
counterpart in the reference, whose cache is one tensor of max_seq_len positions a
sequence, torchpp/llmops/kvcache.py:39-48)."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence, Tuple

import torch

from torchplusplus_amd._native import ext as _ext

_C = _ext()

PAGE_SIZES = tuple(2 ** i for i in range(4, 11))  # rows of a page


def qkv_rope_paged(qkv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor, k_pages: torch.Tensor,
                   v_pages: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                   q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None,
                   eps: float = 1e-6, with_k: bool = True) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """From a packed batch's fused projection qkv [N, (Hq + 2 Hkv) * D] (not
    changed): per-head RMSNorm of q and k (weights [D], None: no norm), RoPE by row
    positions[t] (int32 [N]) of the tables cos, sin [ctx, D], one rounding. The
    rotated keys and the values of token t are written into row slots[t] %
    page_size of page slots[t] // page_size (int64 [N]) of k_pages, v_pages [pages,
    Hkv, page_size, D].

    Slots are distinct (of two equal ones either token's row may stay); one outside
    the pages (e.g. -1) is not written. A token at a position outside [0, ctx) is
    padding: its q and k are 0, no slot is written. D in {64, 128, 256}, rows
    16-byte aligned. Returns q [N, Hq, D] and the rotated k [N, Hkv, D] (None if not
    with_k: a decode step reads them from the pages)."""
    return _C.qkv_rope_paged(qkv, positions, slots, k_pages, v_pages, cos, sin, q_norm, k_norm, eps, with_k)


@dataclass
class PagedStep:
    """What a packed batch's tokens are to a PagedKVCache, the same for every layer.
    A decode step has one token a sequence and their block_tables and seqlens (the new
    token counted in). A prefill step has cu_seqlens, and, where tokens follow cached
    ones, the slots that hold each sequence's positions from 0 on (key_slots) and their
    cu_seqlens_k."""

    positions: torch.Tensor
    slots: torch.Tensor
    cu_seqlens: Optional[torch.Tensor] = None
    cu_seqlens_k: Optional[torch.Tensor] = None
    key_slots: Optional[torch.Tensor] = None
    block_tables: Optional[torch.Tensor] = None
    seqlens: Optional[torch.Tensor] = None


class PagedKVCache:
    """Keys and values of `n_layers` layers in pages of `page_size` rows, dealt to
    sequences as they grow; one table of pages serves every layer. k_pages[i],
    v_pages[i] are layer i's [num_pages, n_kv_heads, page_size, head_dim].

    allocate() begins a sequence, grow() deals it pages, free() takes them back;
    prefill_step() and decode_step() give what a model's layers ask for, of
    block_tables(), slots() and next_slots(). The table is kept on the host; page
    contents are not cleared."""

    def __init__(self, num_pages: int, page_size: int, n_layers: int, n_kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.float16, device=torch.device("cuda")):
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page_size}")
        if num_pages < 1 or n_layers < 1:
            raise ValueError("at least one page and one layer are needed")
        self.num_pages, self.page_size = num_pages, page_size
        self.n_layers, self.n_kv_heads, self.head_dim = n_layers, n_kv_heads, head_dim
        self.dtype, self.device = dtype, device
        shape = (n_layers, num_pages, n_kv_heads, page_size, head_dim)
        self.k_pages = torch.zeros(shape, dtype=dtype, device=device)
        self.v_pages = torch.zeros(shape, dtype=dtype, device=device)
        self._unused: List[int] = list(range(num_pages - 1, -1, -1))
        self._tables: Dict[int, List[int]] = {}
        self._next = 0

    @property
    def free_pages(self) -> int:
        return len(self._unused)

    def pages_of(self, seq: int) -> List[int]:
        return list(self._tables[seq])

    def allocate(self, length: int = 0) -> int:
        """A new sequence with pages for `length` positions; its handle."""
        seq = self._next
        self._tables[seq] = []
        try:
            self.grow(seq, length)
        except (ValueError, RuntimeError):
            del self._tables[seq]
            raise
        self._next += 1
        return seq

    def grow(self, seq: int, length: int) -> None:
        """Pages for `length` positions (RuntimeError, and nothing dealt, where there
        are not enough)."""
        if length < 0:
            raise ValueError(f"length {length} is below 0")
        table = self._tables[seq]
        need = -(-length // self.page_size) - len(table)
        if need > len(self._unused):
            raise RuntimeError(f"out of pages: {need} needed, {len(self._unused)} of {self.num_pages} unused")
        for _ in range(need):
            table.append(self._unused.pop())

    def free(self, seq: int) -> None:
        self._unused.extend(reversed(self._tables.pop(seq)))

    def block_tables(self, seqs: Sequence[int], width: Optional[int] = None) -> torch.Tensor:
        """int32 [len(seqs), width] on the device (default: the longest table's), -1
        past a sequence's pages."""
        rows = [self._tables[s] for s in seqs]
        most = max([len(r) for r in rows], default=0)
        if width is not None and width < most:
            raise ValueError(f"a table of {most} pages does not fit {width}")
        width = most if width is None else width
        flat = [r + [-1] * (width - len(r)) for r in rows]
        return torch.tensor(flat, dtype=torch.int32).view(len(rows), width).to(self.device)

    @staticmethod
    def _check(seqs, starts, counts) -> None:
        if not len(seqs) == len(starts) == len(counts):
            raise ValueError(f"{len(seqs)} sequences need one start and one count each, got {len(starts)} and {len(counts)}")
        if min([*starts, *counts], default=0) < 0:
            raise ValueError(f"starts {list(starts)} and counts {list(counts)} must not be below 0")

    def slots(self, seqs: Sequence[int], starts: Sequence[int], counts: Sequence[int]
              ) -> Tuple[torch.Tensor, torch.Tensor]:
        """Positions starts[i] .. starts[i] + counts[i] - 1 of every sequence in turn, and
        their slots: int32 and int64 [sum of counts] on the device."""
        self._check(seqs, starts, counts)
        pos, slots = [], []
        for s, a, n in zip(seqs, starts, counts):
            table = torch.tensor(self._tables[s], dtype=torch.int64)
            if a + n > len(table) * self.page_size:
                raise ValueError(f"positions {a} to {a + n} of a sequence with pages for {len(table) * self.page_size}")
            p = torch.arange(a, a + n)
            pos.append(p)
            slots.append(table[p // self.page_size] * self.page_size + p % self.page_size)
        cat = lambda x: torch.cat(x) if x else torch.empty(0, dtype=torch.int64)  # noqa: E731
        return cat(pos).int().to(self.device), cat(slots).to(self.device)

    def next_slots(self, block_tables: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        """The slot of position positions[b] of every sequence of a table: int64 [B],
        -1 where the sequence has no page for it. On the device alone (for a decode
        step, captured or not)."""
        if positions.shape != block_tables.shape[:1]:
            raise ValueError(f"a table of {block_tables.shape[0]} sequences needs one position each, got {tuple(positions.shape)}")
        if block_tables.shape[1] == 0:  # (nothing to gather from)
            return torch.full_like(positions, -1, dtype=torch.int64)
        p = positions.long()
        entry = torch.div(p, self.page_size, rounding_mode="floor").unsqueeze(1)
        inside = (entry >= 0) & (entry < block_tables.shape[1])
        page = block_tables.long().gather(1, torch.where(inside, entry, 0))
        slot = page * self.page_size + (p % self.page_size).unsqueeze(1)
        return torch.where(inside & (page >= 0), slot, -1).squeeze(1)

    def prefill_step(self, seqs: Sequence[int], starts: Sequence[int], counts: Sequence[int]) -> PagedStep:
        """counts[i] new tokens of each sequence behind its first starts[i], packed in
        turn (RuntimeError, and nothing dealt, where there are not enough pages)."""
        self._check(seqs, starts, counts)
        if len(set(seqs)) < len(seqs):
            raise ValueError("a sequence is given twice")
        need = [max(-(-(a + n) // self.page_size) - len(self._tables[s]), 0) for s, a, n in zip(seqs, starts, counts)]
        if sum(need) > len(self._unused):
            raise RuntimeError(f"out of pages: {sum(need)} needed, {len(self._unused)} of {self.num_pages} unused")
        for s, a, n in zip(seqs, starts, counts):
            self.grow(s, a + n)
        ends = lambda x: torch.tensor([0, *x], dtype=torch.int64).cumsum(0).int().to(self.device)  # noqa: E731
        step = PagedStep(*self.slots(seqs, starts, counts), cu_seqlens=ends(counts))
        if any(starts):
            lengths = [a + n for a, n in zip(starts, counts)]
            step.key_slots = self.slots(seqs, [0] * len(seqs), lengths)[1]
            step.cu_seqlens_k = ends(lengths)
        return step

    def decode_step(self, block_tables: torch.Tensor, positions: torch.Tensor) -> PagedStep:
        """One new token of every sequence of a table, at positions[b] (int32 [B]; its page
        is dealt already): on the device alone, as next_slots."""
        return PagedStep(positions, self.next_slots(block_tables, positions), block_tables=block_tables,
                         seqlens=positions + 1)

    def read(self, layer: int, slots: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """The rows of `slots` (int64 [N]) as packed keys and values [N, n_kv_heads, D]."""
        page, row = torch.div(slots, self.page_size, rounding_mode="floor"), slots % self.page_size
        return self.k_pages[layer][page, :, row], self.v_pages[layer][page, :, row]
