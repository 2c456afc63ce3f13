"""A paged key/value cache: the memory behind ops.paged_append and ops.paged_attention.

AutoKernel's models (models/llama_7b.py:67-88) recompute every key of a sequence in each forward;
here a sequence's keys and values stay in pages of `page_size` slots, which it gets as it grows and
gives back when it is released, so sequences of any length share one allocation made up front
(a token of 32 layers x 32 heads x 128 in 16 bits takes 0.5 MiB: 340,000 of them fill 180 GB).
The bookkeeping is on the host; what a step needs of it goes to the device as a Batch.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from ._lib import AkError


class CacheFull(AkError):
    """A step needs more pages than are free.  `answers`, where LlamaB200.generate met it: the tokens of each
    prompt that were sampled before."""
    answers: list[list[int]] | None = None


@dataclass
class Batch:
    """The device lists of one step (arguments of the paged operators) and what the host knows."""
    page_table: torch.Tensor  # int32 [B, pages of the longest sequence]
    cu_q: torch.Tensor        # int32 [B + 1]: the packed tokens of each sequence
    kv_lens: torch.Tensor     # int32 [B]: keys with the new tokens
    n_tokens: int             # new tokens of all sequences
    max_len: int              # keys of the longest sequence

    @property
    def lists(self) -> tuple:
        return self.page_table, self.cu_q, self.kv_lens


class PagedCache:
    """Keys and values [num_pages, kv_heads, page_size, head_dim] of every layer, and the pages of each
    sequence.  Sequences are numbers from add(); extend() makes room for new tokens."""

    def __init__(self, n_layers: int, kv_heads: int, head_dim: int, num_pages: int, page_size: int = 64,
                 dtype: torch.dtype = torch.float16, device="cuda"):
        if min(n_layers, kv_heads, head_dim, num_pages, page_size) < 1:
            raise ValueError("PagedCache: every size must be at least 1")
        self.page_size, self.num_pages, self.device = page_size, num_pages, torch.device(device)
        shape = (num_pages, kv_heads, page_size, head_dim)
        self.k = [torch.empty(shape, dtype=dtype, device=device) for _ in range(n_layers)]
        self.v = [torch.empty(shape, dtype=dtype, device=device) for _ in range(n_layers)]
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages: dict[int, list[int]] = {}
        self._lens: dict[int, int] = {}
        self._next = 0

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def add(self) -> int:
        """A new, empty sequence."""
        seq = self._next
        self._next += 1
        self._pages[seq], self._lens[seq] = [], 0
        return seq

    def length(self, seq: int) -> int:
        return self._lens[seq]

    def pages(self, seq: int) -> list[int]:
        return list(self._pages[seq])

    def release(self, seq: int) -> None:
        """Give the sequence's pages back (the next step on the same stream may fill them)."""
        self._free.extend(reversed(self._pages.pop(seq)))
        del self._lens[seq]

    def truncate(self, seq: int, length: int) -> None:
        """Forget the keys from position `length` on, and give back the pages that hold none of the rest: for
        tokens that extend() counted and no step wrote, or that a caller takes back."""
        if not 0 <= length <= self._lens[seq]:
            raise ValueError(f"PagedCache.truncate: length must lie in [0, {self._lens[seq]}], got {length}")
        pages, kept = self._pages[seq], -(-length // self.page_size)
        self._free.extend(reversed(pages[kept:]))
        del pages[kept:]
        self._lens[seq] = length

    def extend(self, seqs: list[int], counts: list[int]) -> Batch:
        """Room for counts[i] >= 1 new tokens of sequence seqs[i], and the lists of that step.  The tokens
        count as keys from here on: a step that is not run after all is taken back by truncate().  Raises
        CacheFull, with nothing changed, when the pages do not suffice."""
        if len(seqs) != len(counts) or not seqs:
            raise ValueError("PagedCache.extend: need one count per sequence, and a sequence")
        if len(set(seqs)) != len(seqs):
            raise ValueError("PagedCache.extend: a sequence is named twice")
        if min(counts) < 1:
            raise ValueError("PagedCache.extend: every count must be at least 1")
        lens = [self._lens[s] + c for s, c in zip(seqs, counts)]
        more = [-(-n // self.page_size) - len(self._pages[s]) for s, n in zip(seqs, lens)]
        if sum(more) > len(self._free):
            raise CacheFull(f"paged cache is full: {sum(more)} pages needed, {len(self._free)} free")
        for s, n, m in zip(seqs, lens, more):
            self._pages[s].extend(self._free.pop() for _ in range(m))
            self._lens[s] = n
        width = max(len(self._pages[s]) for s in seqs)
        cu = [0]
        for c in counts:
            cu.append(cu[-1] + c)
        # one copy to the device for all three lists; unused entries name no page
        flat = [p for s in seqs for p in self._pages[s] + [-1] * (width - len(self._pages[s]))]
        B = len(seqs)
        t = torch.tensor(flat + cu + lens, dtype=torch.int32).to(self.device)
        n = B * width
        return Batch(t[:n].view(B, width), t[n:n + B + 1], t[n + B + 1:], cu[-1], max(lens))


__all__ = ["Batch", "CacheFull", "PagedCache"]
