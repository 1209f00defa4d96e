"""A paged key-value cache of one layer: pages on the GPU, and a native pool that says which belong to which sequence."""
from __future__ import annotations

from typing import List, Optional, Sequence

import torch

from ..ops.attention import cache_append, copy_pages, paged_attention


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x, or a copy of it where its rows are not what the kernels load (16 bytes at a time)."""
    fits = x.stride(-1) == 1 and all(s % 8 == 0 or n == 1 for s, n in zip(x.stride()[:-1], x.shape)) and x.data_ptr() % 16 == 0
    return x if fits else x.clone(memory_format=torch.contiguous_format)


class PagedKVCache:
    """``data`` is ``[pages, 2, kv_heads, page_size, head_dim]``; ``pool`` (``flashoverlap_class.PagePool``) keeps the
    sequences.  Everything on the GPU goes to the current stream: pages that ``free`` gives back may be written by what
    comes later in that stream, so a cache is used from one stream, or the streams are ordered by the caller.

    An operation that is refused, for want of pages or for what it is given, raises and leaves the cache as it was."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype=torch.bfloat16, device=None):
        if kv_heads < 1 or page_size < 1 or head_dim < 1 or head_dim % 8:
            raise ValueError("kv_heads, page_size and head_dim must be positive, head_dim a multiple of 8")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"a cache holds float16 or bfloat16, not {dtype}")
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        if device.type != "cuda":
            raise ValueError("the cache lives on a GPU")
        self.data = torch.zeros((pages, 2, kv_heads, page_size, head_dim), dtype=dtype, device=device)
        self.pool = torch.classes.flashoverlap_class.PagePool(pages, page_size)

    def add(self) -> int:
        """A new, empty sequence; returns its number."""
        return self.pool.add(0)

    def length(self, seq: int) -> int:
        return self.pool.length(seq)

    def _on_device(self, *parts: torch.Tensor) -> List[torch.Tensor]:
        """CPU tensors of int32 on the GPU, in one copy."""
        flat = torch.cat([p.reshape(-1) for p in parts]).to(self.data.device)
        return [f.view(p.shape) for f, p in zip(flat.split([p.numel() for p in parts]), parts)]

    def append(self, seqs: Sequence[int], k: torch.Tensor, v: torch.Tensor, counts: Optional[Sequence[int]] = None) -> None:
        """Stores ``k``, ``v`` ``[len(seqs), tokens, kv_heads, head_dim]`` behind the sequences' tokens (of a padded batch the
        first ``counts[i]`` tokens of sequence ``seqs[i]``)."""
        seqs, tokens = list(seqs), k.shape[1]
        if k.shape[0] != len(seqs) or (counts is not None and not all(0 <= c <= tokens for c in counts)):
            raise ValueError("one row of tokens for each sequence, and counts within them")
        for x in (k, v):
            if x.shape != k.shape or x.shape[2:] != self.data.shape[2::2] or x.dtype != self.data.dtype or x.device != self.data.device:
                raise ValueError("k and v must have the cache's heads, dtype and device")
            if x.requires_grad and torch.is_grad_enabled():
                raise ValueError("storing has no backward pass: call it under torch.no_grad()")
        starts = self.pool.lengths(seqs)
        new = [tokens] * len(seqs) if counts is None else [int(c) for c in counts]
        self.pool.grow(seqs, new)
        try:
            table, starts, stored = self._on_device(self.pool.table(seqs, 0), starts, torch.tensor(new, dtype=torch.int32))
            cache_append(_rows(k), _rows(v), self.data, table, starts, None if counts is None else stored)
        except BaseException:
            self.pool.shrink(seqs, new)  # the sequences do not end in tokens that have not been stored
            raise

    def take_back(self, seqs: Sequence[int], counts: Sequence[int]) -> None:
        """Removes the last ``counts[i]`` tokens of sequence ``seqs[i]``.  Refused where a sequence would end inside a page
        that it shares with a fork."""
        self.pool.shrink(list(seqs), [int(c) for c in counts])

    def attend(self, seqs: Sequence[int], q: torch.Tensor, window: int = 0, sinks: int = 0, scale: Optional[float] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of each sequence's last token, ``q[len(seqs), heads, head_dim]``, over its tokens."""
        table, lengths = self._on_device(self.pool.table(list(seqs), 0), self.pool.lengths(list(seqs)))
        return paged_attention(q, self.data, table, lengths, window=window, sinks=sinks, scale=scale, out=out)

    def fork(self, seq: int) -> int:
        """A new sequence with the tokens of another: full pages are shared, a last page that is not full is copied."""
        new, moves = self.pool.fork(seq)
        try:
            if moves.shape[0]:
                copy_pages(self.data, moves)
        except BaseException:
            self.pool.free(new)
            raise
        return new

    def free(self, seq: int) -> None:
        self.pool.free(seq)

    def compact(self) -> int:
        """Moves the pages in use to the front; returns how many were moved.  Tables made before are no longer right."""
        copy_pages(self.data, torch.empty((0, 2), dtype=torch.int32))  # (refused, if copying is, before the pool changes)
        moves = self.pool.compact()
        if moves.shape[0]:
            copy_pages(self.data, moves)
        return moves.shape[0]
