"""Attention of a decoder and its paged key-value cache, as functions of tensors.

The token at position j is visible from position i if ``j <= i < length`` (the sequence's length) and (``window == 0`` or
``j > i - window`` or ``j < sinks``): positions behind the length see nothing.  Query head h reads key and value head
``h // (heads // kv_heads)``.  A row that sees nothing is zero.  float16 and bfloat16, head_dim 64 or 128; scores, sums and
the statistics of the softmax are fp32, weights are rounded to the type of the values before they meet them.

A cache is ``[pages, 2, kv_heads, page_size, head_dim]``, keys at 0 and values at 1; pages may lie apart (one layer of
``[pages, layers, 2, ...]``).  Position j of sequence s lies in page ``page_table[s, j // page_size]`` at place
``j % page_size``.  Page numbers and lengths stay on the GPU and are not read by the host; the kernels check them.

Forward only: tensors that require a gradient are refused unless gradients are off.

The waits inside the prompt's kernel have a limit (``attention_set_timeout_ms``, 10 s by default).  One that runs out makes
the rows that its part of the work had not finished NaN, and is reported: later calls of ``prompt_attention`` on that device
raise, and ``attention_status`` says so, until ``attention_reset``.
"""
from __future__ import annotations

from typing import Optional

import torch

from .functional import _check


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int = 0, sinks: int = 0,
                     lengths: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of ``q[batch, sq, heads, head_dim]`` over ``k``, ``v`` ``[batch, sk, kv_heads, head_dim]``.

    The queries are the last ``sq`` of the ``sk`` tokens.  ``lengths[batch]`` (int32): how many of the ``sk`` tokens
    sequence b has; rows behind them are zero, and what stands there is not read into any result.  Strided views are fine
    as long as rows are contiguous and begin on 16-byte boundaries.  ``scale`` defaults to ``head_dim ** -0.5``.  ``out`` must
    be contiguous and may not lie between the first and the last value of q, k or v."""
    _check(q)
    if out is None:
        return torch.ops.flashoverlap_op.prompt_attention_new.default(q, k, v, window, sinks, lengths, scale)
    torch.ops.flashoverlap_op.prompt_attention.default(q, k, v, out, window, sinks, lengths, scale)
    return out


def _device_index(device) -> int:
    index = None if device is None else torch.device(device).index
    return torch.cuda.current_device() if index is None else index


def attention_status(device=None) -> str:
    """Waits for the device; "ok", or what ``prompt_attention`` has reported on it since the last ``attention_reset``."""
    index = _device_index(device)
    torch.cuda.synchronize(index)
    code, warp, cta = torch.ops.flashoverlap_op.attention_status.default(index)
    return "ok" if code == 0 else f"a wait ran out [code {code}, warp {warp} of CTA {cta}]"


def attention_reset(device=None) -> None:
    """Waits for the device and forgets what has been reported on it."""
    index = _device_index(device)
    torch.cuda.synchronize(index)
    torch.ops.flashoverlap_op.attention_reset.default(index)


def attention_set_timeout_ms(ms: float) -> float:
    """Limit of a wait in kernels launched from now on (a captured graph keeps the one of its capture); returns the one
    before."""
    return torch.ops.flashoverlap_op.attention_set_timeout_ns.default(round(ms * 1e6)) / 1e6


def paged_attention(q: torch.Tensor, cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                    window: int = 0, sinks: int = 0, scale: Optional[float] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one token per sequence, ``q[seqs, heads, head_dim]``, over what ``cache`` holds of it.

    ``page_table[seqs, width]`` and ``lengths[seqs]`` are int32 on the GPU; a length counts the token that asks, whose key
    and value are in the cache already (``cache_append``).  Sequences of length 0 give zero.  A visible token whose table
    entry is missing or no page of the cache is not read; all of that sequence's rows come out as NaN."""
    _check(q)
    if out is None:
        return torch.ops.flashoverlap_op.paged_attention_new.default(q, cache, page_table, lengths, window, sinks, scale)
    torch.ops.flashoverlap_op.paged_attention.default(q, cache, page_table, lengths, out, window, sinks, scale)
    return out


def cache_append(k: torch.Tensor, v: torch.Tensor, cache: torch.Tensor, page_table: torch.Tensor, starts: torch.Tensor,
                 counts: Optional[torch.Tensor] = None) -> None:
    """Stores token i of ``k``, ``v`` ``[seqs, tokens, kv_heads, head_dim]`` at position ``starts[s] + i`` of sequence s,
    for ``i < counts[s]`` (all without ``counts``).

    Positions below zero, behind the table's row, or in a page that the cache does not have are left out.  No two tokens
    of a call may go to one place: pages that are written belong to one sequence."""
    _check(k)
    torch.ops.flashoverlap_op.cache_append.default(k, v, cache, page_table, starts, counts)


def copy_pages(cache: torch.Tensor, moves: torch.Tensor) -> None:
    """Copies page ``moves[i, 0]`` of ``cache`` to page ``moves[i, 1]`` for all i.

    ``moves`` is an integer tensor ``[n, 2]`` on the CPU and is read before the call returns (a captured graph keeps the
    moves it was captured with).  A page may be copied to several others; none may be written twice, or written and
    read.  ``cache`` may be any tensor whose entries along its first dimension are contiguous."""
    _check(cache)
    torch.ops.flashoverlap_op.copy_pages.default(cache, moves)
