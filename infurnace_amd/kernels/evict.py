"""evict_pages: eviction of cache pages by accumulated attention weight (HIP, gfx950).

The reference has no counterpart (its cache rows only grow); this works on the block tables of its
documented paged layout (docs/architecture.md:234-240).  The weights are what the 8-bit cache's decode
calls add up in ``page_weights``.
"""
from __future__ import annotations

import torch

from .. import _capi
from . import _fast
from ._carrier import accepts_carriers
from ._common import PagedAttentionError, current_stream, ptr
from .kv_fp8 import _current
from .paged_attention import _check

__all__ = ["evict_pages"]


def evict_pages(block_tables: torch.Tensor, sequence_lengths: torch.Tensor, page_weights: torch.Tensor, keep_pages: int,
                *, sink_pages: int = 1, recent_pages: int = 1, active_mask: torch.Tensor | None = None,
                block_size: int = 16) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Cut every row of more than ``keep_pages`` pages to that many; returns new
    (block_tables, sequence_lengths, page_weights, num_evicted).

    ``block_tables`` int32 [B, max_pages], ``sequence_lengths`` int32 [B], ``page_weights`` fp32
    [B, Hkv, max_pages].  A row keeps its first ``sink_pages``, its last ``recent_pages`` (at least one: it
    may be partial) and, of the others, those of largest weight summed over the kv heads, ties to the lower
    position (NaN is lowest).  Tables and weights close up in order; a row's evicted ids follow its kept ones
    (``num_evicted`` int32 [B] of them), for the caller to release.  Tokens keep the rotary positions they were
    stored with; the length only counts what is held.  No page is moved or written, so shared pages are safe.
    """
    got = _fast.evict(block_tables, sequence_lengths, page_weights, keep_pages, sink_pages, recent_pages, active_mask,
                      block_size)
    if got is not None:
        return got
    return _evict(block_tables, sequence_lengths, page_weights, keep_pages, sink_pages, recent_pages, active_mask,
                  block_size)


@accepts_carriers
def _evict(block_tables, sequence_lengths, page_weights, keep_pages, sink_pages, recent_pages, active_mask, block_size):
    err = PagedAttentionError
    if not isinstance(block_tables, torch.Tensor) or block_tables.ndim != 2:
        raise err("block_tables must be a rank-2 [B, max_pages] int32 tensor")
    dev = block_tables.device
    if dev.type != "cuda":
        raise err(f"block_tables must be a GPU tensor, got device {dev}")
    n, max_pages = block_tables.shape
    _check("block_tables", block_tables, (n, max_pages), (torch.int32,), dev)
    if max_pages < 1:
        raise err("block_tables must have at least one column")
    _check("sequence_lengths", sequence_lengths, (n,), (torch.int32,), dev)
    if not isinstance(page_weights, torch.Tensor) or page_weights.ndim != 3 or page_weights.shape[1] < 1:
        raise err("page_weights must be a rank-3 [B, Hkv, max_pages] float32 tensor")
    hkv = page_weights.shape[1]
    _check("page_weights", page_weights, (n, hkv, max_pages), (torch.float32,), dev)
    if active_mask is not None:
        _check("active_mask", active_mask, (n,), (torch.bool, torch.uint8), dev)
    keep, sink, recent = int(keep_pages), int(sink_pages), int(recent_pages)
    if sink < 0 or recent < 1 or keep < sink + recent:
        raise err(f"keep_pages {keep} must hold sink_pages {sink} (>= 0) and recent_pages {recent} (>= 1)")
    if keep >= max_pages:  # no row holds more
        keep, sink, recent = max_pages, 0, 1
    tables, lens = torch.empty_like(block_tables), torch.empty_like(sequence_lengths)
    weights, gone = torch.empty_like(page_weights), torch.empty_like(sequence_lengths)
    if n == 0:
        return tables, lens, weights, gone
    with _current(dev):
        _capi.call("ifn_evict_pages", ptr(tables), ptr(lens), ptr(weights), ptr(gone), ptr(block_tables), max_pages,
                   ptr(sequence_lengths), ptr(active_mask), ptr(page_weights), n, hkv, block_size, keep, sink, recent,
                   current_stream(dev))
    return tables, lens, weights, gone
