"""The 8-bit KV cache: quantising append, decode and prefill attention (HIP, gfx950).

The fp16 pool's operations (``store_kv``, ``paged_attention``, ``store_kv_and_decode``; reference
docs/architecture.md:242-253, modules src/infurnace/kernels/kv_store.py and paged_attention.py are
0-byte placeholders) over a cache of half the bytes, for a decode that is bound by them.  A layer's
cache is two tensors:

  * ``kv_pool`` [2, pages, Hkv, 16, D] ``torch.float8_e4m3fn`` (K = 0, V = 1; or the codes' bytes as uint8),
    or all layers' with a leading layer axis;
  * ``scales`` [2, pages, Hkv] fp32: one power of two for each block, the 16 tokens of a page and one
    kv head, of K or of V.  A value is its code times its block's scale.

``infurnace_amd.cache.PagedKVCacheFP8`` allocates both.  A block that starts (a token at offset 0 of
its page) takes the smallest scale that holds its new rows (max |x| <= 448 scale); rows that come
later raise it where they need to, and the block's earlier codes are rounded to the new scale.  Rows
of fp16 decode to fp16 numbers exactly, so the attention equals ``paged_attention`` over the fp16 pool
of the decoded values, within its tolerance.
"""
from __future__ import annotations

import contextlib
import math

import torch

from .. import _capi
from . import _fast
from ._carrier import accepts_carriers
from ._common import KVStoreError, PagedAttentionError, current_stream, ptr
from .paged_attention import _WORKSPACES, _check, _row_keys, _validate_pages, workspace_for

__all__ = ["store_kv_fp8", "paged_attention_fp8", "store_kv_fp8_and_decode", "EMPTY_SCALE"]

BLOCK = 16                  # tokens per page (and block)
EMPTY_SCALE = 2.0 ** -32    # scale of a block that holds nothing
_F8 = torch.float8_e4m3fn


def _check_cache(kv_pool, scales, layer: int, err: type[ValueError]):
    """(one layer's codes [2, P, Hkv, 16, D], its scales [2, P, Hkv], (P, Hkv, D))."""
    if not isinstance(kv_pool, torch.Tensor) or not isinstance(scales, torch.Tensor):
        raise err("kv_pool and scales must be torch tensors")
    if kv_pool.dtype == torch.uint8:  # (array libraries without the type hold the codes as bytes)
        kv_pool = kv_pool.view(_F8)
    if kv_pool.dtype != _F8:
        raise err(f"kv_pool dtype must be float8_e4m3fn (or uint8, the codes' bytes), got {kv_pool.dtype}")
    if scales.dtype != torch.float32:
        raise err(f"scales dtype must be float32, got {scales.dtype}")
    if kv_pool.ndim not in (5, 6):
        raise err(f"kv_pool must be rank 6 [layers, 2, pages, Hkv, {BLOCK}, D] or rank 5, got rank {kv_pool.ndim}")
    if kv_pool.shape[-5] != 2 or kv_pool.shape[-2] != BLOCK:
        raise err(f"kv_pool must be [..., 2, pages, Hkv, {BLOCK}, D], got {tuple(kv_pool.shape)}")
    if tuple(scales.shape) != tuple(kv_pool.shape[:-2]):
        raise err(f"scales shape must be {tuple(kv_pool.shape[:-2])}, got {tuple(scales.shape)}")
    if not kv_pool.is_contiguous() or not scales.is_contiguous():
        raise err("kv_pool and scales must be contiguous")
    if kv_pool.device.type != "cuda":
        raise err(f"kv_pool must be a GPU tensor, got device {kv_pool.device}")
    if scales.device != kv_pool.device:
        raise err(f"scales must be on {kv_pool.device}, got {scales.device}")
    layers = kv_pool.shape[0] if kv_pool.ndim == 6 else 1
    if not 0 <= layer < layers:
        raise err(f"layer {layer} out of range [0, {layers})")
    if kv_pool.ndim == 6:
        kv_pool, scales = kv_pool[layer], scales[layer]
    _, P, hkv, _, d = kv_pool.shape
    if P < 1 or hkv < 1 or d < 1:
        raise err(f"kv_pool has an empty axis: {tuple(kv_pool.shape)}")
    return kv_pool, scales, (P, hkv, d)


def _current(device: torch.device):
    """The device a call's tensors are on, made current for it."""
    return contextlib.nullcontext() if device.index in (None, torch.cuda.current_device()) else torch.cuda.device(device)


def _workspace(device: torch.device, stream: int, nbytes: int) -> torch.Tensor:
    """The stream's workspace; under graph capture one of the graph's own, whose tickets each replay clears (a
    cached one could be replaced, or used by another graph, while this graph lives)."""
    if not torch.cuda.is_current_stream_capturing():
        return workspace_for(device, stream, nbytes)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    ws[:_TICKET_BYTES].zero_()
    return ws


_TICKET_BYTES = 256 << 10  # the tickets at a workspace's start: zero before a call, and after it


def _check_rows(name: str, t, shape: tuple, device, err: type[ValueError]) -> None:
    if not isinstance(t, torch.Tensor):
        raise err(f"{name} must be a torch.Tensor")
    if t.dtype != torch.float16 or tuple(t.shape) != shape or t.device != device or not t.is_contiguous():
        raise err(f"{name} must be a contiguous float16 {list(shape)} tensor on {device}, got {t.dtype} "
                  f"{list(t.shape)} on {t.device}")


def _validate_slots(slots: torch.Tensor, active, num_slots: int) -> None:
    """Validate mode: active slots in the pool and distinct."""
    s = slots.detach().cpu().long()
    if active is not None:
        s = s[active.detach().cpu().bool()]
    if s.numel() == 0:
        return
    if int(s.min()) < 0 or int(s.max()) >= num_slots:
        raise KVStoreError(f"active slot outside [0, {num_slots})")
    if s.numel() != torch.unique(s).numel():
        raise KVStoreError("two active rows map to the same slot")


def _validate_scales(scales: torch.Tensor, table: torch.Tensor, keys: torch.Tensor) -> None:
    """Validate mode: the scales of every page that is read are positive powers of two."""
    need = (keys + BLOCK - 1) // BLOCK
    used = torch.arange(table.shape[1], device=table.device)[None, :] < need[:, None]
    got = scales[:, table[used].long()]
    if not bool(((got > 0) & torch.isfinite(got) & (torch.frexp(got)[0] == 0.5)).all()):
        raise PagedAttentionError("scales of pages that are read must be positive powers of two")


def _validate_append(table: torch.Tensor, keys: torch.Tensor, stores: torch.Tensor, num_pages: int) -> None:
    """Validate mode: the page that a row's new token goes to (rows with ``stores``) is read by no other row."""
    need = (keys + BLOCK - 1) // BLOCK
    used = torch.arange(table.shape[1], device=table.device)[None, :] < need[:, None]
    times = torch.bincount(table[used].long(), minlength=num_pages)
    live = (need > 0) & stores
    last = table[live].gather(1, need[live][:, None] - 1).long()
    if bool((times[last] != 1).any()):
        raise PagedAttentionError("the last page of a row is in another row's table: its new token cannot be appended here")


def store_kv_fp8(kv_pool: torch.Tensor, scales: torch.Tensor, slot_mapping: torch.Tensor,
                 active_mask: torch.Tensor | None, new_k: torch.Tensor, new_v: torch.Tensor, *, layer: int = 0,
                 validate: bool = False) -> None:
    """Append ``new_k`` / ``new_v`` [T, Hkv, D] fp16 to the 8-bit cache in place (``ifn_store_kv_fp8``).

    ``slot_mapping`` int32 [T] and ``active_mask`` bool/uint8 [T] or None as for ``store_kv``: rows that are
    inactive or whose slot is outside the pool write nothing.  A page is filled from its offset 0 up: the
    token at offset 0 starts its blocks anew.  A call's tokens may be in any order, those of a sequence in
    order side by side being the fastest.  Active slots are distinct; ``validate=True`` adds a
    synchronising host check of that.
    """
    if not validate and _fast.store_fp8(kv_pool, scales, slot_mapping, active_mask, new_k, new_v, layer) is not None:
        return None
    return _store(kv_pool, scales, slot_mapping, active_mask, new_k, new_v, layer, validate)


@accepts_carriers
def _store(kv_pool, scales, slot_mapping, active_mask, new_k, new_v, layer, validate) -> None:
    pool_layer, scales_layer, (P, hkv, d) = _check_cache(kv_pool, scales, layer, KVStoreError)
    dev = pool_layer.device
    if not isinstance(new_k, torch.Tensor) or new_k.ndim != 3:
        raise KVStoreError("new_k must be a rank-3 [T, Hkv, D] tensor")
    T = new_k.shape[0]
    _check_rows("new_k", new_k, (T, hkv, d), dev, KVStoreError)
    _check_rows("new_v", new_v, (T, hkv, d), dev, KVStoreError)
    from .kv_store import _check_index
    sm = _check_index("slot_mapping", slot_mapping, T, dev, (torch.int32,))
    if sm is None:
        raise KVStoreError("store_kv_fp8 needs a slot_mapping")
    am = _check_index("active_mask", active_mask, T, dev, (torch.bool, torch.uint8))
    if validate:
        _validate_slots(sm, am, P * BLOCK)
    if T == 0:
        return
    with _current(dev):
        _capi.call("ifn_store_kv_fp8", ptr(pool_layer), ptr(scales_layer), P, ptr(sm), ptr(am), ptr(new_k), ptr(new_v),
                   T, hkv, d, BLOCK, current_stream(dev))


@accepts_carriers
def _decode(query, kv_pool, scales, block_tables, sequence_lengths, active_mask, new_k, new_v, append, layer, scale, out,
            max_seq_len, page_weights, validate):
    err = PagedAttentionError
    pool_layer, scales_layer, (P, hkv, d) = _check_cache(kv_pool, scales, layer, err)
    dev = pool_layer.device
    if not isinstance(query, torch.Tensor) or query.ndim != 3:
        raise err("query must be a rank-3 tensor ([B, Hq, D] decode or [T, Hq, D] prefill)")
    n, hq, _ = query.shape
    if hq < 1 or hq % hkv:
        raise err(f"num_q_heads {hq} is not a positive multiple of num_kv_heads {hkv}")
    _check_rows("query", query, (n, hq, d), dev, err)
    if not isinstance(block_tables, torch.Tensor) or block_tables.ndim != 2:
        raise err("block_tables must be a rank-2 [B, max_pages] int32 tensor")
    max_pages = block_tables.shape[1]
    _check("block_tables", block_tables, (n, max_pages), (torch.int32,), dev)
    _check("sequence_lengths", sequence_lengths, (n,), (torch.int32,), dev)
    if active_mask is not None:
        _check("active_mask", active_mask, (n,), (torch.bool, torch.uint8), dev)
    if max_pages < 1:
        raise err("block_tables must have at least one column")
    if append:
        _check_rows("new_k", new_k, (n, hkv, d), dev, err)
        _check_rows("new_v", new_v, (n, hkv, d), dev, err)
    if page_weights is not None:
        _check("page_weights", page_weights, (n, hkv, max_pages), (torch.float32,), dev)
    if out is None:
        out = torch.zeros_like(query) if active_mask is not None else torch.empty_like(query)
    else:
        _check("out", out, (n, hq, d), (torch.float16,), dev)
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    if not scale > 0:
        raise err(f"scale must be positive, got {scale}")
    cap = max_pages * BLOCK
    msl = cap if max_seq_len is None else min(int(max_seq_len), cap)
    if msl < 0:
        raise err("max_seq_len must be non-negative")
    if n == 0:
        return out
    if validate:
        keys = _row_keys(sequence_lengths, active_mask, msl)
        _validate_pages(block_tables, keys, P, BLOCK, "paged_attention_fp8")
        _validate_scales(scales_layer, block_tables, keys)
        if append:
            _validate_append(block_tables, keys, sequence_lengths <= msl, P)
    with _current(dev):
        stream = current_stream(dev)
        nbytes = _capi.lib().ifn_paged_decode_fp8_workspace_bytes(n, hq, hkv, d, BLOCK, max_pages, msl,
                                                                  page_weights is not None)
        ws = _workspace(dev, stream, nbytes)
        head = (ptr(out), ptr(query), ptr(pool_layer), ptr(scales_layer), P, ptr(block_tables), max_pages,
                ptr(sequence_lengths), ptr(active_mask))
        tail = (ptr(page_weights), n, hq, hkv, d, BLOCK, msl, float(scale), ptr(ws), ws.numel(), stream)
        if append:
            _capi.call("ifn_paged_decode_append_fp8", *head, ptr(new_k), ptr(new_v), *tail)
        else:
            _capi.call("ifn_paged_decode_fp8", *head, *tail)
    return out


def paged_attention_fp8(query: torch.Tensor, kv_pool: torch.Tensor, scales: torch.Tensor, block_tables: torch.Tensor,
                        sequence_lengths: torch.Tensor | None, active_mask: torch.Tensor | None = None, *,
                        layer: int = 0, scale: float | None = None, query_start: int | None = None,
                        out: torch.Tensor | None = None, max_seq_len: int | None = None,
                        page_weights: torch.Tensor | None = None, validate: bool = False) -> torch.Tensor:
    """``paged_attention`` over the 8-bit cache; returns ``out`` (allocated when None).

    Decode (``query_start is None``, ``ifn_paged_decode_fp8``): ``query`` [B, Hq, D] fp16, ``block_tables`` int32
    [B, max_pages], ``sequence_lengths`` int32 [B], ``active_mask`` bool/uint8 [B] or None, ``max_seq_len`` as for
    ``paged_attention``; Hq / Hkv up to 16, head_dim 64, 128 or 256.  ``page_weights`` fp32
    [B, Hkv, max_pages]: to entry (b, h, j) the attention probability that kv head h's queries give the keys of
    row b's page j is added (over a row's pages the sum is Hq / Hkv a call), for ``evict_pages``.

    Prefill (``query_start`` given, ``ifn_paged_prefill_fp8``): ``query`` [T, Hq, D] of one sequence whose chunk
    is already stored, ``block_tables`` int32 [max_pages] or [1, max_pages], ``sequence_lengths`` and
    ``active_mask`` None; row i attends keys [0, query_start + i].  head_dim 64 or 128.

    ``validate=True`` (it synchronises): the table entries that are read name pages of the pool, and their scales
    are powers of two.
    """
    if query_start is None:
        if not validate:
            o = _fast.decode_fp8(query, kv_pool, scales, block_tables, sequence_lengths, active_mask, None, None, layer,
                                 scale, out, max_seq_len, page_weights, _WORKSPACES)
            if o is not None:
                return o
        return _decode(query, kv_pool, scales, block_tables, sequence_lengths, active_mask, None, None, False, layer,
                       scale, out, max_seq_len, page_weights, validate)
    if (sequence_lengths is None and active_mask is None and max_seq_len is None and page_weights is None and
            not validate):
        o = _fast.prefill_fp8(query, kv_pool, scales, block_tables, query_start, layer, scale, out, _WORKSPACES)
        if o is not None:
            return o
    return _prefill(query, kv_pool, scales, block_tables, sequence_lengths, active_mask, layer, scale, query_start, out,
                    max_seq_len, page_weights, validate)


@accepts_carriers
def _prefill(query, kv_pool, scales, block_tables, sequence_lengths, active_mask, layer, scale, query_start, out,
             max_seq_len, page_weights, validate):
    err = PagedAttentionError
    pool_layer, scales_layer, (P, hkv, d) = _check_cache(kv_pool, scales, layer, err)
    dev = pool_layer.device
    if sequence_lengths is not None or active_mask is not None or max_seq_len is not None or page_weights is not None:
        raise err("prefill takes no sequence_lengths, active_mask, max_seq_len or page_weights")
    if not isinstance(query, torch.Tensor) or query.ndim != 3:
        raise err("query must be a rank-3 tensor ([B, Hq, D] decode or [T, Hq, D] prefill)")
    n, hq, _ = query.shape
    if hq < 1 or hq % hkv:
        raise err(f"num_q_heads {hq} is not a positive multiple of num_kv_heads {hkv}")
    _check_rows("query", query, (n, hq, d), dev, err)
    query_start = int(query_start)
    if query_start < 0:
        raise err(f"query_start must be non-negative, got {query_start}")
    if not isinstance(block_tables, torch.Tensor):
        raise err("block_tables must be a torch.Tensor")
    table = block_tables.reshape(-1) if block_tables.ndim == 2 and block_tables.shape[0] == 1 else block_tables
    if table.ndim != 1:
        raise err("prefill block_tables must be [max_pages] or [1, max_pages]")
    _check("block_tables", table, (table.shape[0],), (torch.int32,), dev)
    total = query_start + n
    if total > table.shape[0] * BLOCK:
        raise err(f"query_start + T = {total} exceeds the table's {table.shape[0] * BLOCK} slots")
    if out is None:
        out = torch.empty_like(query)
    else:
        _check("out", out, (n, hq, d), (torch.float16,), dev)
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    if not scale > 0:
        raise err(f"scale must be positive, got {scale}")
    if n == 0:
        return out
    if validate:
        keys = torch.full((1,), total, dtype=torch.int64, device=dev)
        _validate_pages(table[None, :], keys, P, BLOCK, "paged_attention_fp8 (prefill)")
        _validate_scales(scales_layer, table[None, :], keys)
    with _current(dev):
        stream = current_stream(dev)
        nbytes = _capi.lib().ifn_paged_prefill_fp8_workspace_bytes(n, query_start, hq, hkv, d, BLOCK)
        ws = _workspace(dev, stream, nbytes)
        _capi.call("ifn_paged_prefill_fp8", ptr(out), ptr(query), ptr(pool_layer), ptr(scales_layer), P, ptr(table),
                   table.shape[0], query_start, n, hq, hkv, d, BLOCK, float(scale), ptr(ws), ws.numel(), stream)
    return out


def store_kv_fp8_and_decode(query: torch.Tensor, kv_pool: torch.Tensor, scales: torch.Tensor, block_tables: torch.Tensor,
                            sequence_lengths: torch.Tensor, active_mask: torch.Tensor | None, new_k: torch.Tensor,
                            new_v: torch.Tensor, *, layer: int = 0, scale: float | None = None,
                            out: torch.Tensor | None = None, max_seq_len: int | None = None,
                            page_weights: torch.Tensor | None = None, validate: bool = False) -> torch.Tensor:
    """One decode step's append and attention over the 8-bit cache in one launch (``ifn_paged_decode_append_fp8``).

    Row b's ``new_k`` / ``new_v`` [B, Hkv, D] fp16 are stored at position ``sequence_lengths[b] - 1`` of its table:
    the same cache and output as ``store_kv_fp8`` of those slots followed by ``paged_attention_fp8``.  Rows that
    are inactive, empty or longer than ``max_seq_len`` store nothing.  A row's last page must be in no other
    row's table (true of any paged KV state; ``validate=True`` checks it).
    """
    if not validate and new_k is not None:
        o = _fast.decode_fp8(query, kv_pool, scales, block_tables, sequence_lengths, active_mask, new_k, new_v, layer,
                             scale, out, max_seq_len, page_weights, _WORKSPACES)
        if o is not None:
            return o
    return _decode(query, kv_pool, scales, block_tables, sequence_lengths, active_mask, new_k, new_v, True, layer, scale,
                   out, max_seq_len, page_weights, validate)
