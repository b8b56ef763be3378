"""Eviction from the cache by accumulated attention weight.

No counterpart in the reference, which keeps every token until its request
ends.  A pool that tracks key weights (``LayerBlockPool.track_key_weights``)
holds, for every head and cached token, the sum of the attention weights that
all queries so far gave it; each ``paged_attention`` on the pool adds its own.
``BatchedPagedKVCache.evict(keep, recent)`` then cuts every longer sequence of
the batch to ``keep`` tokens: the ``recent`` last ones and, per head, those of
the others with the largest sums.  Kept rows move together in order, so block
tables shrink and the freed blocks go back to the pool.  Works on plain and on
4-bit pools.

``accumulate_key_weights`` and ``evict_by_weight`` are the same operators on
pool tensors, block table and lengths.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .kv4 import (aligned_rows, check_heads, int32_rows, need_cuda, on_device, pool_shape, status_at, stream_at,
                  strides_of, table_args, workspace_of)

PLAIN_HEAD_DIMS = (16, 32, 64, 128, 256)
_MOST = 2 ** 31 - 1  # positions are 32-bit


def _pool_args(what: str, k_pool, v_pool, head_dim: int | None):
    """(blocks, H, block_size, D, type code) of a plain or 4-bit pool."""
    if k_pool.dim() != 4:
        raise ValueError(f"b2pa.{what}: k_pool must be a 4-d pool, not {tuple(k_pool.shape)}")
    if k_pool.dtype is torch.uint8:
        D = k_pool.shape[3] * 16 // 9 if head_dim is None else head_dim
        return (*pool_shape(what, D, k_pool, v_pool), D, _lib.DTYPE_KV4)
    code = _lib.dtype_code(k_pool.dtype)
    D = k_pool.shape[3]
    for t in (k_pool,) if v_pool is None else (k_pool, v_pool):
        if t.dtype is not k_pool.dtype or t.shape != k_pool.shape or not t.is_contiguous():
            raise ValueError(f"b2pa.{what}: pools must be contiguous [blocks, H, block_size, D] of one type and shape")
    if D not in PLAIN_HEAD_DIMS or (head_dim is not None and head_dim != D):
        raise ValueError(f"b2pa.{what}: head_dim {head_dim or D} does not fit k_pool of shape {tuple(k_pool.shape)}")
    return k_pool.shape[0], k_pool.shape[1], k_pool.shape[2], D, code


def _check_weights(what: str, name: str, w: torch.Tensor, shape: tuple) -> None:
    if w.dtype is not torch.float32 or w.shape != shape or not w.is_contiguous():
        raise ValueError(f"b2pa.{what}: {name} must be a contiguous float32 tensor of shape {shape}")


def accumulate_key_weights(q: torch.Tensor, k_pool: torch.Tensor, key_weights: torch.Tensor, page_table: torch.Tensor,
                           seq_lens: torch.Tensor, current_lengths: torch.Tensor, window: int | None = None,
                           out: torch.Tensor | None = None) -> torch.Tensor:
    """Adds to each cached key's sum in ``key_weights`` (fp32 [blocks, H, block_size]) the attention weights that the
    queries ``q`` [B, H, T, D] give it: those of ``t < current_lengths[b]``, or of the last ``window`` of them.
    ``k_pool`` is a plain pool of q's type or a 4-bit one.  The sums go to ``out`` (default: ``key_weights`` itself),
    whose other slots stay as they are; returns it.  A page belongs to one sequence of the call."""
    what = "accumulate_key_weights"
    out = key_weights if out is None else out
    if _lib.calls().key_weights(q, k_pool, key_weights, page_table, seq_lens, current_lengths, window,
                                out) is not NotImplemented:
        return out
    dev = need_cuda(what, q=q, k_pool=k_pool, key_weights=key_weights, page_table=page_table, seq_lens=seq_lens,
                    current_lengths=current_lengths, out=out)
    if q.dim() != 4:
        raise ValueError(f"b2pa.{what}: q must be [B, H, T, D], not {tuple(q.shape)}")
    B, _, T, D = q.shape
    blocks, H, bs, _, pool_code = _pool_args(what, k_pool, None, D)
    check_heads(what, "q", q, H)
    code = _lib.dtype_code(q.dtype)
    if pool_code != _lib.DTYPE_KV4 and pool_code != code:
        raise TypeError(f"pool dtype {k_pool.dtype} differs from q dtype {q.dtype}")
    if window is not None:
        if window < 1:
            raise ValueError(f"b2pa.{what}: window {window} < 1")
        window = min(window, T)
    for name, w in (("key_weights", key_weights), ("out", out)):
        _check_weights(what, name, w, (blocks, H, bs))
    table, pt_stride, pages = table_args(what, "page_table", page_table, B)
    seq_lens = int32_rows(what, "seq_lens", seq_lens, B)
    cur = int32_rows(what, "current_lengths", current_lengths, B)
    launch_key_weights(aligned_rows(q), k_pool, pool_code, key_weights, out, table, pt_stride, pages, seq_lens, cur,
                       window)
    return out


def launch_key_weights(q, k_pool, pool_code: int, key_weights, out, table, pt_stride: int, pages: int, seq_lens, cur,
                       window: int | None, ws: torch.Tensor | None = None) -> None:
    """b2pa_key_weights on checked arguments."""
    B, H, T, D = q.shape
    dev = q.get_device()
    code = _lib.dtype_code(q.dtype)
    bs = k_pool.shape[2]
    with on_device(dev):
        if ws is None:
            at, nbytes, ws = workspace_of(dev, "b2pa_key_weights_workspace_size", B, H, T, D, pages, bs, code, pool_code)
        else:
            at, nbytes = ws.data_ptr(), ws.numel()
        rc = _lib.load().b2pa_key_weights(
            q.data_ptr(), strides_of(q), k_pool.data_ptr(), pool_code, k_pool.shape[0], table.data_ptr(), pt_stride,
            pages, seq_lens.data_ptr(), cur.data_ptr(), window or 0, key_weights.data_ptr(), out.data_ptr(), B, H, T, D,
            bs, 1.0 / math.sqrt(D), code, at, nbytes, status_at(dev), stream_at(dev))
    if rc:
        _lib.check(rc, "b2pa_key_weights")


def evict_by_weight(k_pool: torch.Tensor, v_pool: torch.Tensor, key_weights: torch.Tensor, page_table: torch.Tensor,
                    seq_lens: torch.Tensor, keep: int, recent: int = 0,
                    out_table: torch.Tensor | None = None) -> torch.Tensor:
    """Cuts each sequence of n cached tokens to ``k = min(keep, n)``, each head for itself: the last ``min(recent, k)``
    stay, and of the others those with the largest ``key_weights`` (ties: the lower position).  The kept rows of both
    pools and their weights move, in order, to positions 0 .. k-1: in the same pages, or in those of ``out_table``
    ([B, >= ceil(keep / block_size)]; none of them in ``page_table``).  Slots behind the k-th row in its page are
    zeroed; pages behind it are left to the caller.  Returns the kept positions, int32 [B, H, keep], -1 behind k."""
    kept = _lib.calls().evict(k_pool, v_pool, key_weights, page_table, seq_lens, keep, recent, out_table)
    if kept is not NotImplemented:
        return kept
    what = "evict_by_weight"
    dev = need_cuda(what, k_pool=k_pool, v_pool=v_pool, key_weights=key_weights, page_table=page_table,
                    seq_lens=seq_lens, out_table=page_table if out_table is None else out_table)
    blocks, H, bs, D, pool_code = _pool_args(what, k_pool, v_pool, None)
    _check_weights(what, "key_weights", key_weights, (blocks, H, bs))
    if keep < 1 or recent < 0:
        raise ValueError(f"b2pa.{what}: keep must be at least 1 and recent not negative, got {keep} and {recent}")
    if keep > _MOST:
        raise ValueError(f"b2pa.{what}: keep {keep} is above {_MOST}")
    recent = min(recent, keep)
    B = page_table.shape[0]
    table, pt_stride, pages = table_args(what, "page_table", page_table, B)
    seq_lens = int32_rows(what, "seq_lens", seq_lens, B)
    out_stride = 0
    if out_table is not None:
        out_table, out_stride, out_pages = table_args(what, "out_table", out_table, B)
        if out_pages * bs < keep:
            raise ValueError(f"b2pa.{what}: out_table has {out_pages} pages a row, {-(-keep // bs)} needed")
    kept = torch.empty(B, H, keep, dtype=torch.int32, device=k_pool.device)
    with on_device(dev):
        rc = _lib.load().b2pa_evict(
            k_pool.data_ptr(), v_pool.data_ptr(), pool_code, key_weights.data_ptr(), blocks, table.data_ptr(),
            pt_stride, pages, out_table.data_ptr() if out_table is not None else None, out_stride,
            seq_lens.data_ptr(), keep, recent, kept.data_ptr(), B, H, D, bs, status_at(dev), stream_at(dev))
    if rc:
        _lib.check(rc, "b2pa_evict")
    return kept


# ------------------------------------------------------------- cache objects
def accumulate_from(kv_cache, q: torch.Tensor, current_lengths) -> None:
    """Adds the weights of ``q`` to the sums of ``kv_cache``'s pool, which tracks them (paged_attention calls this)."""
    from ._metadata import block_table_and_lengths, device_lengths

    pool = kv_cache.pool
    dev = q.device
    B, _, T, _ = q.shape
    if isinstance(current_lengths, torch.Tensor) and current_lengths.is_cuda:
        table, seq_lens, pages = block_table_and_lengths(kv_cache, dev, transient=True)
        cur = device_lengths(current_lengths, B)
    else:
        if current_lengths is None:
            row = T
        elif isinstance(current_lengths, torch.Tensor):
            row = current_lengths.numpy()
        elif isinstance(current_lengths, int):
            row = current_lengths
        else:
            row = [int(x) for x in current_lengths]
        table, seq_lens, cur, pages = block_table_and_lengths(kv_cache, dev, [row], transient=True)
    if pages == 0:
        return
    kb = pool.k_blocks
    launch_key_weights(aligned_rows(q), kb, _lib.DTYPE_KV4 if kb.dtype == torch.uint8 else _lib.dtype_code(kb.dtype),
                       pool.key_weights, pool.key_weights, table, table.stride(0), pages, seq_lens, cur,
                       min(pool.key_weight_window or T, T))


def evict_batch(cache, keep: int, recent: int = 0) -> torch.Tensor:
    """``BatchedPagedKVCache.evict``: cuts the sequences of ``cache`` in place and releases their freed blocks."""
    from ._metadata import block_table_and_lengths, note_released_rows
    from .paged_kv import flush_pending

    pool = cache.pool
    if getattr(pool, "_b2pa_step", None) is not None:
        raise RuntimeError("b2pa: a batch cannot be evicted inside an open DecodeStep")
    if keep < 1 or recent < 0:
        raise ValueError(f"b2pa: keep must be at least 1 and recent not negative, got {keep} and {recent}")
    if not getattr(pool, "_tracks_weights", False):
        raise RuntimeError("b2pa: the pool does not track key weights (call pool.track_key_weights() first)")
    if pool.k_blocks is None:
        raise RuntimeError("b2pa: nothing to evict from: the pool has no blocks before its first append")
    states = cache.states
    if any(s.pool is not pool for s in states):
        raise ValueError("b2pa: all states of a BatchedPagedKVCache must share its pool")
    if len({id(s) for s in states}) != len(states):
        raise ValueError("b2pa: a request occurs twice in the batch to evict")
    if getattr(pool, "_b2pa_pending", None) is not None:
        flush_pending(pool)
    dev = pool.k_blocks.device
    with on_device(dev.index):
        note_released_rows(cache, dev)
        table, seq_lens, pages = block_table_and_lengths(cache, dev, transient=True)
        most = max(1, min(keep, max((s.seq_len for s in states), default=1)))  # no sequence keeps more
        kept = evict_by_weight(pool.k_blocks, pool.v_blocks, pool.key_weights, table[:, :pages], seq_lens, most, recent)
        left = -(-keep // pool.block_size)
        freed = []
        for s in states:
            if s.seq_len > keep:
                freed += s.block_ids[left:]
                # a new list: cached copies of the block table go by the list's identity and length
                s.block_ids = s.block_ids[:left]
                s.seq_len = keep
        pool.release_blocks(freed)
    return kept
