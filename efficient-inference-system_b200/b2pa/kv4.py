"""KV cache held in 4 bits.

No counterpart in the reference, whose pools have the model's type
(src/cache/paged_kv.py:54-62).  Decode reads the whole cache once per token
and the cache bounds how many requests fit the GPU; in 4 bits it takes 4.5
bits a value instead of 16 or 32.  Rows of D channels are stored in groups of
16 with one 8-bit floating scale each (the format is in include/b2pa.h).

Two levels, as for the plain pools:

* ``Kv4BlockPool`` is a ``LayerBlockPool`` whose pages are 4-bit;
  ``append_batch``, ``paged_attention``, ``DecodeStep``, ``DecodeGraph`` and
  ``FusedDecoder`` work on it as on a plain pool;
* ``kv4_append``, ``kv4_read``, ``paged_attention_decode_kv4`` and
  ``paged_attention_prefill_kv4`` take the pool tensors, block table and
  lengths, like ``paged_attention_decode_b200``.

Pools are uint8 ``[blocks, H, block_size, D * 9 / 16]``; head_dim 64, 128 or
256, q and new rows in fp32, bf16 or fp16.
"""
from __future__ import annotations

import contextlib
import math

import torch

from . import _lib
from .paged_kv import LayerBlockPool

HEAD_DIMS = (64, 128, 256)


class Kv4BlockPool(LayerBlockPool):
    """Block pool of one layer with K and V in 4 bits.  ``dtype`` is the type
    of the rows appended; ``k_blocks`` / ``v_blocks`` are uint8 ``[blocks, H,
    block_size, D * 9 / 16]``."""

    def ensure_initialized(self, num_heads: int, head_dim: int, dtype: torch.dtype, device: torch.device) -> None:
        if self.k_blocks is None and head_dim not in HEAD_DIMS:
            raise ValueError(f"b2pa.Kv4BlockPool: head_dim {head_dim} is not one of {HEAD_DIMS}")
        super().ensure_initialized(num_heads, head_dim, dtype, device)

    def _new_blocks(self, count: int) -> torch.Tensor:
        return torch.zeros(count, self.num_heads, self.block_size, self.head_dim * 9 // 16, dtype=torch.uint8,
                           device=self.device)


# ------------------------------------------------------------ argument checks
# Small calls are bound by the host, 13 us each with these checks and ctypes, so
# arguments that need no conversion go through csrc/py_calls.cpp first; these
# checks are for all others and for what has to be refused.
_current_device = torch._C._cuda_getDevice
_capturing = torch._C._cuda_isCurrentStreamCapturing
_NO_GUARD = contextlib.nullcontext()


def on_device(index: int):
    """Makes device ``index`` current for the launches of a call, if it is not."""
    return _NO_GUARD if index == _current_device() else torch.cuda.device(index)


def need_cuda(what: str, **tensors) -> int:
    """The index of the one CUDA device that holds all of ``tensors``."""
    index = -1
    for name, t in tensors.items():
        i = t.get_device()
        if i < 0:
            raise RuntimeError(f"b2pa: {name} must be a CUDA tensor (this package has no CPU path)")
        if i != index:
            if index >= 0:
                raise ValueError(f"b2pa.{what}: {name} is on {t.device}, not cuda:{index}")
            index = i
    return index


def int32_rows(what: str, name: str, t: torch.Tensor, B: int) -> torch.Tensor:
    """A [B] tensor of lengths or positions, int32 and contiguous."""
    if t.shape != (B,):
        raise ValueError(f"b2pa.{what}: {name} must have shape ({B},), not {tuple(t.shape)}")
    if t.dtype is torch.int32 and (B <= 1 or t.stride(0) == 1):
        return t
    return t.to(torch.int32).contiguous()


def table_args(what: str, name: str, t: torch.Tensor, B: int):
    """(tensor, row stride, pages) of a [B, pages] int32 block table."""
    if t.dim() != 2 or t.shape[0] != B:
        raise ValueError(f"b2pa.{what}: {name} must have shape ({B}, pages), not {tuple(t.shape)}")
    pages = t.shape[1]
    row, col = t.stride()
    if t.dtype is not torch.int32 or (pages > 1 and col != 1) or (B > 1 and row < pages):
        t = t.to(torch.int32).contiguous()
        row = pages
    return t, max(row, pages), pages


def pool_shape(what: str, head_dim: int, k_pool: torch.Tensor, v_pool: torch.Tensor | None = None) -> tuple[int, int, int]:
    """(blocks, H, block_size) of 4-bit pools, checked against ``head_dim``."""
    shape = k_pool.shape
    for t in (k_pool,) if v_pool is None else (k_pool, v_pool):
        if t.dtype is not torch.uint8 or t.dim() != 4 or not t.is_contiguous():
            raise TypeError(f"b2pa.{what}: 4-bit pools must be contiguous uint8 [blocks, H, block_size, D * 9 / 16] tensors")
        if t.shape != shape:
            raise ValueError(f"b2pa.{what}: k_pool and v_pool have different shapes")
    if head_dim not in HEAD_DIMS or shape[3] != head_dim * 9 // 16:
        raise ValueError(f"b2pa.{what}: head_dim {head_dim} does not fit pools of shape {tuple(shape)} "
                         f"(head_dim must be one of {HEAD_DIMS})")
    return shape[0], shape[1], shape[2]


def check_heads(what: str, name: str, t: torch.Tensor, H: int) -> None:
    if t.dim() != 4 or t.shape[1] != H:
        raise ValueError(f"b2pa.{what}: {name} must be [B, {H}, T, D], not {tuple(t.shape)}")


def aligned_rows(q: torch.Tensor) -> torch.Tensor:
    """``q`` itself when its rows are whole 16-byte words, else a copy."""
    b, h, t, d = q.stride()
    if d == 1 and q.data_ptr() % 16 == 0 and (b | h | t) * q.element_size() % 16 == 0:
        return q
    return q.clone(memory_format=torch.contiguous_format)


_strides: dict[tuple, object] = {}


def strides_of(t: torch.Tensor):
    """``_lib.strides4``, remembered by value."""
    key = t.stride()
    got = _strides.get(key)
    if got is None:
        if len(_strides) > 4096:
            _strides.clear()
        got = _strides[key] = _lib.strides4(t)
    return got


_sizes: dict[tuple, int] = {}


def workspace_of(index: int, fn: str, *sizes: int) -> tuple[int | None, int, torch.Tensor | None]:
    """(address, bytes, buffer) of the scratch that ``fn``(sizes) asks for; the answer depends on the sizes and the
    device alone and is remembered."""
    key = (index, fn, sizes)
    nbytes = _sizes.get(key)
    if nbytes is None:
        if len(_sizes) > 4096:
            _sizes.clear()
        nbytes = _sizes[key] = getattr(_lib.load(), fn)(*sizes)
    if not nbytes:
        return None, 0, None
    device = torch.device("cuda", index)
    # A stream under capture gets a buffer from the graph's own memory, so that captured graphs neither share scratch
    # nor lose it when the cached buffer is replaced by a larger one.
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if _capturing() else _lib.workspace(device, nbytes)
    return ws.data_ptr(), nbytes, ws


_status_at: dict[int, int] = {}


def status_at(index: int) -> int:
    """Address of the status word of device ``index``."""
    got = _status_at.get(index)
    if got is None:
        got = _status_at[index] = _lib.status_buffer(torch.device("cuda", index)).data_ptr()
        _lib.calls().set_status(index, got)
    return got


stream_at = torch._C._cuda_getCurrentRawStream


# ----------------------------------------------------------------- operators
def kv4_append(k_new: torch.Tensor, v_new: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
               page_table: torch.Tensor, start_pos: torch.Tensor, lengths: torch.Tensor,
               seq_lens_out: torch.Tensor | None = None) -> None:
    """Quantises rows ``t < lengths[b]`` of ``k_new`` / ``v_new`` ([B, H, T, D]) into positions ``start_pos[b] + t``
    of the 4-bit pools.  ``seq_lens_out`` (int64 [B]) receives the lengths after the append."""
    if _lib.calls().kv4_append(k_new, v_new, k_pool, v_pool, page_table, start_pos, lengths,
                               seq_lens_out) is not NotImplemented:
        return
    what = "kv4_append"
    dev = need_cuda(what, k_new=k_new, v_new=v_new, k_pool=k_pool, v_pool=v_pool, page_table=page_table,
                    start_pos=start_pos, lengths=lengths)
    if k_new.shape != v_new.shape or k_new.dtype is not v_new.dtype:
        raise ValueError("b2pa.kv4_append: k_new and v_new must have the same shape and dtype")
    if k_new.dim() != 4:
        raise ValueError(f"b2pa.kv4_append: k_new must be [B, H, T, D], not {tuple(k_new.shape)}")
    B, _, T, D = k_new.shape
    blocks, H, bs = pool_shape(what, D, k_pool, v_pool)
    check_heads(what, "k_new", k_new, H)
    table, pt_stride, pages = table_args(what, "page_table", page_table, B)
    start_pos = int32_rows(what, "start_pos", start_pos, B)
    lengths = int32_rows(what, "lengths", lengths, B)
    if seq_lens_out is not None and (seq_lens_out.dtype != torch.int64 or seq_lens_out.shape != (B,)
                                     or not seq_lens_out.is_contiguous() or seq_lens_out.get_device() != dev):
        raise ValueError("b2pa.kv4_append: seq_lens_out must be a contiguous int64 [B] tensor on the same device")
    code = _lib.dtype_code(k_new.dtype)
    with on_device(dev):
        rc = _lib.load().b2pa_kv4_append(
            k_new.data_ptr(), strides_of(k_new), v_new.data_ptr(), strides_of(v_new), k_pool.data_ptr(),
            v_pool.data_ptr(), blocks, table.data_ptr(), pt_stride, pages, start_pos.data_ptr(), lengths.data_ptr(),
            seq_lens_out.data_ptr() if seq_lens_out is not None else None, B, H, T, D, bs, code, status_at(dev),
            stream_at(dev))
    if rc:
        _lib.check(rc, "b2pa_kv4_append")


def kv4_read(k_pool: torch.Tensor, v_pool: torch.Tensor, page_table: torch.Tensor, start_pos: torch.Tensor,
             lengths: torch.Tensor, T: int, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """The values stored at positions ``start_pos[b] + t``, t < lengths[b], as ``(k, v)`` of shape [B, H, T, D] in
    ``dtype`` (exact in fp32, bf16 and fp16); rows behind ``lengths[b]`` are zeros."""
    out = _lib.calls().kv4_read(k_pool, v_pool, page_table, start_pos, lengths, T, dtype)
    if out is not NotImplemented:
        return out
    what = "kv4_read"
    dev = need_cuda(what, k_pool=k_pool, v_pool=v_pool, page_table=page_table, start_pos=start_pos, lengths=lengths)
    if T < 0:
        raise ValueError(f"b2pa.kv4_read: T {T} < 0")
    D = k_pool.shape[-1] * 16 // 9
    blocks, H, bs = pool_shape(what, D, k_pool, v_pool)
    code = _lib.dtype_code(dtype)
    B = page_table.shape[0]
    table, pt_stride, pages = table_args(what, "page_table", page_table, B)
    start_pos = int32_rows(what, "start_pos", start_pos, B)
    lengths = int32_rows(what, "lengths", lengths, B)
    k = torch.empty(B, H, T, D, dtype=dtype, device=k_pool.device)
    v = torch.empty_like(k)
    with on_device(dev):
        rc = _lib.load().b2pa_kv4_read(
            k_pool.data_ptr(), v_pool.data_ptr(), blocks, table.data_ptr(), pt_stride, pages, start_pos.data_ptr(),
            lengths.data_ptr(), k.data_ptr(), strides_of(k), v.data_ptr(), strides_of(v), B, H, T, D, bs, code,
            status_at(dev), stream_at(dev))
    if rc:
        _lib.check(rc, "b2pa_kv4_read")
    return k, v


def _attend(what: str, q, k_pool, v_pool, page_table, seq_lens, current_lengths, pages=None) -> torch.Tensor:
    decode = what == "paged_attention_decode_kv4"
    calls = _lib.calls()
    call = calls.decode_kv4 if decode else calls.prefill_kv4
    out = call(q, k_pool, v_pool, page_table, seq_lens, current_lengths, pages)
    if out is not NotImplemented:
        return out
    dev = need_cuda(what, q=q, k_pool=k_pool, v_pool=v_pool, page_table=page_table, seq_lens=seq_lens,
                    current_lengths=current_lengths)
    if q.dim() != 4:
        raise ValueError(f"b2pa.{what}: q must be [B, H, T, D], not {tuple(q.shape)}")
    B, _, T, D = q.shape
    blocks, H, bs = pool_shape(what, D, k_pool, v_pool)
    check_heads(what, "q", q, H)
    code = _lib.dtype_code(q.dtype)
    if decode and T != 1:
        raise ValueError(f"b2pa.{what}: q has {T} tokens per sequence, not 1")
    table, pt_stride, width = table_args(what, "page_table", page_table, B)
    if pages is None:
        pages = width
    seq_lens = int32_rows(what, "seq_lens", seq_lens, B)
    cur = int32_rows(what, "current_lengths", current_lengths, B)
    q = aligned_rows(q)
    out = torch.empty_like(q)
    lib = _lib.load()
    with on_device(dev):
        if decode:
            rc = lib.b2pa_paged_decode_kv4(
                q.data_ptr(), strides_of(q), k_pool.data_ptr(), v_pool.data_ptr(), blocks, table.data_ptr(), pt_stride,
                pages, seq_lens.data_ptr(), cur.data_ptr(), out.data_ptr(), strides_of(out), B, H, D, bs,
                1.0 / math.sqrt(D), code, status_at(dev), stream_at(dev))
        else:
            at, nbytes, ws = workspace_of(dev, "b2pa_paged_prefill_kv4_workspace_size", B, H, T, D, pages, bs, code)
            rc = lib.b2pa_paged_prefill_kv4(
                q.data_ptr(), strides_of(q), k_pool.data_ptr(), v_pool.data_ptr(), blocks, table.data_ptr(), pt_stride,
                pages, seq_lens.data_ptr(), cur.data_ptr(), out.data_ptr(), strides_of(out), B, H, T, D, bs,
                1.0 / math.sqrt(D), code, at, nbytes, status_at(dev), stream_at(dev))
    if rc:
        _lib.check(rc, "b2pa_paged_decode_kv4" if decode else "b2pa_paged_prefill_kv4")
    return out


def paged_attention_decode_kv4(q, k_pool, v_pool, page_table, seq_lens, current_lengths) -> torch.Tensor:
    """Single-query paged attention over 4-bit pools: ``paged_attention_decode_b200`` with a 4-bit cache."""
    return _attend("paged_attention_decode_kv4", q, k_pool, v_pool, page_table, seq_lens, current_lengths)


def paged_attention_prefill_kv4(q, k_pool, v_pool, page_table, seq_lens, current_lengths) -> torch.Tensor:
    """Chunked-prefill paged attention over 4-bit pools: ``paged_attention_prefill_b200`` with a 4-bit cache."""
    return _attend("paged_attention_prefill_kv4", q, k_pool, v_pool, page_table, seq_lens, current_lengths)
