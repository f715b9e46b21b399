"""A paged key / value cache held in few bits: encoded as it is written, decoded as it is read back.

``KVCache`` names the four tensors of a cache.  ``codes`` are ``(pages, page_size, heads, dim)`` int8 with
``scales`` float32 ``(pages, page_size, heads)`` -- per (token, head) the arithmetic of
:func:`quantize_per_token` -- or, in MXFP4 along the head dimension, uint8 ``(pages, page_size, heads,
dim / 2)`` with uint8 scale bytes ``(pages, page_size, heads, dim / 32)``.  Slot ``s`` is token ``s %
page_size`` of page ``s // page_size``."""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _lib
from ._mx import _FLOATS, _addr

_FORMATS = {"int8": _lib.KV_INT8, "mxfp4": _lib.KV_MXFP4}


class KVCache(NamedTuple):
    k_codes: torch.Tensor
    k_scales: torch.Tensor
    v_codes: torch.Tensor
    v_scales: torch.Tensor


def kv_cache_alloc(num_pages: int, page_size: int, heads: int, head_dim: int, fmt: str = "int8", device=None) -> KVCache:
    """A cache of zeros; ``fmt`` is ``"int8"`` (head_dim a multiple of 16) or ``"mxfp4"`` (of 32); up to 4096
    heads of up to 1024 values.  A cache without pages is one that every slot and every page lies outside."""
    if fmt not in _FORMATS:
        raise ValueError(f"cache format must be one of {sorted(_FORMATS)}, got {fmt!r}")
    step = 16 if fmt == "int8" else 32
    if head_dim <= 0 or head_dim % step or head_dim > 1024:
        raise _lib.ShapeMismatch(f"head_dim must be a multiple of {step} up to 1024 for {fmt}, got {head_dim}")
    if num_pages < 0 or page_size <= 0 or heads <= 0 or heads > 4096:
        raise _lib.ShapeMismatch(f"{num_pages} pages of {page_size} tokens x {heads} heads")
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else device
    lead = (num_pages, page_size, heads)

    def side():
        if fmt == "int8":
            return torch.zeros((*lead, head_dim), dtype=torch.int8, device=dev), torch.zeros(lead, device=dev)
        return (torch.zeros((*lead, head_dim // 2), dtype=torch.uint8, device=dev),
                torch.zeros((*lead, head_dim // 32), dtype=torch.uint8, device=dev))

    return KVCache(*side(), *side())


def _check_cache(cache) -> tuple:
    """``(format, pages, page_size, heads, dim, device)`` of a cache whose tensors agree with each other."""
    kc, ks, vc, vs = cache
    _lib.require_cuda(kc, "cache k_codes")
    shape = kc.shape
    if len(shape) != 4:
        raise _lib.ShapeMismatch(f"cache codes must be (pages, page_size, heads, ..), got {tuple(shape)}")
    pages, page, heads, width = shape
    if kc.dtype == torch.int8:
        fmt, dim, scale_dtype, scale_shape = _lib.KV_INT8, width, torch.float32, shape[:3]
    elif kc.dtype == torch.uint8:
        fmt, dim, scale_dtype, scale_shape = _lib.KV_MXFP4, width * 2, torch.uint8, (pages, page, heads, width // 16)
    else:
        raise _lib.DtypeMismatch(f"cache codes must be int8 or uint8 (MXFP4), got {kc.dtype}")
    dev = kc.device
    if not (ks.device == dev and vc.device == dev and vs.device == dev):
        raise _lib.DeviceMismatch(f"the tensors of a cache must be on one device, got {[str(t.device) for t in cache]}")
    if ks.dtype != scale_dtype or vc.dtype != kc.dtype or vs.dtype != scale_dtype:
        raise _lib.DtypeMismatch(f"cache of {kc.dtype} codes: expected {scale_dtype} scales, got {[t.dtype for t in cache]}")
    if ks.shape != scale_shape or vc.shape != shape or vs.shape != scale_shape:
        raise _lib.ShapeMismatch(f"codes {tuple(shape)} go with scales {tuple(scale_shape)}, got {[tuple(t.shape) for t in cache]}")
    if not (kc.is_contiguous() and ks.is_contiguous() and vc.is_contiguous() and vs.is_contiguous()):
        raise _lib.ShapeMismatch("the tensors of a cache must be contiguous")
    return fmt, pages, page, heads, dim, dev


def _row_view(t: torch.Tensor) -> bool:
    """Whether the kernel can walk ``(tokens, heads, dim)`` as it lies: contiguous dim, 16-byte rows."""
    sn, sh, one = t.stride()
    step = 16 // t.element_size()
    return one == 1 and sn % step == 0 and sh % step == 0 and t.data_ptr() % 16 == 0


def _distinct_rows(t: torch.Tensor) -> bool:
    """Whether the rows of ``(tokens, heads, dim)`` lie apart, tokens or heads outermost."""
    (n, h, d), (sn, sh, _) = t.shape, t.stride()
    return ((h <= 1 or sh >= d) and (n <= 1 or sn >= (h - 1) * sh + d)) or \
           ((n <= 1 or sn >= d) and (h <= 1 or sh >= (n - 1) * sn + d))


def _rows_meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two ``(tokens, heads, dim)`` tensors, each of distinct rows, share an address.  Answered for
    equal strides (halves of one buffer, however they interleave) and equal beginnings."""
    if a.numel() == 0:
        return False
    apart = abs(a.data_ptr() - b.data_ptr()) // a.element_size()
    d = a.shape[2]
    steps, others = (sorted(((s, c) for s, c in zip(t.stride()[:2], t.shape) if c > 1), reverse=True) for t in (a, b))
    if apart and (steps != others or apart >= sum(s * (c - 1) for s, c in steps) + d):
        return False
    left = [apart]  # what is left of the distance after whole steps of the longer stride, then of the shorter
    for step, count in steps:
        left = [r - i * step for r in left for i in (r // step, r // step + 1) if -count < i < count]
    return any(-d < r < d for r in left)


def kv_cache_write(cache: KVCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Encode the new rows ``k``, ``v`` ``(tokens, heads, dim)`` (float32 or bfloat16; strided views such as
    slices of a fused projection are read in place) into ``slots`` ``(tokens,)`` (int32 or int64).

    A negative slot is padding and skipped.  A slot past the cache is skipped and sets the device
    status word (``lucid_b200._lib.check_device_status``); nothing is synchronised here.  When a slot
    occurs twice the later token stays.  A row that holds a NaN or an infinity reads back as NaN (in
    MXFP4: its blocks of 32 that do)."""
    fmt, pages, page, heads, dim, dev = _check_cache(cache)
    _lib.require_cuda(k, "k")
    _lib.require_cuda(v, "v")
    _lib.require_cuda(slots, "slots")
    if k.device != dev or v.device != dev or slots.device != dev:
        raise _lib.DeviceMismatch(f"k on {k.device}, v on {v.device}, slots on {slots.device}, the cache on {dev}")
    if k.dtype not in _FLOATS or v.dtype != k.dtype:
        raise _lib.DtypeMismatch(f"k and v must both be float32 or both bfloat16, got {k.dtype}, {v.dtype}")
    if slots.dtype != torch.int64 and slots.dtype != torch.int32:
        raise _lib.DtypeMismatch(f"slots must be int32 or int64, got {slots.dtype}")
    shape = k.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != dim or v.shape != shape or slots.shape != shape[:1]:
        raise _lib.ShapeMismatch(f"expected k and v (tokens, {heads}, {dim}) and slots (tokens,), got {tuple(shape)}, "
                                 f"{tuple(v.shape)}, {tuple(slots.shape)}")
    k = k if _row_view(k) else k.detach().clone(memory_format=torch.contiguous_format)
    v = v if _row_view(v) else v.detach().clone(memory_format=torch.contiguous_format)
    slots = slots.contiguous()
    kt, kh, _ = k.stride()
    vt, vh, _ = v.stride()
    kc, ks, vc, vs = cache
    tokens = shape[0]
    room = tokens if tokens > 256 else 0  # lq_kv_write_workspace_bytes
    ws = torch.empty(room, dtype=torch.uint8, device=dev) if room else None
    _lib.call("lq_kv_write", dev, k.data_ptr(), v.data_ptr(), _lib.code_of(k.dtype), tokens, heads, dim, kt, kh, vt, vh,
              slots.data_ptr(), 64 if slots.dtype == torch.int64 else 32, pages * page, fmt, kc.data_ptr(), ks.data_ptr(),
              vc.data_ptr(), vs.data_ptr(), _addr(ws), room, _lib.status_ptr(dev))


def kv_cache_read(cache: KVCache, block_tables: torch.Tensor, cu_seqlens: torch.Tensor, total: int,
                  starts: torch.Tensor | None = None, out=None, out_dtype: torch.dtype = torch.float32):
    """``(k, v)``, each ``(total, heads, dim)``: the rows of every sequence, packed one after the other.

    ``block_tables`` is int32 ``(sequences, max_pages)``, the pages of each sequence in order;
    ``cu_seqlens`` int32 ``(sequences + 1,)`` says which output rows belong to which sequence, and row
    ``cu_seqlens[b] + i`` is its token ``starts[b] + i`` (``starts`` int32, default zeros).  ``total`` is the
    number of output rows, known to the host.  ``out=(k, v)`` writes into given float32 / bfloat16
    tensors of any token and head stride, no two rows of which overlap; rows that no sequence covers keep
    what they held there, and are zeros in tensors allocated here.  A token past its row of the table, or a page outside
    the cache, reads as zeros and sets the device status word."""
    fmt, pages, page, heads, dim, dev = _check_cache(cache)
    _lib.require_cuda(block_tables, "block_tables")
    _lib.require_cuda(cu_seqlens, "cu_seqlens")
    if block_tables.device != dev or cu_seqlens.device != dev:
        raise _lib.DeviceMismatch(f"block_tables on {block_tables.device}, cu_seqlens on {cu_seqlens.device}, the cache on {dev}")
    if block_tables.dtype != torch.int32 or cu_seqlens.dtype != torch.int32:
        raise _lib.DtypeMismatch(f"block_tables and cu_seqlens must be int32, got {block_tables.dtype}, {cu_seqlens.dtype}")
    if block_tables.dim() != 2:
        raise _lib.ShapeMismatch(f"block_tables must be (sequences, max_pages), got {tuple(block_tables.shape)}")
    seqs, max_blocks = block_tables.shape
    if cu_seqlens.shape != (seqs + 1,):
        raise _lib.ShapeMismatch(f"{seqs} rows of block_tables need {seqs + 1} cu_seqlens, got {tuple(cu_seqlens.shape)}")
    if starts is not None:
        _lib.require_cuda(starts, "starts")
        if starts.device != dev:
            raise _lib.DeviceMismatch(f"starts on {starts.device}, the cache on {dev}")
        if starts.dtype != torch.int32:
            raise _lib.DtypeMismatch(f"starts must be int32, got {starts.dtype}")
        if starts.shape != (seqs,):
            raise _lib.ShapeMismatch(f"{seqs} sequences, starts {tuple(starts.shape)}")
        starts = starts.contiguous()
    total = int(total)
    if total < 0 or total >= 1 << 31:
        raise _lib.ShapeMismatch(f"total must be in [0, 2^31), got {total}")
    if out is None:
        if out_dtype not in _FLOATS:
            raise _lib.DtypeMismatch(f"kv_cache_read writes float32 or bfloat16, got {out_dtype}")
        ok = torch.empty(total, heads, dim, dtype=out_dtype, device=dev)
        ov = torch.empty(total, heads, dim, dtype=out_dtype, device=dev)
    else:
        ok, ov = out
        shape = (total, heads, dim)
        for t in (ok, ov):
            if not isinstance(t, torch.Tensor) or t.device != dev:
                raise _lib.DeviceMismatch(f"out= must be tensors on {dev}")
            if t.dtype not in _FLOATS or t.dtype != ok.dtype:
                raise _lib.DtypeMismatch(f"out= must be two float32 or two bfloat16 tensors, got {ok.dtype}, {ov.dtype}")
            if t.shape != shape:
                raise _lib.ShapeMismatch(f"out= is {tuple(t.shape)}, expected {shape}")
            if not _row_view(t) or not _distinct_rows(t):
                raise _lib.ShapeMismatch("out= needs a contiguous last axis and 16-byte aligned rows that do not overlap")
        if _rows_meet(ok, ov):
            raise _lib.ShapeMismatch("out= has keys and values in the same memory")
    table = block_tables if max_blocks <= 1 or block_tables.stride(1) == 1 else block_tables.contiguous()
    cu = cu_seqlens.contiguous()
    kt, kh, _ = ok.stride()
    vt, vh, _ = ov.stride()
    kc, ks, vc, vs = cache
    _lib.call("lq_kv_read", dev, kc.data_ptr(), ks.data_ptr(), vc.data_ptr(), vs.data_ptr(), fmt, pages, page, heads, dim,
              table.data_ptr(), table.stride(0), max_blocks, cu.data_ptr(), _addr(starts), seqs, total, ok.data_ptr(),
              ov.data_ptr(), _lib.code_of(ok.dtype), kt, kh, vt, vh, int(out is None), _lib.status_ptr(dev))
    return ok, ov
