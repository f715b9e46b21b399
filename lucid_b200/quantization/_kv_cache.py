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
    """A cache of zeros; ``fmt`` is ``"int8"`` (head_dim a multiple of 16) or ``"mxfp4"`` (of 32)."""
    if fmt not in _FORMATS:
        raise ValueError(f"cache format must be one of {sorted(_FORMATS)}, got {fmt!r}")
    step = 16 if fmt == "int8" else 32
    if head_dim <= 0 or head_dim % step or head_dim > 1024:
        raise _lib.ShapeMismatch(f"head_dim must be a multiple of {step} up to 1024 for {fmt}, got {head_dim}")
    if num_pages < 0 or page_size <= 0 or heads <= 0:
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
    """``(format, pages, page_size, heads, dim)`` of a cache whose tensors agree with each other."""
    kc, ks, vc, vs = cache
    _lib.require_cuda(kc, "cache k_codes")
    if kc.dim() != 4:
        raise _lib.ShapeMismatch(f"cache codes must be (pages, page_size, heads, ..), got {tuple(kc.shape)}")
    if kc.dtype == torch.int8:
        fmt, dim, scale_dtype, scale_shape = _lib.KV_INT8, kc.shape[3], torch.float32, kc.shape[:3]
    elif kc.dtype == torch.uint8:
        fmt, dim, scale_dtype = _lib.KV_MXFP4, kc.shape[3] * 2, torch.uint8
        scale_shape = (*kc.shape[:3], kc.shape[3] // 16)
    else:
        raise _lib.DtypeMismatch(f"cache codes must be int8 or uint8 (MXFP4), got {kc.dtype}")
    for name, t, dtype, shape in (("k_scales", ks, scale_dtype, scale_shape), ("v_codes", vc, kc.dtype, kc.shape),
                                  ("v_scales", vs, scale_dtype, scale_shape)):
        if not isinstance(t, torch.Tensor) or t.device != kc.device:
            raise _lib.DeviceMismatch(f"cache {name} must be a tensor on {kc.device}")
        if t.dtype != dtype:
            raise _lib.DtypeMismatch(f"cache {name} must be {dtype}, got {t.dtype}")
        if t.shape != shape:
            raise _lib.ShapeMismatch(f"cache {name} is {tuple(t.shape)}, expected {tuple(shape)}")
    if not (kc.is_contiguous() and ks.is_contiguous() and vc.is_contiguous() and vs.is_contiguous()):
        raise _lib.ShapeMismatch("the tensors of a cache must be contiguous")
    return fmt, kc.shape[0], kc.shape[1], kc.shape[2], dim


def _row_view(t: torch.Tensor) -> bool:
    """Whether the kernel can walk ``(tokens, heads, dim)`` as it lies: contiguous dim, 16-byte rows."""
    step = 16 // t.element_size()
    return t.stride(2) == 1 and t.stride(0) % step == 0 and t.stride(1) % step == 0 and t.data_ptr() % 16 == 0


def _distinct_rows(t: torch.Tensor) -> bool:
    """Whether the rows of ``(tokens, heads, dim)`` lie apart, tokens or heads outermost."""
    (n, h, d), (sn, sh, _) = t.shape, t.stride()
    return ((h <= 1 or sh >= d) and (n <= 1 or sn >= (h - 1) * sh + d)) or \
           ((n <= 1 or sn >= d) and (h <= 1 or sh >= (n - 1) * sn + d))


def kv_cache_write(cache: KVCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Encode the new rows ``k``, ``v`` ``(tokens, heads, dim)`` (float32 or bfloat16; strided views such as
    slices of a fused projection are read in place) into ``slots`` ``(tokens,)`` (int32 or int64).

    A negative slot is padding and skipped.  A slot past the cache is skipped and sets the device
    status word (``lucid_b200._lib.check_device_status``); nothing is synchronised here.  When a slot
    occurs twice the later token stays.  A row that holds a NaN or an infinity reads back as NaN (in
    MXFP4: its blocks of 32 that do)."""
    fmt, pages, page, heads, dim = _check_cache(cache)
    dev = cache.k_codes.device
    for name, t in (("k", k), ("v", v)):
        _lib.require_cuda(t, name)
        if t.device != dev:
            raise _lib.DeviceMismatch(f"{name} on {t.device}, the cache on {dev}")
        if t.dtype not in _FLOATS:
            raise _lib.DtypeMismatch(f"{name} must be float32 or bfloat16, got {t.dtype}")
        if t.dim() != 3 or t.shape[1] != heads or t.shape[2] != dim:
            raise _lib.ShapeMismatch(f"{name} is {tuple(t.shape)}, expected (tokens, {heads}, {dim})")
    if k.dtype != v.dtype:
        raise _lib.DtypeMismatch(f"k is {k.dtype}, v {v.dtype}")
    _lib.require_cuda(slots, "slots")
    if slots.device != dev:
        raise _lib.DeviceMismatch(f"slots on {slots.device}, the cache on {dev}")
    if slots.dtype not in (torch.int32, torch.int64):
        raise _lib.DtypeMismatch(f"slots must be int32 or int64, got {slots.dtype}")
    tokens = k.shape[0]
    if v.shape[0] != tokens or tuple(slots.shape) != (tokens,):
        raise _lib.ShapeMismatch(f"{tokens} rows of k, {v.shape[0]} of v, slots {tuple(slots.shape)}")
    k, v = k.detach(), v.detach()
    k = k if _row_view(k) else k.clone(memory_format=torch.contiguous_format)
    v = v if _row_view(v) else v.clone(memory_format=torch.contiguous_format)
    slots = slots.contiguous()
    _lib.call("lq_kv_write", dev, k.data_ptr(), v.data_ptr(), _lib.code_of(k.dtype), tokens, heads, dim, k.stride(0), k.stride(1),
          v.stride(0), v.stride(1), slots.data_ptr(), 64 if slots.dtype == torch.int64 else 32, pages * page, fmt,
          *(t.data_ptr() for t in cache), _lib.status_word(dev).data_ptr())


def kv_cache_read(cache: KVCache, block_tables: torch.Tensor, cu_seqlens: torch.Tensor, total: int,
                  starts: torch.Tensor | None = None, out=None, out_dtype: torch.dtype = torch.float32):
    """``(k, v)``, each ``(total, heads, dim)``: the rows of every sequence, packed one after the other.

    ``block_tables`` is int32 ``(sequences, max_pages)``, the pages of each sequence in order;
    ``cu_seqlens`` int32 ``(sequences + 1,)`` says which output rows belong to which sequence, and row
    ``cu_seqlens[b] + i`` is its token ``starts[b] + i`` (``starts`` int32, default zeros).  ``total`` is the
    number of output rows, known to the host.  ``out=(k, v)`` writes into given float32 / bfloat16
    tensors of any token and head stride; rows that no sequence covers keep what they held there,
    and are zeros in tensors allocated here.  A token past its row of the table, or a page outside
    the cache, reads as zeros and sets the device status word."""
    fmt, pages, page, heads, dim = _check_cache(cache)
    dev = cache.k_codes.device
    for name, t, dims in (("block_tables", block_tables, 2), ("cu_seqlens", cu_seqlens, 1), ("starts", starts, 1)):
        if t is None:
            continue
        _lib.require_cuda(t, name)
        if t.device != dev:
            raise _lib.DeviceMismatch(f"{name} on {t.device}, the cache on {dev}")
        if t.dtype != torch.int32:
            raise _lib.DtypeMismatch(f"{name} must be int32, got {t.dtype}")
        if t.dim() != dims:
            raise _lib.ShapeMismatch(f"{name} must have {dims} axes, got {tuple(t.shape)}")
    seqs, max_blocks = block_tables.shape
    if cu_seqlens.shape[0] != seqs + 1 or (starts is not None and starts.shape[0] != seqs):
        raise _lib.ShapeMismatch(f"{seqs} rows of block_tables, cu_seqlens {tuple(cu_seqlens.shape)}"
                                 + ("" if starts is None else f", starts {tuple(starts.shape)}"))
    total = int(total)
    if total < 0 or total >= 1 << 31:
        raise _lib.ShapeMismatch(f"total must be in [0, 2^31), got {total}")
    shape = (total, heads, dim)
    if out is None:
        if out_dtype not in _FLOATS:
            raise _lib.DtypeMismatch(f"kv_cache_read writes float32 or bfloat16, got {out_dtype}")
        ok = torch.empty(shape, dtype=out_dtype, device=dev)
        ov = torch.empty(shape, dtype=out_dtype, device=dev)
    else:
        ok, ov = out
        for t in (ok, ov):
            if not isinstance(t, torch.Tensor) or t.device != dev:
                raise _lib.DeviceMismatch(f"out= must be tensors on {dev}")
            if t.dtype not in _FLOATS or t.dtype != ok.dtype:
                raise _lib.DtypeMismatch(f"out= must be two float32 or two bfloat16 tensors, got {ok.dtype}, {ov.dtype}")
            if t.shape != shape:
                raise _lib.ShapeMismatch(f"out= is {tuple(t.shape)}, expected {shape}")
            if not _row_view(t) or not _distinct_rows(t):
                raise _lib.ShapeMismatch("out= needs a contiguous last axis and 16-byte aligned rows that do not overlap")
    table = block_tables if max_blocks <= 1 or block_tables.stride(1) == 1 else block_tables.contiguous()
    cu = cu_seqlens.contiguous()
    st = None if starts is None else starts.contiguous()
    _lib.call("lq_kv_read", dev, *(t.data_ptr() for t in cache), fmt, pages, page, heads, dim, table.data_ptr(), table.stride(0),
          max_blocks, cu.data_ptr(), _addr(st), seqs, total, ok.data_ptr(), ov.data_ptr(), _lib.code_of(ok.dtype),
          ok.stride(0), ok.stride(1), ov.stride(0), ov.stride(1), int(out is None), _lib.status_word(dev).data_ptr())
    return ok, ov
