"""The quantized key / value cache as a module: its tensors are buffers, so it moves with the model it
belongs to, whose changes of type leave it alone (they are state of a run, not of a checkpoint, and stay out of
``state_dict``)."""

from __future__ import annotations

import torch

from ...quantization._kv_cache import KVCache, kv_cache_alloc, kv_cache_read, kv_cache_write


class PagedKVCache(torch.nn.Module):
    """``num_pages`` pages of ``page_size`` tokens, ``heads`` x ``head_dim`` values each for keys and for
    values; ``fmt`` ``"int8"`` or ``"mxfp4"`` (:mod:`lucid_b200.quantization._kv_cache`).  Like the other
    modules it is made on the CPU and moved by ``.cuda()``, or made where ``device`` says."""

    def __init__(self, num_pages: int, page_size: int, heads: int, head_dim: int, fmt: str = "int8", device=None) -> None:
        super().__init__()
        self.page_size, self.heads, self.head_dim, self.fmt = page_size, heads, head_dim, fmt
        alloc = kv_cache_alloc(num_pages, page_size, heads, head_dim, fmt, "cpu" if device is None else device)
        for name, t in alloc._asdict().items():
            self.register_buffer(name, t, persistent=False)

    def _apply(self, fn, recurse=True):
        # ``model.to(torch.bfloat16)`` means the model's weights: the types of a cache are those of its format, and its
        # float32 scales would lose bits on the way
        def keep_type(t):
            moved = fn(t)
            return moved if moved.dtype == t.dtype else t.to(moved.device)

        return super()._apply(keep_type, recurse)

    @property
    def cache(self) -> KVCache:
        return KVCache(self.k_codes, self.k_scales, self.v_codes, self.v_scales)

    def write(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """:func:`~lucid_b200.quantization.kv_cache_write`."""
        kv_cache_write(self.cache, k, v, slots)

    def read(self, block_tables, cu_seqlens, total, starts=None, out=None, out_dtype: torch.dtype = torch.float32):
        """:func:`~lucid_b200.quantization.kv_cache_read`."""
        return kv_cache_read(self.cache, block_tables, cu_seqlens, total, starts=starts, out=out, out_dtype=out_dtype)

    def extra_repr(self) -> str:
        return (f"{self.k_codes.shape[0]} pages x {self.page_size} tokens, heads={self.heads}, "
                f"head_dim={self.head_dim}, format={self.fmt}")
