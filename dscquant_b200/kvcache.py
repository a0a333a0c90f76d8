"""The 4-bit paged key/value cache of one attention layer (no counterpart in the reference).

A page holds `page_size` tokens of every key head. The keys (and the values) of one token and head are one
row of head_dim 4-bit codes, two a byte (the even element in the low nibble), with a (step, low) pair of the
cache's type; element = code * step + low. `ops.kv4_append` writes rows, `ops.kv4_attention` attends to them,
`ops.kv4_read` gives their values back. Which pages belong to which sequence is the caller's: a page table
[sequences, pages] of int32 page ids.
"""
from __future__ import annotations

import torch

from . import _lib

_TYPES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


class PagedKV4:
    """PagedKV4(k_codes, k_affine, v_codes, v_affine) over tensors in hand, or PagedKV4.allocate(...).

    codes [pages, kv_heads, page_size, head_dim / 2] uint8, affine [pages, kv_heads, page_size, 2] bf16 or f16
    (step, low). Checked once, here; the attributes cannot be set afterwards."""

    __slots__ = ("k_codes", "k_affine", "v_codes", "v_affine", "pages", "kv_heads", "page_size", "head_dim", "dtype",
                 "device", "index", "type_code")

    def __init__(self, k_codes: torch.Tensor, k_affine: torch.Tensor, v_codes: torch.Tensor,
                 v_affine: torch.Tensor) -> None:
        shape, dtype = k_codes.shape, k_affine.dtype
        if len(shape) != 4 or shape[3] not in (32, 64):
            raise RuntimeError("codes must be [pages, kv_heads, page_size, head_dim / 2] with head_dim 64 or 128")
        pages, heads, ps, half = shape
        if ps < 16 or ps > 1024 or ps & (ps - 1):
            raise RuntimeError("page_size must be a power of two from 16 to 1024")
        if dtype not in _TYPES:
            raise RuntimeError("affine must be bf16 or f16")
        if v_codes.shape != shape or not (k_affine.shape == v_affine.shape == (pages, heads, ps, 2)) or \
                k_codes.dtype is not torch.uint8 or v_codes.dtype is not torch.uint8 or v_affine.dtype is not dtype:
            raise RuntimeError("codes must be uint8 and alike, affine [pages, kv_heads, page_size, 2] of one type")
        if not (k_codes.is_cuda and k_codes.is_contiguous() and k_affine.is_contiguous() and
                v_codes.is_contiguous() and v_affine.is_contiguous() and
                k_codes.device == k_affine.device == v_codes.device == v_affine.device):
            raise RuntimeError("the cache's tensors must be contiguous CUDA tensors on one device")
        device = k_codes.device
        for name, value in zip(self.__slots__, (k_codes, k_affine, v_codes, v_affine, pages, heads, ps, half * 2,
                                                dtype, device, device.index, _TYPES[dtype])):
            object.__setattr__(self, name, value)

    def __setattr__(self, name: str, value) -> None:
        raise AttributeError("a PagedKV4 keeps the tensors it was made with")

    @classmethod
    def allocate(cls, pages: int, kv_heads: int, head_dim: int, page_size: int = 64,
                 dtype: torch.dtype = torch.bfloat16, device="cuda") -> "PagedKV4":
        """An empty cache. What its slots hold before they are appended to is never read."""
        codes = [torch.empty((pages, kv_heads, page_size, head_dim // 2), dtype=torch.uint8, device=device)
                 for _ in range(2)]
        affine = [torch.empty((pages, kv_heads, page_size, 2), dtype=dtype, device=device) for _ in range(2)]
        return cls(codes[0], affine[0], codes[1], affine[1])

    def nbytes(self) -> int:
        """Bytes of the cache's tensors: what a caller that sizes its page pool has to count."""
        return sum(t.numel() * t.element_size() for t in (self.k_codes, self.k_affine, self.v_codes, self.v_affine))
