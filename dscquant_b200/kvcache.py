"""The 4-bit paged key/value cache of one attention layer (no counterpart in the reference).

A page holds `page_size` tokens of every key head. The keys (and the values) of one token and head are one
row of head_dim 4-bit codes, two a byte (the even element in the low nibble), with a (step, low) pair of the
cache's type; element = code * step + low. `ops.kv4_append` writes rows, `ops.kv4_attention` attends to them,
`ops.kv4_read` gives their values back. Which pages belong to which sequence is the caller's: a page table
[sequences, pages] of int32 page ids.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch


@dataclass
class PagedKV4:
    k_codes: torch.Tensor   # [pages, kv_heads, page_size, head_dim / 2] u8
    k_affine: torch.Tensor  # [pages, kv_heads, page_size, 2] bf16 or f16: step, low
    v_codes: torch.Tensor
    v_affine: torch.Tensor

    def __post_init__(self) -> None:
        c, a = self.k_codes, self.k_affine
        shape = c.shape
        if len(shape) != 4 or shape[3] not in (32, 64):
            raise RuntimeError("codes must be [pages, kv_heads, page_size, head_dim / 2] with head_dim 64 or 128")
        ps = shape[2]
        if ps < 16 or ps > 1024 or ps & (ps - 1):
            raise RuntimeError("page_size must be a power of two from 16 to 1024")
        if a.dtype not in (torch.bfloat16, torch.float16):
            raise RuntimeError("affine must be bf16 or f16")
        pairs = (*shape[:3], 2)
        for t, want, dtype in ((c, shape, torch.uint8), (self.v_codes, shape, torch.uint8), (a, pairs, a.dtype),
                               (self.v_affine, pairs, a.dtype)):
            if t.shape != want or t.dtype != dtype:
                raise RuntimeError("codes must be uint8 and alike, affine [pages, kv_heads, page_size, 2] of one type")
            if not t.is_cuda or t.device != c.device or not t.is_contiguous():
                raise RuntimeError("the cache's tensors must be contiguous CUDA tensors on one device")

    @classmethod
    def allocate(cls, pages: int, kv_heads: int, head_dim: int, page_size: int = 64,
                 dtype: torch.dtype = torch.bfloat16, device="cuda") -> "PagedKV4":
        """An empty cache. What its slots hold before they are appended to is never read."""
        codes = [torch.empty((pages, kv_heads, page_size, head_dim // 2), dtype=torch.uint8, device=device)
                 for _ in range(2)]
        affine = [torch.empty((pages, kv_heads, page_size, 2), dtype=dtype, device=device) for _ in range(2)]
        return cls(codes[0], affine[0], codes[1], affine[1])

    @property
    def dtype(self) -> torch.dtype:
        return self.k_affine.dtype

    @property
    def device(self) -> torch.device:
        return self.k_codes.device

    @property
    def kv_heads(self) -> int:
        return self.k_codes.shape[1]

    @property
    def page_size(self) -> int:
        return self.k_codes.shape[2]

    @property
    def head_dim(self) -> int:
        return self.k_codes.shape[3] * 2

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k_codes, self.k_affine, self.v_codes, self.v_affine))
