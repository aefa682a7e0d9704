"""Streamed global attention: frames arrive one after another.

``BlockCache`` holds the keys and values of what was seen, in 8 bits, in
pages of 64 tokens that a page table hands to the sequences.
"""
from __future__ import annotations

import torch

from . import ops


class BlockCache:
    """8-bit keys and values of ``heads`` key heads, ``pages`` pages of 64 tokens.

    ``kc`` / ``vc``: e4m3 codes (values transposed within a page), ``ks`` /
    ``vs``: the rows' powers of two, ``mean``: each page's mean key in bf16
    (``include/vasc_stream.h`` has the layout). ``ops.cache_write`` fills it,
    ``ops.cache_read`` / ``cache_select`` / ``cache_attn`` read it. Which pages
    belong to whom is the caller's page table. The cache starts as zeros.
    """

    def __init__(self, pages: int, heads: int, head_dim: int, device="cuda"):
        if pages < 1 or heads < 1:
            raise ValueError(f"a cache needs pages and heads, got {pages} and {heads}")
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim {head_dim} not built (64, 128)")
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("the block cache lives on a GPU (the HIP path has no CPU fallback)")
        self.pages, self.heads, self.head_dim = int(pages), int(heads), int(head_dim)
        u8 = dict(device=device, dtype=torch.uint8)
        page = ops.BLOCK_K
        self.kc = torch.zeros(pages, heads, page, head_dim, **u8)
        self.vc = torch.zeros(pages, heads, head_dim, page, **u8)
        self.ks = torch.zeros(pages, heads, page, **u8)
        self.vs = torch.zeros(pages, heads, page, **u8)
        self.mean = torch.zeros(pages, heads, head_dim, device=device, dtype=torch.bfloat16)

    @property
    def nbytes(self) -> int:
        """Bytes of device memory: 2 + 2/D bytes a value pair, and the means."""
        return sum(t.numel() * t.element_size() for t in (self.kc, self.vc, self.ks, self.vs, self.mean))
