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
        self._kc = torch.zeros(pages, heads, page, head_dim, **u8)
        self._vc = torch.zeros(pages, heads, head_dim, page, **u8)
        self._ks = torch.zeros(pages, heads, page, **u8)
        self._vs = torch.zeros(pages, heads, page, **u8)
        self._mean = torch.zeros(pages, heads, head_dim, device=device, dtype=torch.bfloat16)
        self.device_index = self._kc.get_device()
        # the buffers stay where they are, so a call need not ask for their addresses again
        self.pointers = tuple(t.data_ptr() for t in (self._kc, self._vc, self._ks, self._vs))
        self.mean_pointer = self._mean.data_ptr()

    kc = property(lambda self: self._kc)
    vc = property(lambda self: self._vc)
    ks = property(lambda self: self._ks)
    vs = property(lambda self: self._vs)
    mean = property(lambda self: self._mean)

    @property
    def nbytes(self) -> int:
        """Bytes of device memory: 2 + 2/D bytes a value pair, and the means."""
        return sum(t.numel() * t.element_size() for t in (self.kc, self.vc, self.ks, self.vs, self.mean))
