"""A page cache: the tensors behind w8a8_pages (include/gpt2_w8a8.h).

Sequences that go on from one prompt hold its pages once. ``ops.pages_extend``,
``pages_write``, ``pages_fork``, ``pages_free``, ``pages_compact`` and
``attention_pages`` take a ``PageCache``; a decode step of a batch is

    pos0 = ops.pages_extend(cache, n_new)                  # once a step
    ops.pages_write(cache, layer, K, V, pos0)              # each layer
    O = ops.attention_pages(Q, cache, layer, n_head, n_new=n_new, max_ctx=...,
                            shared_pages=prefix, n_shared=...)

with n_new 1 for the slots that go on and 0 for those that have ended, and
``prefix = cache.table[s].clone()`` of a slot s that holds the prompt, taken after
the fork and again after each ``pages_compact`` (the row itself is emptied when
the slot is freed). Sequences of several prompts: a call for each, with n_new 0
for the others' sequences, into one ``out``.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

HEAD_DIM = 64


class PageCache:
    """K, V [n_pages, n_layer, n_kv_head, page, 64] bf16 (pages may be strided),
    table [n_slot, max_pages], n_ctx [n_slot], refs [n_pages] int32."""

    __slots__ = ("K", "V", "table", "n_ctx", "refs", "device", "n_pages", "n_layer", "n_kv_head",
                 "page", "n_slot", "max_pages", "index", "c", "ref")

    def __init__(self, K: torch.Tensor, V: torch.Tensor, table: torch.Tensor,
                 n_ctx: torch.Tensor, refs: torch.Tensor):
        for name, t in (("K", K), ("V", V)):
            if t.dtype != torch.bfloat16:
                raise TypeError(f"{name}: expected {torch.bfloat16}, got {t.dtype}")
        for name, t in (("table", table), ("n_ctx", n_ctx), ("refs", refs)):
            if t.dtype != torch.int32:
                raise TypeError(f"{name}: expected {torch.int32}, got {t.dtype}")
            if not t.is_contiguous():
                raise ValueError(f"{name}: expected a contiguous tensor")
        if K.dim() != 5 or K.shape != V.shape or K.shape[4] != HEAD_DIM or K.shape[0] == 0:
            raise ValueError("K, V: expected [n_pages, n_layer, n_kv_head, page, 64] each")
        if K.stride() != V.stride() or not K[0].is_contiguous():
            raise ValueError("K, V: expected contiguous pages, equally strided")
        self.n_pages, self.n_layer, self.n_kv_head, self.page = K.shape[:4]
        if table.dim() != 2 or n_ctx.shape != table.shape[:1] or refs.shape != K.shape[:1]:
            raise ValueError("expected table [n_slot, max_pages], n_ctx [n_slot], refs [n_pages]")
        if any(t.device != K.device for t in (V, table, n_ctx, refs)):
            raise ValueError("the cache's tensors are on different devices")
        self.n_slot, self.max_pages = table.shape
        self.device = K.device
        self.index = K.get_device()  # -1: not on a GPU
        self.K, self.V, self.table, self.n_ctx, self.refs = K, V, table, n_ctx, refs
        self.c = _lib.Pages(K.data_ptr(), V.data_ptr(),
                            K.stride(0) if self.n_pages > 1 else K[0].numel(), self.n_pages,
                            self.page, self.n_layer, self.n_kv_head, table.data_ptr(),
                            self.max_pages, self.n_slot, n_ctx.data_ptr(), refs.data_ptr())
        self.ref = ctypes.byref(self.c)  # w8a8_pages *

    @classmethod
    def empty(cls, n_pages: int, n_slot: int, max_pages: int, n_layer: int, n_kv_head: int,
              page: int = 32, device="cuda") -> "PageCache":
        """An empty cache; max_pages bounds the pages of one sequence."""
        pool = torch.empty((2, n_pages, n_layer, n_kv_head, page, HEAD_DIM),
                           dtype=torch.bfloat16, device=device)
        i32 = dict(dtype=torch.int32, device=device)
        return cls(pool[0], pool[1], torch.full((n_slot, max_pages), -1, **i32),
                   torch.zeros(n_slot, **i32), torch.zeros(n_pages, **i32))
