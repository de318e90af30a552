"""A KV cache in pages, for takes that start from one prompt (no counterpart in the reference, whose takes hold a dense
cache each, app/engine.py:380-388).

The prompt's keys and values are computed and stored once; a take is a fork of the prompt's sequence, which shares its
whole pages and owns what comes behind them.  All state lives on the device, so a step's ``extend`` can be captured into a
graph and the host keeps no books.  The operations are those of kernels.py (page_free, page_fork, page_extend,
page_compact) on the cache's tensors.
"""
from __future__ import annotations

import torch

from . import kernels as K

__all__ = ["PagedCache"]


class PagedCache:
    """Pages of ``page`` slots for ``layers`` layers and ``seqs`` sequences of at most ``max_pages`` pages.

    kv [layers, 2, pages, kv_heads, page, head_dim] fp16 (keys, values); ref [pages] int32 owners of each page; table
    [seqs, max_pages] int32; length [seqs] int64 slots held; err [1] int32, what was refused since the last ``reset``
    (include/ecdecode.h lists the bits).  Calls on one cache must be ordered (one stream, or events between streams).
    Sequence numbers are int32 tensors on the cache's device, or sequences of ints, which are copied there (not under
    graph capture)."""

    def __init__(self, layers, seqs, pages, kv_heads, head_dim, max_pages=None, page=64, device="cuda"):
        dev = torch.device(device)
        if dev.type != "cuda":
            raise RuntimeError("PagedCache needs a ROCm GPU device")
        max_pages = pages if max_pages is None else int(max_pages)
        if min(layers, seqs, pages, kv_heads, page, max_pages) < 1 or head_dim < 8 or head_dim % 8 or page < 16 or page & (page - 1):
            raise ValueError("PagedCache: positive sizes, a head_dim in multiples of 8 and a page of 16, 32, 64, .. slots")
        if seqs > 1024:
            raise ValueError("PagedCache: at most 1024 sequences")
        self.page = int(page)
        self.kv = torch.zeros(layers, 2, pages, kv_heads, page, head_dim, device=dev, dtype=torch.float16)
        self.dev = self.kv.device
        self.ref = torch.zeros(pages, device=dev, dtype=torch.int32)
        self.table = torch.full((seqs, max_pages), -1, device=dev, dtype=torch.int32)
        self.length = torch.zeros(seqs, device=dev, dtype=torch.int64)
        self.err = torch.zeros(1, device=dev, dtype=torch.int32)

    def layer(self, i):
        """(keys, values) of layer i, [pages, kv_heads, page, head_dim] each."""
        return self.kv[i, 0], self.kv[i, 1]

    def _ids(self, v):
        return v if isinstance(v, torch.Tensor) else torch.tensor(list(v), dtype=torch.int32, device=self.dev)

    def extend(self, pos):
        """Every sequence b holds slot pos[b] (int64 [seqs]) afterwards; -1 leaves it alone, and so does a slot it holds."""
        K.page_extend(self.ref, self.table, self.length, pos, self.page, self.err)

    def fork(self, src, dst):
        """Sequence dst[i], which holds nothing, becomes a copy of src[i]."""
        K.page_fork(self.kv, self.ref, self.table, self.length, self._ids(src), self._ids(dst), self.err)

    def free(self, seqs):
        """The sequences give their pages back."""
        K.page_free(self.ref, self.table, self.length, self._ids(seqs), self.page, self.err)

    def compact(self, pages):
        """The same sequences in a new cache of ``pages`` pages, the ones in use at its front; this one stays as it is.
        Bit 16 of this cache's error word (and an empty new cache) where they do not fit."""
        layers, _, _, heads, page, hd = self.kv.shape
        new = PagedCache(layers, self.table.shape[0], pages, heads, hd, self.table.shape[1], page, self.dev)
        K.page_compact(self.kv, self.ref, self.table, self.length, new.kv, new.ref, new.table, new.length, self.err)
        return new

    def error(self):
        """The error word (host sync)."""
        return int(self.err.item())

    def reset(self):
        """Every page free, every sequence empty, the error word 0."""
        self.ref.zero_()
        self.table.fill_(-1)
        self.length.zero_()
        self.err.zero_()

    @property
    def nbytes(self):
        return self.kv.numel() * 2
