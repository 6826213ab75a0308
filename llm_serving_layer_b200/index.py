"""
Page index of a paged-KV pool: int8 bounds of each page's keys per KV head,
which page-sparse attention scores pages with (``B200PagedBackend.plan_sparse``).

For a page whose keys have elementwise minimum ``lo`` and maximum ``hi``,
``scale = max(|lo|, |hi|) * (1/127)``, ``codes[0] = floor(lo / scale)`` and
``codes[1] = ceil(hi / scale)``. A page with a key that is no number has a NaN
scale and scores above every number; infinite bounds have an infinite scale and
the codes -127 / 127. An entry belongs to the physical block, so
sequences that share a page (radix prefix sharing) share its entry. Only entries
of completed pages are read (a query's own page is always attended), so nothing
is kept up to date token by token: the backend writes the entries of the pages
that a step completes, or of the blocks that it fills, after every ``append_kv``,
``append_attend``, ``rope_append``, ``copy_block(s)`` and swap-in while the index
lives. ``update`` and ``rebuild`` are for what is written past the backend (into
``k_pool`` itself, by the C entry points, by a CUDA graph captured before the
index was made) or before it existed.

The reference has no counterpart (its attention reads every page).
"""

from __future__ import annotations

import ctypes
import weakref
from typing import Any, Iterable

import torch

from . import _native as N

__all__ = ["PageIndex"]


class PageIndex:
    """Index of every page of ``backend``'s pool: ``codes`` int8
    ``[layers, blocks, kv heads, 2, head_dim]`` and ``scales`` fp32
    ``[layers, blocks, kv heads]`` on its device (1/31 of the pool's bytes for
    16-token fp16 pages). Fresh entries are zero."""

    def __init__(self, backend: Any):
        if backend.dtype not in (torch.float16, torch.bfloat16, torch.float32):
            raise ValueError(f"the page index takes fp16, bf16 or fp32 pools, not {backend.dtype}")
        if backend.head_dim > 256:
            raise ValueError(f"the page index takes head_dim up to 256, not {backend.head_dim}")
        self.backend = backend
        shape = (backend.num_layers, backend.num_blocks, backend.n_kv_heads)
        self.codes = torch.zeros((*shape, 2, backend.head_dim), dtype=torch.int8, device=backend.device)
        self.scales = torch.zeros(shape, dtype=torch.float32, device=backend.device)
        self._desc = N.PageIndexDesc(self.codes.data_ptr(), self.scales.data_ptr())
        self._pdesc = ctypes.byref(self._desc)
        # the backend's writers keep this index current until it is dropped
        backend._indexes.append(weakref.ref(self, backend._indexes.remove))

    def nbytes(self) -> int:
        return self.codes.numel() + 4 * self.scales.numel()

    def update(self, layer_idx: int, meta: Any) -> None:
        """Entries of the pages completed by the step ``meta`` describes, once
        layer ``layer_idx`` holds its keys (the backend's writers do this
        themselves)."""
        bk = self.backend
        bk._check_layer(layer_idx)
        if getattr(meta, "slot_mapping", None) is None:
            raise ValueError("PageIndex.update requires meta.slot_mapping")
        self._write(layer_idx, bk._i32(meta.slot_mapping))

    def _write(self, layer_idx: int, ids: torch.Tensor) -> None:
        """int32 ids on the device: the slots of a step in one layer, or blocks
        in every layer (``layer_idx`` -1)."""
        bk = self.backend
        with torch.cuda.device(bk.device):
            if layer_idx >= 0:
                N.check(bk._lib.pkv_page_index_update(bk._pdesc, self._pdesc, layer_idx, ids.data_ptr(), ids.numel(),
                                                      bk._status_ptr, N.raw_stream(bk._dev_index)), "PageIndex.update")
            else:
                N.check(bk._lib.pkv_page_index_rebuild(bk._pdesc, self._pdesc, ids.data_ptr(), ids.numel(),
                                                       bk._status_ptr, N.raw_stream(bk._dev_index)),
                        "PageIndex.rebuild")

    def rebuild(self, block_ids: Iterable[int] | torch.Tensor) -> None:
        """Entries of these blocks in every layer, from the pool: for blocks
        filled before the index was made, or past the backend. ``IndexError``
        for ids outside the pool."""
        bk = self.backend
        ids = torch.as_tensor(list(block_ids) if not isinstance(block_ids, torch.Tensor) else block_ids,
                              dtype=torch.int32).flatten()
        if ids.numel() == 0:
            return
        lo, hi = int(ids.min()), int(ids.max())
        if lo < 0 or hi >= bk.num_blocks:
            raise IndexError(f"rebuild: block ids outside [0, {bk.num_blocks})")
        self._write(-1, ids.to(bk.device))
