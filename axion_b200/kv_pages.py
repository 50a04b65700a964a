"""Page table of a paged KV cache whose sequences share pages (include/axkv.h, axkv_pages).

One :class:`KVPages` holds the block table and the reference counts of a cache
of any number of layers and moves page contents in every layer's pool: the
``pages`` of :class:`~axion_b200.paged_kv.PagedKVCache4`, or fp16 or fp32 pages
``[n_pages, n_kv_heads, 16, head_dim]`` that a caller of the C ABI names in an
``axkv_cache_t`` with this table (:class:`~axion_b200.paged_kv.PagedKVCache` has
a table of its own, which does not share pages).
Everything stays on the device: no call synchronizes or reads back, so serving
loops can capture them.  Threads may share a table on one stream: a call's
kernels are launched together.  Invalid entries and a pool without enough free pages
are reported in the device status word (``ops.status()``); such a reserve or
fork changes nothing.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from .paged_kv import _DeviceCalls


class KVPages(_DeviceCalls):
    page_size = 16
    _what = "KVPages"

    def __init__(self, pools: list[torch.Tensor], block_table: torch.Tensor,
                 ref_count: torch.Tensor):
        """`pools`: contiguous CUDA tensors [n_pages, ...] of one page size;
        `block_table` int32 [sequences, max_blocks], -1 where a row holds no
        page (a row's pages come first); `ref_count` int32 [n_pages], the table
        entries that name each page.  The tensors are used as they are."""
        dev = block_table.device
        if not block_table.is_cuda:
            raise RuntimeError("KVPages: tensors must be CUDA tensors (axion_b200 has no CPU path)")
        if block_table.dtype != torch.int32 or block_table.dim() != 2 \
                or not block_table.is_contiguous() or block_table.numel() == 0:
            raise RuntimeError("KVPages: block_table must be contiguous int32 [sequences, max_blocks]")
        if ref_count.dtype != torch.int32 or ref_count.dim() != 1 or ref_count.device != dev \
                or not ref_count.is_contiguous() or ref_count.numel() == 0:
            raise RuntimeError("KVPages: ref_count must be contiguous int32 [n_pages] on the "
                               "table's device")
        n_pages = ref_count.shape[0]
        size = 0
        for t in pools:
            per = t.numel() // n_pages * t.element_size() if t.dim() else 0
            if t.device != dev or not t.is_contiguous() or t.dim() < 2 or t.shape[0] != n_pages \
                    or t.data_ptr() % 16 or per == 0 or per % 16 or per != (size or per):
                raise RuntimeError("KVPages: pools must be contiguous [n_pages, ...] tensors of one "
                                   "page size, a multiple of 16 bytes, on the table's device")
            size = per
        self.pools, self.block_table, self.ref_count = list(pools), block_table, ref_count
        self.max_seqs, self.max_blocks = block_table.shape
        self.n_pages = n_pages
        self._ptrs = torch.tensor([t.data_ptr() for t in pools], dtype=torch.int64).to(dev)
        self.c = _lib.axkv_pages_t(block_table.data_ptr(), ref_count.data_ptr(),
                                   self._ptrs.data_ptr(), size, len(pools), self.max_seqs,
                                   self.max_blocks, n_pages)
        self._ref = C.byref(self.c)
        self._set_device(block_table)
        self._lib = _lib.load()
        self._need = self._lib.axkv_pages_workspace(self._ref, 0)

    @classmethod
    def empty(cls, pools: list[torch.Tensor], max_seqs: int, max_blocks: int) -> "KVPages":
        """A table of empty sequences over pools whose pages are all free."""
        if not pools:
            raise RuntimeError("KVPages: at least one pool")
        dev = pools[0].device
        return cls(pools, torch.full((max_seqs, max_blocks), -1, dtype=torch.int32, device=dev),
                   torch.zeros(pools[0].shape[0], dtype=torch.int32, device=dev))

    def _list(self, *ts: torch.Tensor) -> tuple[int, list[int]]:
        """The common length of request tensors, and their addresses."""
        n = ts[0].shape[0] if ts[0].dim() == 1 else -1
        return n, [self._ints(t, n, "requests") for t in ts]

    def reserve(self, seqs: torch.Tensor, tokens: torch.Tensor) -> None:
        """Pages for tokens[i] tokens of sequence seqs[i] (each named once)."""
        n, at = self._list(seqs, tokens)
        self._call_ws(self._need + 4 * n, self._lib.axkv_pages_reserve, *at, n)

    def fork(self, parents: torch.Tensor, children: torch.Tensor, tokens: torch.Tensor) -> None:
        """Empty sequence children[i] becomes a copy of the first tokens[i]
        tokens of parents[i]: full pages shared, a partly filled one copied.
        Appending to either leaves the other as it is; writing again into a
        shared page (after taking a sequence back) does not."""
        n, at = self._list(parents, children, tokens)
        self._call_ws(self._need + 4 * n, self._lib.axkv_pages_fork, *at, n)

    def free(self, seqs: torch.Tensor) -> None:
        """Sequences give their pages up."""
        n, at = self._list(seqs)
        self._call_alone(self._lib.axkv_pages_free, *at, n)

    def compact(self) -> torch.Tensor:
        """Live pages to the front of every pool; their number (int32 [1])."""
        n = torch.empty(1, dtype=torch.int32, device=self._device)
        self._call_ws(self._need, self._lib.axkv_pages_compact, n.data_ptr())
        return n

    def copy(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Page src[i] to page dst[i] in every pool (no destination twice, none a source)."""
        n, at = self._list(src, dst)
        self._call_alone(self._lib.axkv_pages_copy, *at, n)
