"""Page table of a paged KV cache whose sequences share pages (include/axkv.h, axkv_pages).

One :class:`KVPages` holds the block table and the reference counts of a cache
of any number of layers and moves page contents in every layer's pool: the
``k`` and ``v`` tensors of :class:`~axion_b200.paged_kv.PagedKVCache`-like fp16
or fp32 pages, or the ``pages`` of :class:`~axion_b200.paged_kv.PagedKVCache4`.
Everything stays on the device: no call synchronizes or reads back, so serving
loops can capture them.  Invalid entries and a pool without enough free pages
are reported in the device status word (``ops.status()``); such a reserve or
fork changes nothing.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import check
from .paged_kv import _on


class KVPages:
    page_size = 16

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
        self._lib = _lib.load()

    @classmethod
    def empty(cls, pools: list[torch.Tensor], max_seqs: int, max_blocks: int) -> "KVPages":
        """A table of empty sequences over pools whose pages are all free."""
        if not pools:
            raise RuntimeError("KVPages: at least one pool")
        dev = pools[0].device
        return cls(pools, torch.full((max_seqs, max_blocks), -1, dtype=torch.int32, device=dev),
                   torch.zeros(pools[0].shape[0], dtype=torch.int32, device=dev))

    def _ints(self, what: str, *ts: torch.Tensor) -> list[int]:
        n = ts[0].shape[0] if ts[0].dim() == 1 else -1
        for t in ts:
            if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != n \
                    or t.device != self.block_table.device or not t.is_contiguous():
                raise RuntimeError(f"KVPages: {what} must be contiguous int32 tensors of one length "
                                   "on the table's device")
        return [t.data_ptr() for t in ts]

    def _workspace(self, n: int) -> torch.Tensor:
        need = self._lib.axkv_pages_workspace(self._ref, n)
        return torch.empty(need, dtype=torch.uint8, device=self.block_table.device)

    def _stream(self) -> int:
        return torch.cuda.current_stream(self.block_table.device).cuda_stream

    def reserve(self, seqs: torch.Tensor, tokens: torch.Tensor) -> None:
        """Pages for tokens[i] tokens of sequence seqs[i] (each named once)."""
        s, t = self._ints("seqs and tokens", seqs, tokens)
        with _on(self.block_table.device):
            ws = self._workspace(seqs.shape[0])
            check(self._lib.axkv_pages_reserve(self._ref, s, t, seqs.shape[0], ws.data_ptr(),
                                               ws.numel(), self._stream()))

    def fork(self, parents: torch.Tensor, children: torch.Tensor, tokens: torch.Tensor) -> None:
        """Empty sequence children[i] becomes a copy of the first tokens[i]
        tokens of parents[i]: full pages shared, a partly filled one copied."""
        a, b, t = self._ints("parents, children and tokens", parents, children, tokens)
        with _on(self.block_table.device):
            ws = self._workspace(parents.shape[0])
            check(self._lib.axkv_pages_fork(self._ref, a, b, t, parents.shape[0], ws.data_ptr(),
                                            ws.numel(), self._stream()))

    def free(self, seqs: torch.Tensor) -> None:
        """Sequences give their pages up."""
        s, = self._ints("seqs", seqs)
        with _on(self.block_table.device):
            check(self._lib.axkv_pages_free(self._ref, s, seqs.shape[0], self._stream()))

    def compact(self) -> torch.Tensor:
        """Live pages to the front of every pool; their number (int32 [1])."""
        with _on(self.block_table.device):
            n = torch.empty(1, dtype=torch.int32, device=self.block_table.device)
            ws = self._workspace(0)
            check(self._lib.axkv_pages_compact(self._ref, n.data_ptr(), ws.data_ptr(), ws.numel(),
                                               self._stream()))
        return n

    def copy(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Page src[i] to page dst[i] in every pool (no destination twice, none a source)."""
        a, b = self._ints("src and dst", src, dst)
        with _on(self.block_table.device):
            check(self._lib.axkv_pages_copy(self._ref, a, b, src.shape[0], self._stream()))
