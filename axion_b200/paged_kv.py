"""Paged KV cache over the C ABI of include/axkv.h, under the reference's names.

Mirrors PagedKVCache (inference/cpp/runtime/paged_kv.hpp:18-41, paged_kv.cpp):
``initialize(hidden, page)``, ``append(K, V)``, ``materialize_keys()``,
``materialize_values()``, for several sequences at once, plus the decode
attention over the cache (mha_attention_incremental, mha.cpp:227-285).  Pages
are fp16 (or fp32) per KV head, 16 tokens each, in device memory owned here;
sequence s owns pages s * max_blocks onwards (identity block table).
"""
from __future__ import annotations

import ctypes as C
import threading

import torch

from . import _lib
from ._lib import check


class PagedKVCache:
    page_size = 16

    def __init__(self, n_kv_heads: int, head_dim: int, max_seqs: int = 1, max_tokens: int = 4096,
                 kv_fp32: bool = False, device=None):
        self.n_kv_heads, self.head_dim = n_kv_heads, head_dim
        self.hidden_size = n_kv_heads * head_dim
        self.max_seqs = max_seqs
        self.max_blocks = (max_tokens + self.page_size - 1) // self.page_size
        dev = torch.device(device) if device is not None else torch.device("cuda")
        dt = torch.float32 if kv_fp32 else torch.float16
        n_pages = max_seqs * self.max_blocks
        shape = (n_pages, n_kv_heads, self.page_size, head_dim)
        self.k = torch.zeros(shape, dtype=dt, device=dev)
        self.v = torch.zeros(shape, dtype=dt, device=dev)
        self.block_table = torch.arange(n_pages, dtype=torch.int32, device=dev)
        self.used = [0] * max_seqs
        self.c = _lib.axkv_cache_t(self.k.data_ptr(), self.v.data_ptr(),
                                   self.block_table.data_ptr(), n_pages, self.max_blocks,
                                   n_kv_heads, head_dim, self.page_size, 1 if kv_fp32 else 0)
        self._ws = None
        self._lib = _lib.load()

    def initialize(self, hidden: int, page: int = 16) -> None:
        """PagedKVCache::initialize: empties the cache; hidden must be
        n_kv_heads * head_dim and page 16 (the device page)."""
        if hidden != self.hidden_size or page != self.page_size:
            raise RuntimeError(f"PagedKVCache: hidden {hidden} / page {page} do not match "
                               f"{self.hidden_size} / {self.page_size}")
        self.used = [0] * self.max_seqs

    def _stream(self) -> C.c_void_p:
        return C.c_void_p(torch.cuda.current_stream(self.k.device).cuda_stream)

    def append(self, K: torch.Tensor, V: torch.Tensor, seq: int = 0) -> None:
        """Append rows K, V [rows, hidden] (fp32, device) to sequence `seq`."""
        if K.shape != V.shape or K.dim() != 2 or K.shape[1] != self.hidden_size:
            raise RuntimeError("PagedKVCache::append: K and V must be [rows, hidden]")
        n = K.shape[0]
        if self.used[seq] + n > self.max_blocks * self.page_size:
            raise RuntimeError("PagedKVCache::append: sequence full")
        pos = torch.arange(self.used[seq], self.used[seq] + n, dtype=torch.int32,
                           device=self.k.device)
        sq = torch.full((n,), seq, dtype=torch.int32, device=self.k.device)
        Kc, Vc = K.float().contiguous(), V.float().contiguous()
        check(self._lib.axkv_paged_append(C.byref(self.c), C.c_void_p(Kc.data_ptr()),
                                          C.c_void_p(Vc.data_ptr()), n, C.c_void_p(sq.data_ptr()),
                                          C.c_void_p(pos.data_ptr()), self._stream()))
        self.used[seq] += n

    def _gather(self, pages: torch.Tensor, seq: int) -> torch.Tensor:
        n = self.used[seq]
        nb = (n + self.page_size - 1) // self.page_size
        p = pages[seq * self.max_blocks: seq * self.max_blocks + nb]      # [nb, kv, 16, hd]
        return p.permute(0, 2, 1, 3).reshape(nb * self.page_size, self.hidden_size)[:n].float()

    def materialize_keys(self, seq: int = 0) -> torch.Tensor:
        return self._gather(self.k, seq)

    def materialize_values(self, seq: int = 0) -> torch.Tensor:
        return self._gather(self.v, seq)

    def attention(self, q: torch.Tensor, n_heads: int) -> torch.Tensor:
        """Decode attention of one query row per sequence ([n_seq, n_heads *
        head_dim], fp32, device) over all its cached tokens."""
        n_seq = q.shape[0]
        qpos = torch.tensor([self.used[s] - 1 for s in range(n_seq)], dtype=torch.int32,
                            device=self.k.device)
        if min(self.used[:n_seq]) <= 0:
            raise RuntimeError("PagedKVCache: attention over an empty sequence")
        need = self._lib.axkv_decode_attn_workspace(C.byref(self.c), n_seq, n_heads)
        if need < 0:
            raise RuntimeError("PagedKVCache: unsupported attention shape")
        if self._ws is None or self._ws.numel() < need:
            self._ws = torch.zeros(need, dtype=torch.uint8, device=self.k.device)
        qc = q.float().contiguous()
        out = torch.empty_like(qc)
        check(self._lib.axkv_paged_decode_attn(C.byref(self.c), C.c_void_p(qc.data_ptr()), n_seq,
                                               n_heads, C.c_void_p(qpos.data_ptr()),
                                               C.c_void_p(out.data_ptr()),
                                               C.c_void_p(self._ws.data_ptr()), self._ws.numel(),
                                               self._stream()))
        return out

    def prefill_attention(self, q: torch.Tensor, n_heads: int, T: int, p0: int,
                          quantize: bool = False):
        """Causal attention (mha_attention, mha.cpp:126-198) of positions p0 ..
        p0 + T - 1 of every sequence: q rows [n_seq * T, n_heads * head_dim]
        (row s * T + t = sequence s, position p0 + t), their K/V already
        appended.  quantize: (xq int8 rows, dxT transposed block scales) for
        the next Q8_0 product instead of fp32 rows."""
        n_seq = q.shape[0] // T
        if n_seq * T != q.shape[0] or any(self.used[s] < p0 + T for s in range(n_seq)):
            raise RuntimeError("PagedKVCache: prefill rows must be appended first")
        qc = q.float().contiguous()
        dev = self.k.device
        if quantize:
            rows, width = qc.shape[0], n_heads * self.head_dim
            xq = torch.empty(rows, width, dtype=torch.int8, device=dev)
            dxT = torch.empty(width // 32, (rows + 3) // 4 * 4, dtype=torch.float32, device=dev)
            check(self._lib.axkv_paged_prefill_attn(
                C.byref(self.c), C.c_void_p(qc.data_ptr()), qc.shape[1], n_seq, T, p0, n_heads,
                None, C.c_void_p(xq.data_ptr()), C.c_void_p(dxT.data_ptr()), self._stream()))
            return xq, dxT
        out = torch.empty_like(qc)
        check(self._lib.axkv_paged_prefill_attn(C.byref(self.c), C.c_void_p(qc.data_ptr()),
                                                qc.shape[1], n_seq, T, p0, n_heads,
                                                C.c_void_p(out.data_ptr()), None, None,
                                                self._stream()))
        return out


class _DeviceCalls:
    """Argument checks and the current stream of the objects below.  A call takes
    a few microseconds on the device, so these stay off the slower torch paths."""

    _what = ""

    def _set_device(self, t: torch.Tensor) -> None:
        self._dev = t.get_device()
        self._device = t.device
        self._ws: dict[int, torch.Tensor] = {}
        self._lock = threading.Lock()

    def _ints(self, t: torch.Tensor | None, n: int, what: str) -> int | None:
        """The address of n contiguous int32 on the object's device (None stays)."""
        if t is None:
            return None
        if t.dtype is not torch.int32 or t.get_device() != self._dev or t.dim() != 1 \
                or t.shape[0] != n or not t.is_contiguous():
            raise RuntimeError(f"{self._what}: {what} must be contiguous int32 [{n}] on the "
                               "device of the object's tensors")
        return t.data_ptr()

    def _call(self, fn, *args) -> None:
        """fn(self._ref, *args, stream) on the object's device and its current stream."""
        stream = torch._C._cuda_getCurrentRawStream(self._dev)
        if torch._C._cuda_getDevice() == self._dev:
            rc = fn(self._ref, *args, stream)
        else:
            with torch.cuda.device(self._device):
                rc = fn(self._ref, *args, stream)
        if rc:
            check(rc)

    def _call_alone(self, fn, *args) -> None:
        """_call, not between the kernels of another thread's call."""
        with self._lock:
            self._call(fn, *args)

    def _call_ws(self, need: int, fn, *args) -> None:
        """_call with a workspace of `need` bytes: kept per stream, on which calls
        follow one another (the kernels of a call too: threads take turns); a
        captured graph's is its own."""
        if torch._C._cuda_getDevice() != self._dev:   # capture is asked of the current device
            with torch.cuda.device(self._device):
                return self._call_ws(need, fn, *args)
        if torch.cuda.is_current_stream_capturing():
            ws = torch.empty(need, dtype=torch.uint8, device=self._device)
            return self._call(fn, *args, ws.data_ptr(), need)
        key = torch._C._cuda_getCurrentRawStream(self._dev)
        with self._lock:
            ws = self._ws.get(key)
            if ws is None or ws.numel() < need:
                ws = self._ws[key] = torch.empty(need, dtype=torch.uint8, device=self._device)
            self._call(fn, *args, ws.data_ptr(), ws.numel())


class PagedKVCache4(_DeviceCalls):
    """The paged cache in 4 bits (include/axkv.h, axkv4_cache): K and V as 4-bit
    codes with a step and a zero point per token and 32 dims, 0.5625 byte per
    value, under the method names of :class:`PagedKVCache`.

    Without arguments of its own the cache is one layer of ``max_seqs``
    sequences with an identity block table.  ``pages`` (uint8 [n_pages,
    n_kv_heads, 18 * head_dim]) and ``block_table`` (int32 [sequences,
    max_blocks], -1: no page) make it a view of a caller's memory, e.g. one
    layer of a pool whose table a :class:`~axion_b200.kv_pages.KVPages`
    manages; sequences and positions are then named by the caller
    (``append_rows``, ``decode_attention``, ``chunk_attention``).

    Calls go to the current stream of the cache's device.  Each stream and each
    captured graph has a workspace of its own, so calls of one cache on several
    streams and replayed graphs may run at once.
    """

    page_size = 16
    _what = "PagedKVCache4"

    def __init__(self, n_kv_heads: int, head_dim: int, max_seqs: int = 1, max_tokens: int = 4096,
                 device=None, *, pages: torch.Tensor | None = None,
                 block_table: torch.Tensor | None = None):
        if head_dim not in (32, 64, 128):
            raise RuntimeError(f"PagedKVCache4: head_dim {head_dim} (32, 64, 128)")
        if n_kv_heads <= 0 or max_seqs <= 0 or max_tokens <= 0:
            raise RuntimeError("PagedKVCache4: sizes must be positive")
        self.n_kv_heads, self.head_dim = n_kv_heads, head_dim
        self.hidden_size = n_kv_heads * head_dim
        if (pages is None) != (block_table is None):
            raise RuntimeError("PagedKVCache4: pages and block_table come together")
        if pages is None:
            dev = torch.device(device) if device is not None else torch.device("cuda")
            blocks = (max_tokens + self.page_size - 1) // self.page_size
            pages = torch.zeros(max_seqs * blocks, n_kv_heads, 18 * head_dim, dtype=torch.uint8,
                                device=dev)
            block_table = torch.arange(max_seqs * blocks, dtype=torch.int32,
                                       device=dev).view(max_seqs, blocks)
        if not pages.is_cuda or block_table.device != pages.device:
            raise RuntimeError("PagedKVCache4: pages and block_table must be CUDA tensors of one "
                               "device (axion_b200 has no CPU path)")
        if (pages.dtype != torch.uint8 or pages.dim() != 3 or not pages.is_contiguous()
                or tuple(pages.shape[1:]) != (n_kv_heads, 18 * head_dim) or pages.shape[0] == 0):
            raise RuntimeError(f"PagedKVCache4: pages must be contiguous uint8 [n_pages, "
                               f"{n_kv_heads}, {18 * head_dim}]")
        if (block_table.dtype != torch.int32 or block_table.dim() != 2
                or not block_table.is_contiguous() or block_table.numel() == 0):
            raise RuntimeError("PagedKVCache4: block_table must be contiguous int32 [sequences, "
                               "max_blocks]")
        self.pages, self.block_table = pages, block_table
        self.max_seqs, self.max_blocks = block_table.shape
        self.used = [0] * self.max_seqs
        self.c = _lib.axkv4_cache_t(pages.data_ptr(), block_table.data_ptr(), self.max_seqs,
                                    self.max_blocks, pages.shape[0], n_kv_heads, head_dim,
                                    self.page_size)
        self._ref = C.byref(self.c)
        self._set_device(pages)
        self._need: dict[tuple, int] = {}
        self._lib = _lib.load()

    # -- arguments ---------------------------------------------------------------
    def _rows(self, t: torch.Tensor, width: int, what: str) -> torch.Tensor:
        """fp32 rows [n, width], 16-byte aligned, with a row pitch the kernels take."""
        if t.dim() != 2 or t.shape[1] != width or t.get_device() != self._dev:
            raise RuntimeError(f"PagedKVCache4: {what} must be [rows, {width}] on the cache's device")
        if t.dtype is not torch.float32:
            t = t.float()
        pitch, step = t.stride()
        if t.shape[0] and (step != 1 or pitch % 4 or pitch < width or t.data_ptr() % 16):
            t = t.clone(memory_format=torch.contiguous_format)
        return t

    def _out(self, out: torch.Tensor | None, q: torch.Tensor) -> torch.Tensor:
        if out is None:
            return q.new_empty(q.shape)
        if out.shape != q.shape or out.dtype != torch.float32 or out.get_device() != self._dev \
                or not out.is_contiguous() or out.data_ptr() % 16:
            raise RuntimeError("PagedKVCache4: out must be contiguous fp32 like q, 16-byte aligned")
        return out

    def _workspace(self, fn, *sizes: int) -> int:
        """Workspace bytes of a call of these sizes."""
        key = (fn.__name__, *sizes)
        need = self._need.get(key)
        if need is None:
            with torch.cuda.device(self._device):
                need = fn(self._ref, *sizes)
            if need < 0:
                raise RuntimeError(self._lib.axq8_last_error().decode(errors="replace")
                                   or "PagedKVCache4: unsupported attention shape")
            self._need[key] = need
        return need

    # -- rows of a caller's sequences ----------------------------------------------
    def append_rows(self, K: torch.Tensor, V: torch.Tensor, row_seq: torch.Tensor,
                    row_pos: torch.Tensor) -> None:
        """K, V rows [n, hidden] (fp32, device) to positions row_pos of sequences
        row_seq (int32 [n], device), no position twice."""
        K, V = self._rows(K, self.hidden_size, "K"), self._rows(V, self.hidden_size, "V")
        n = K.shape[0]
        if V.shape[0] != n:
            raise RuntimeError("PagedKVCache4: K and V must be [rows, hidden]")
        if n and K.stride(0) != V.stride(0):
            K, V = K.contiguous(), V.contiguous()
        self._call(self._lib.axkv4_append, K.data_ptr(), V.data_ptr(),
                   K.stride(0) if n else self.hidden_size, n, self._ints(row_seq, n, "row_seq"),
                   self._ints(row_pos, n, "row_pos"))

    def read_rows(self, row_seq: torch.Tensor, row_pos: torch.Tensor):
        """The values held at those positions: (K, V) fp32 [n, hidden]."""
        n = row_seq.shape[0]
        kv = torch.empty((2, n, self.hidden_size), dtype=torch.float32, device=self._device)
        k = kv.data_ptr()
        self._call(self._lib.axkv4_read, k, k + n * self.hidden_size * 4, self.hidden_size, n,
                   self._ints(row_seq, n, "row_seq"), self._ints(row_pos, n, "row_pos"))
        return kv.unbind()

    def decode_attention(self, q: torch.Tensor, n_heads: int, q_pos: torch.Tensor,
                         q_seq: torch.Tensor | None = None, out: torch.Tensor | None = None):
        """Attention of row r of q [n, n_heads * head_dim] (fp32, device), at
        position q_pos[r] of sequence q_seq[r] (None: sequence r), over tokens
        0 .. q_pos[r]; rows at negative positions give zeros."""
        q = self._rows(q, n_heads * self.head_dim, "q")
        n = q.shape[0]
        out = self._out(out, q)
        pos, seq = self._ints(q_pos, n, "q_pos"), self._ints(q_seq, n, "q_seq")
        if n:
            need = self._workspace(self._lib.axkv4_decode_attn_workspace, n, n_heads)
            self._call_ws(need, self._lib.axkv4_decode_attn, q.data_ptr(), q.stride(0), n, n_heads,
                          seq, pos, out.data_ptr())
        return out

    def chunk_attention(self, q: torch.Tensor, n_heads: int, q_start: torch.Tensor,
                        q_pos: torch.Tensor, max_rows: int, q_seq: torch.Tensor | None = None,
                        out: torch.Tensor | None = None):
        """Causal attention of ragged chunks: rows q_start[i] .. q_start[i + 1] - 1
        of q are sequence q_seq[i] (None: sequence i) at positions q_pos[i] and
        on, at most max_rows of them, their K and V appended.  Rows of no chunk
        are left as they are in `out` (unset where it is made here).  Single rows
        over long contexts are better off in decode_attention than beside a long
        prompt here: one kernel takes the whole call, by max_rows."""
        q = self._rows(q, n_heads * self.head_dim, "q")
        n, chunks = q.shape[0], q_pos.shape[0]
        out = self._out(out, q)
        start = self._ints(q_start, chunks + 1, "q_start")
        pos, seq = self._ints(q_pos, chunks, "q_pos"), self._ints(q_seq, chunks, "q_seq")
        if n and chunks and max_rows:
            need = self._workspace(self._lib.axkv4_chunk_attn_workspace, chunks, max_rows, n_heads)
            self._call_ws(need, self._lib.axkv4_chunk_attn, q.data_ptr(), q.stride(0), n, chunks,
                          max_rows, n_heads, seq, start, pos, out.data_ptr())
        return out

    # -- the reference's names, sequences filled from their start -------------------
    def initialize(self, hidden: int, page: int = 16) -> None:
        """PagedKVCache::initialize: empties the cache."""
        if hidden != self.hidden_size or page != self.page_size:
            raise RuntimeError(f"PagedKVCache: hidden {hidden} / page {page} do not match "
                               f"{self.hidden_size} / {self.page_size}")
        self.used = [0] * self.max_seqs

    def _span(self, seq: int, a: int, b: int):
        dev = self.pages.device
        return (torch.full((b - a,), seq, dtype=torch.int32, device=dev),
                torch.arange(a, b, dtype=torch.int32, device=dev))

    def append(self, K: torch.Tensor, V: torch.Tensor, seq: int = 0) -> None:
        """Append rows K, V [rows, hidden] (fp32, device) to sequence `seq`."""
        if K.shape != V.shape or K.dim() != 2 or K.shape[1] != self.hidden_size:
            raise RuntimeError("PagedKVCache::append: K and V must be [rows, hidden]")
        n = self.used[seq] + K.shape[0]
        if n > self.max_blocks * self.page_size:
            raise RuntimeError("PagedKVCache::append: sequence full")
        self.append_rows(K, V, *self._span(seq, self.used[seq], n))
        self.used[seq] = n

    def materialize_keys(self, seq: int = 0) -> torch.Tensor:
        return self.read_rows(*self._span(seq, 0, self.used[seq]))[0]

    def materialize_values(self, seq: int = 0) -> torch.Tensor:
        return self.read_rows(*self._span(seq, 0, self.used[seq]))[1]

    def attention(self, q: torch.Tensor, n_heads: int) -> torch.Tensor:
        """Decode attention of one query row per sequence over all its tokens."""
        if q.shape[0] > self.max_seqs or min(self.used[:q.shape[0]], default=1) <= 0:
            raise RuntimeError("PagedKVCache: attention over an empty sequence")
        pos = torch.tensor(self.used[:q.shape[0]], dtype=torch.int32, device=self.pages.device) - 1
        return self.decode_attention(q, n_heads, pos)

    def prefill_attention(self, q: torch.Tensor, n_heads: int, T: int, p0: int) -> torch.Tensor:
        """Causal attention of positions p0 .. p0 + T - 1 of every sequence (row
        s * T + t = sequence s, position p0 + t), their K/V already appended."""
        n_seq = q.shape[0] // T if T > 0 else 0
        if n_seq * T != q.shape[0] or n_seq > self.max_seqs \
                or any(self.used[s] < p0 + T for s in range(n_seq)):
            raise RuntimeError("PagedKVCache: prefill rows must be appended first")
        dev = self.pages.device
        return self.chunk_attention(
            q, n_heads, torch.arange(n_seq + 1, dtype=torch.int32, device=dev) * T,
            torch.full((n_seq,), p0, dtype=torch.int32, device=dev), T)
