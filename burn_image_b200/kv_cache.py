"""A paged, optionally quantised key/value cache and the attention that reads
it, over libbq4 (the ``bq4_cache_*`` calls of include/bq4.h).

The q/k/v projections leave k and v rows; ``KVCache.append`` quantises the
newest of them into the cache, ``KVCache.attention`` attends the newest query
tokens with what is cached, ``KVCache.prefix_attention`` does so for a batch
whose sequences share their first rows, and ``KVCache.read`` widens rows for a
consumer of contiguous k and v such as ``f16.attention``.

Sequences are given by two int32 tensors on the cache's device: a page table
[B, W] (position p of sequence b is row p % page_size of page
``page_table[b, p // page_size]``) and lengths [B], the rows that each
sequence holds, the newest included.  Nothing is copied to the host, so calls
can be captured into a CUDA graph and replayed with new tables and lengths in
the same tensors.  All arithmetic runs in the CUDA kernels; there is no CPU
fallback.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from . import _lib as L
from ._lib import Bq4Error, check

FORMATS = {"f16": L.CACHE_F16, "q8": L.CACHE_Q8, "q4": L.CACHE_Q4}
_DTYPES = {torch.float32: L.DTYPE_F32, torch.float16: L.DTYPE_F16}
_Strides = ctypes.c_int64 * 3
try:  # the handle alone: a tenth of the time that the Stream object takes
    from torch._C import _cuda_getCurrentRawStream as _raw_stream
except ImportError:
    def _raw_stream(index):
        return torch.cuda.current_stream(index).cuda_stream


class KVCache:
    """``pages`` pages of ``page_size`` tokens (a multiple of 16) for
    ``kv_heads`` heads of ``head_dim`` values (a multiple of 8, at most 128).
    format "f16": rows rounded to binary16; "q8": 8 bits a value and one scale
    a row; "q4": 4 bits a value and one scale for each 32 values (symmetric,
    q * scale, bf16 scales).  Which page holds what is the caller's business:
    the cache keeps no page table of its own."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, format: str = "q8",
                 device: Optional[torch.device] = None):
        if format not in FORMATS:
            raise Bq4Error(L.EINVAL_ARG, f"format {format!r} is not one of {', '.join(FORMATS)}")
        for what, size in (("pages", pages), ("page_size", page_size), ("kv_heads", kv_heads), ("head_dim", head_dim)):
            if not 0 < size < 2 ** 31:  # a ctypes field would keep its low bits
                raise Bq4Error(L.EINVAL_SHAPE, f"{what}={size} must be in [1, 2^31)")
        c = L.Cache(None, pages, page_size, kv_heads, head_dim, FORMATS[format], 0)
        n = ctypes.c_size_t()
        check(L.lib().bq4_cache_size(ctypes.byref(c), ctypes.byref(n)))
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        if dev.type != "cuda":
            raise Bq4Error(L.EINVAL_ARG, "a key/value cache lives on a CUDA device")
        if dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        self.pages, self.page_size, self.format = pages, page_size, format
        self.kv_heads, self.head_dim = kv_heads, head_dim
        self.device, self._index = dev, dev.index
        self.data = torch.zeros(n.value, dtype=torch.uint8, device=dev)
        c.data, c.device = self.data.data_ptr(), dev.index
        self._plans = {}       # of attention calls, by their sizes
        self._contiguous = {}  # strides of contiguous rows, by their shape
        self._lib = L.lib()
        self._c = c
        self._ref = ctypes.byref(c)

    @property
    def device_bytes(self) -> int:
        return self.data.numel()

    # The checks below run on every call of a decode loop: they take the common case first and
    # say what is wrong only when something is.

    def _sequences(self, page_table: torch.Tensor, lengths: torch.Tensor, batch: Optional[int] = None):
        if not (page_table.dtype is lengths.dtype is torch.int32 and page_table.device == self.device == lengths.device
                and page_table.dim() == 2 and lengths.dim() == 1):
            raise Bq4Error(L.EINVAL_ARG, f"page_table [B, W] and lengths [B] must be int32 on {self.device}")
        b, w = page_table.shape
        ts, ws = page_table.stride()
        n = lengths.shape[0]
        if (ws != 1 and w > 1) or (n > 1 and lengths.stride(0) != 1):
            raise Bq4Error(L.EINVAL_ARG, "page_table rows and lengths must have unit stride")
        if n != b or (batch is not None and batch != b):
            raise Bq4Error(L.EINVAL_SHAPE, f"page_table holds {b} sequences, lengths {n}"
                           + (f", the rows {batch}" if batch is not None else ""))
        return L.CacheSequences(page_table.data_ptr(), ts, w, lengths.data_ptr(), b)

    def _ints(self, t: torch.Tensor, what: str) -> torch.Tensor:
        if t.dtype is not torch.int32 or t.device != self.device or t.dim() != 1 \
                or (t.shape[0] > 1 and t.stride(0) != 1):
            raise Bq4Error(L.EINVAL_ARG, f"{what} must be int32, one-dimensional and contiguous on {self.device}")
        return t

    def _rows(self, t: torch.Tensor, what: str, heads: Optional[int]) -> torch.Tensor:
        if t.dtype not in _DTYPES or t.device != self.device:
            raise Bq4Error(L.EINVAL_ARG, f"{what} must be float32 or float16 on {self.device}")
        shape = t.shape
        if len(shape) != 4 or shape[3] != self.head_dim or (heads is not None and shape[2] != heads):
            raise Bq4Error(L.EINVAL_SHAPE,
                           f"{what} must be [B, S, {heads or 'heads'}, {self.head_dim}], got {tuple(shape)}")
        return t if t.stride(3) == 1 or t.numel() == 0 else t.contiguous()

    def _strides(self, t: torch.Tensor):
        """The first three strides of a 4-D tensor; those of contiguous ones are made once a shape."""
        if not t.is_contiguous():
            return _Strides(*t.stride()[:3])
        shape = t.shape
        got = self._contiguous.get(shape)
        if got is None:
            if len(self._contiguous) >= 1024:
                self._contiguous.clear()
            got = self._contiguous[shape] = _Strides(*t.stride()[:3])
        return got

    def append(self, key: torch.Tensor, value: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor) -> None:
        """Quantise the newest rows of every sequence into the cache: key and
        value [B, S, kv_heads, head_dim] (float32 or float16, any strides; a
        view of the projection's output will do), row i of sequence b to
        position lengths[b] - S + i.  Positions below 0 are skipped, so a padded batch
        aligns its rows at their ends.  Sequences that share a page must not
        write the same row."""
        k = self._rows(key, "key", self.kv_heads)
        v = value
        if v.shape != k.shape or v.dtype is not k.dtype or v.device != self.device:
            raise Bq4Error(L.EINVAL_SHAPE, "key and value must have one shape and type, on one device")
        if v.stride(3) != 1 and v.numel():
            v = v.contiguous()
        seqs = self._sequences(page_table, lengths, k.shape[0])
        check(self._lib.bq4_cache_append(self._ref, ctypes.byref(seqs), k.data_ptr(), self._strides(k), v.data_ptr(),
                                         self._strides(v), _DTYPES[k.dtype], k.shape[1], _raw_stream(self._index)))

    def read(self, page_table: torch.Tensor, lengths: torch.Tensor, count: int,
             starts: Optional[torch.Tensor] = None,
             dtype: torch.dtype = torch.float16) -> Tuple[torch.Tensor, torch.Tensor]:
        """k and v [B, kv_heads, count, head_dim] of positions starts[b] + i
        (starts: int32 [B]; None reads from 0), q * scale rounded once to
        ``dtype`` (float16 or float32).  A position below 0 or behind the
        sequence's length reads as 0."""
        seqs = self._sequences(page_table, lengths)
        if dtype not in _DTYPES:
            raise Bq4Error(L.EINVAL_ARG, f"rows are read as float16 or float32, not {dtype}")
        if count < 0:
            raise Bq4Error(L.EINVAL_SHAPE, f"count={count}")
        if starts is not None and self._ints(starts, "starts").shape[0] != seqs.batch:
            raise Bq4Error(L.EINVAL_SHAPE, f"starts holds {starts.shape[0]} sequences, page_table {seqs.batch}")
        H, D = self.kv_heads, self.head_dim
        k = page_table.new_empty((seqs.batch, H, count, D), dtype=dtype)
        v = torch.empty_like(k)
        check(self._lib.bq4_cache_read(self._ref, ctypes.byref(seqs), starts.data_ptr() if starts is not None else None,
                                       count, k.data_ptr(), v.data_ptr(), self._strides(k),
                                       _DTYPES[dtype], _raw_stream(self._index)))
        return k, v

    def attention(self, query: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, causal: bool = True,
                  scale: Optional[float] = None, max_length: Optional[int] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """softmax(scale * q k^T) v of the newest query tokens over the cached
        rows: query float16 [B, S, q_heads, head_dim], query head h on kv head
        h // (q_heads // kv_heads).  causal: query i of sequence b sees
        positions below lengths[b] - S + i + 1, else every row.  A query that
        sees nothing gives 0.  Returns float16 [B, S, q_heads, head_dim].
        scale: positive; None: 1 / sqrt(head_dim).  max_length: a bound of the lengths
        known to the host, by which the work is planned (None: the page
        table's width, which costs time where it is far above the
        lengths)."""
        return self._attention(query, None, None, page_table, lengths, causal, scale, max_length, out)

    def prefix_attention(self, query: torch.Tensor, prefix_pages: torch.Tensor, prefix_length: torch.Tensor,
                         page_table: torch.Tensor, lengths: torch.Tensor, causal: bool = True,
                         scale: Optional[float] = None, max_length: Optional[int] = None,
                         out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``attention`` for a batch whose sequences begin with the same rows:
        every query sees the first prefix_length (int32 [1]) rows of the page
        list prefix_pages (int32 [W]), read once for the whole batch, and then
        its own sequence; page_table, lengths, causal and max_length are about
        the sequences' own rows."""
        self._ints(prefix_pages, "prefix_pages")
        if self._ints(prefix_length, "prefix_length").shape[0] != 1:
            raise Bq4Error(L.EINVAL_SHAPE, "prefix_length must hold one value")
        return self._attention(query, prefix_pages, prefix_length, page_table, lengths, causal, scale, max_length, out)

    def _attention(self, query, prefix_pages, prefix_length, page_table, lengths, causal, scale, max_length, out):
        q = self._rows(query, "query", None)
        if q.dtype is not torch.float16:
            raise Bq4Error(L.EINVAL_ARG, "query must be float16")
        # (the library takes a scale of 0 or less for the default)
        if scale is not None and not 0.0 < ctypes.c_float(scale).value < math.inf:
            raise Bq4Error(L.EINVAL_ARG, f"scale={scale} is not a positive float32 (None: 1 / sqrt(head_dim))")
        shape = q.shape
        seqs = self._sequences(page_table, lengths, shape[0])
        if out is None:
            out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
        elif out.shape != shape or out.dtype != torch.float16 or out.device != self.device or not out.is_contiguous():
            raise Bq4Error(L.EINVAL_ARG, f"out must be contiguous float16 {tuple(shape)} on {self.device}")
        width = prefix_pages.shape[0] if prefix_pages is not None else 0
        key = (shape, seqs.table_width, width, max_length)
        plan = self._plans.get(key) or self._plan(key)
        bound, nbytes = plan
        # a workspace of the call's own: calls on several streams, and graphs captured side by side, never share one
        ws = q.new_empty(nbytes // 2)
        tail = (q.data_ptr(), self._strides(q), shape[1], shape[2], causal, scale or 0.0,
                out.data_ptr(), ws.data_ptr(), nbytes, _raw_stream(self._index))
        if prefix_pages is None:
            check(self._lib.bq4_cache_attention(self._ref, ctypes.byref(seqs), bound, *tail))
        else:
            check(self._lib.bq4_cache_prefix_attention(self._ref, prefix_pages.data_ptr(), width,
                                                       prefix_length.data_ptr(), ctypes.byref(seqs), bound, *tail))
        return out

    def _plan(self, key):
        """Bound of the lengths and workspace bytes of an attention call of these sizes."""
        (B, S, Hq, D), table_width, width, max_length = key
        held = table_width * self.page_size
        longest = held if max_length is None else min(max_length, held)
        if longest < 0:
            raise Bq4Error(L.EINVAL_SHAPE, f"max_length={max_length}")
        bound = 0 if max_length is None else longest  # 0: none is known
        n = ctypes.c_size_t()
        check(self._lib.bq4_cache_attention_workspace_size(self._ref, B, S, Hq, bound or -held,
                                                           width * self.page_size, ctypes.byref(n)))
        if len(self._plans) >= 1024:
            self._plans.clear()
        plan = self._plans[key] = (bound, n.value)
        return plan
