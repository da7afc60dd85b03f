"""Paged key/value cache and the attention that reads it, over libfkmoe.so.

The reference's attention layer appends to one growing key and value tensor and scans it head by head
(src/fastkernels/kernels/triton/qwen36_attention.py:321-380, src/fastkernels/reference/qwen36_real.py:317-323); pages,
8-bit storage, windows and ragged batches have no counterpart there.

  paged_kv_append   writes new tokens into the cache, as they are or as e4m3 codes with one scale per token and head
  paged_kv_gather   reads the last tokens of each sequence back
  paged_attention   attention of new tokens (one per sequence in decode, chunks in a prompt) over the cache
  PagedKVCache      one layer's cache with its pages handed out, calling the three

Cache tensors are `[pages, kv_heads, page_size, head_dim]`, any strides with a contiguous last dimension (a cache laid
out `[pages, page_size, kv_heads, head_dim]` is passed as `.transpose(1, 2)`).  The three functions take the same ragged
description: `page_table` int32 `[seqs, max_pages]`, `lengths` int32 `[seqs]` counting the new tokens, `query_starts`
int32 `[seqs + 1]`: rows `query_starts[s] .. query_starts[s+1]-1` of a call are the last tokens of sequence `s`
(`None`: one token per sequence).  All of it is read on the device; nothing synchronises, so calls can be captured in a
CUDA graph and replayed with other lengths.  Page numbers outside the cache (-1 for a page that was given back, say)
are safe: such tokens are skipped, read as zeros, or not visible.  A position must not be mapped to a page that another
position of the same call writes.  Writing and reading back take caches of at most 1024 heads.  No gradients.
"""

from __future__ import annotations

import ctypes as C
import math
import struct
from collections import deque
from typing import Any, Optional

import torch

from . import _lib
from ._lib import AttentionCall, KvCache, KvRows
from .moe import _DTYPES

_CACHE_DTYPES = {**_DTYPES, torch.float8_e4m3fn: _lib.FK_E4M3}
_E4M3 = torch.float8_e4m3fn

# The ABI's structs are filled with one pack each (setting their fields one by one costs more than the checks); the formats
# are the fields of _lib.KvCache, KvRows and AttentionCall in order, without padding.
_CACHE_FIELDS = "8i13q6Q"
_ROW_FIELDS = "2Q4i4qQ"
_CALL_FIELDS = "2Q4i4qQf3iIi2Q"
_PACK_CACHE, _PACK_ROWS, _PACK_CALL = (struct.Struct("=" + f) for f in (_CACHE_FIELDS, _ROW_FIELDS, _CALL_FIELDS))
_CACHE_BYTES = C.sizeof(KvCache)
_FP32_MAX = torch.finfo(torch.float32).max
assert (_PACK_CACHE.size, _PACK_ROWS.size, _PACK_CALL.size) == (_CACHE_BYTES, C.sizeof(KvRows), C.sizeof(AttentionCall) - _CACHE_BYTES)


def _stream(device: torch.device) -> int:
    """The device's current stream, as the ABI takes it."""
    return torch._C._cuda_getCurrentRawStream(device.index)


class _On:
    """Makes `device` the current one for a launch, at no cost where it is already (torch.cuda.device costs microseconds)."""

    __slots__ = ("index", "before")

    def __init__(self, device: torch.device):
        self.index = device.index

    def __enter__(self):
        self.before = torch._C._cuda_getDevice()
        if self.before != self.index:
            torch._C._cuda_setDevice(self.index)

    def __exit__(self, *exc):
        if self.before != self.index:
            torch._C._cuda_setDevice(self.before)


def _check_index(t: Any, what: str, shape: tuple, device: torch.device) -> None:
    if t.dtype != torch.int32 or t.shape != shape:
        raise ValueError(f"{what} must be int32 with shape {list(shape)}, got {t.dtype} {list(t.shape)}")
    if t.device != device:
        raise ValueError(f"{what} must be on {device}")
    if t.stride(-1) != 1 and shape[-1] > 1:
        raise ValueError(f"{what} must be contiguous in its last dimension")


def _pack_cache(into: Any, key_cache, value_cache, page_table, lengths, query_starts, key_scale, value_scale) -> tuple:
    """Checks the description of a cache and a ragged batch and writes it to the front of a struct of the ABI; returns
    (kv_heads, head_dim, seqs)."""
    if not key_cache.is_cuda:
        raise ValueError("key_cache must be a CUDA tensor")
    shape, device, dtype = key_cache.shape, key_cache.device, key_cache.dtype
    if len(shape) != 4 or value_cache.shape != shape:
        raise ValueError("key_cache and value_cache must have the same shape [pages, kv_heads, page_size, head_dim]")
    if value_cache.device != device or value_cache.dtype != dtype:
        raise ValueError("key_cache and value_cache must have the same dtype and device")
    code = _CACHE_DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"the cache must be float32, bfloat16, float16 or float8_e4m3fn, got {dtype}")
    pages, heads, page_size, dim = shape
    if pages < 1 or heads < 1 or page_size < 1:
        raise ValueError("the cache must have at least one page, head and row per page")
    if dim < 1 or dim > _lib.MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be between 1 and {_lib.MAX_HEAD_DIM}")
    k0, k1, k2, k3 = key_cache.stride()
    v0, v1, v2, v3 = value_cache.stride()
    if dim > 1 and (k3 != 1 or v3 != 1):
        raise ValueError("key_cache and value_cache must be contiguous in their last dimension")
    if page_table.ndim != 2:
        raise ValueError("page_table must have shape [seqs, max_pages]")
    seqs, max_pages = table_shape = page_table.shape
    _check_index(page_table, "page_table", table_shape, device)
    _check_index(lengths, "lengths", (seqs,), device)
    if max_pages * page_size >= (1 << 31) - 1024:
        raise ValueError("page_table must hold less than 2^31 - 1024 positions per sequence")
    if query_starts is not None:
        _check_index(query_starts, "query_starts", (seqs + 1,), device)
    if dtype == _E4M3:
        for name, t in (("key_scale", key_scale), ("value_scale", value_scale)):
            if t is None:
                raise ValueError(f"{name} is required with a float8_e4m3fn cache")
            if t.dtype != torch.float32 or t.shape != shape[:3] or t.device != device:
                raise ValueError(f"{name} must be float32 [pages, kv_heads, page_size] on the cache's device")
        scales = (*key_scale.stride(), *value_scale.stride())
        scale_at = key_scale.data_ptr(), value_scale.data_ptr()
    else:
        if key_scale is not None or value_scale is not None:
            raise ValueError("key_scale and value_scale belong to a float8_e4m3fn cache")
        scales, scale_at = (0, 0, 0, 0, 0, 0), (0, 0)
    _PACK_CACHE.pack_into(into, 0, pages, heads, page_size, dim, code, seqs, max_pages, 0, page_table.stride(0), k0, k1, k2, v0, v1, v2, *scales,
                          key_cache.data_ptr(), value_cache.data_ptr(), *scale_at, page_table.data_ptr(), lengths.data_ptr())
    return heads, dim, seqs


def _check_rows(t: Any, what: str, rows: int, heads: int, dim: int, key_cache) -> int:
    """Checks `[rows, heads, dim]` rows of a call against the cache; returns the code of their dtype."""
    if t.shape != (rows, heads, dim):
        raise ValueError(f"{what} must have shape [{rows}, {heads}, {dim}], got {list(t.shape)}")
    if t.device != key_cache.device:
        raise ValueError(f"{what} must be on the cache's device")
    dtype = t.dtype
    code = _DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"{what} must be float32, bfloat16 or float16, got {dtype}")
    if dtype != key_cache.dtype and key_cache.dtype != _E4M3:
        raise ValueError(f"{what} must have the cache's dtype {key_cache.dtype}, got {dtype}")
    if dim > 1 and t.stride(2) != 1:
        raise ValueError(f"{what} must be contiguous in its last dimension")
    return code


def _check_heads(heads: int) -> None:
    if heads > _lib.MAX_KV_HEADS:
        raise ValueError(f"the cache must have at most {_lib.MAX_KV_HEADS} heads to be written or read back")


def _check_written(a: Any, b: Any, what: str) -> None:
    """Refuses tensors to be written whose elements share memory (expanded ones): several threads would write to one place."""
    for t in (a, b):
        if 0 in t.stride() and any(stride == 0 and n > 1 for n, stride in zip(t.shape, t.stride())):
            raise ValueError(f"{what} must not be expanded: every element needs a place of its own")


def _span(t: Any) -> tuple[int, int]:
    """First and one-past-last byte that a tensor can touch."""
    if t.numel() == 0:
        return 0, 0
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _overlap(a: Any, b: Any) -> bool:
    """Whether two tensors may touch the same bytes: their spans meet, unless they are interleaved rows of one layout (equal
    strides, all of them multiples of the smallest, which holds a row of each)."""
    (a0, a1), (b0, b1) = _span(a), _span(b)
    if a0 >= b1 or b0 >= a1:
        return False
    if a.shape == b.shape and a.stride() == b.stride() and a.dtype == b.dtype and (b0 - a0) % a.element_size() == 0:
        steps = [s for n, s in zip(a.shape[:-1], a.stride()[:-1]) if n > 1]
        least, width = min(steps, default=0), a.shape[-1]
        if least > 0 and all(s % least == 0 for s in steps):
            shift = (b0 - a0) // a.element_size() % least
            return not width <= shift <= least - width
    return True


def _pack_rows(into: KvRows, key, value, code: int, query_starts, zero_rest: bool) -> None:
    k0, k1, _ = key.stride()
    v0, v1, _ = value.stride()
    _PACK_ROWS.pack_into(into, 0, key.data_ptr(), value.data_ptr(), code, key.shape[0], zero_rest, 0, k0, k1, v0, v1,
                         0 if query_starts is None else query_starts.data_ptr())


def paged_kv_append(key: Any, value: Any, key_cache: Any, value_cache: Any, page_table: Any, lengths: Any, query_starts: Any = None, *,
                    key_scale: Any = None, value_scale: Any = None) -> None:
    """Write `key` and `value` `[rows, kv_heads, head_dim]` into the cache: row `query_starts[s] + i` goes to position
    `lengths[s] - n_s + i` of sequence `s`, `n_s` its number of rows.

    A float8_e4m3fn cache keeps `value = code * scale` with one fp32 scale per token and head in `key_scale` / `value_scale`
    `[pages, kv_heads, page_size]`: scale = max(|x|, 2^-100) / 448, the code is the nearest one (ties to even) to
    x * 448 / max.  A row with an infinity or a NaN reads back as NaN.  Rows behind the last sequence are ignored.  `key` and `value` must not be views of the cache.
    """
    c, r = KvCache(), KvRows()
    heads, dim, _ = _pack_cache(c, key_cache, value_cache, page_table, lengths, query_starts, key_scale, value_scale)
    _check_heads(heads)
    rows = key.shape[0]
    code = _check_rows(key, "key", rows, heads, dim, key_cache)
    if code != _check_rows(value, "value", rows, heads, dim, key_cache):
        raise ValueError("key and value must have the same dtype")
    _check_written(key_cache, value_cache, "key_cache and value_cache")
    _pack_rows(r, key, value, code, query_starts, False)
    device = key_cache.device
    with _On(device):
        _lib.check(_lib.load().fk_kv_append(C.byref(c), C.byref(r), _stream(device)), "fk_kv_append")


def paged_kv_gather(key_cache: Any, value_cache: Any, page_table: Any, lengths: Any, query_starts: Any, rows: int, *,
                    key_scale: Any = None, value_scale: Any = None, dtype: Optional[torch.dtype] = None, out: Any = None):
    """Read the last tokens of each sequence back: `(key, value)` `[rows, kv_heads, head_dim]`, row `query_starts[s] + i`
    from position `lengths[s] - n_s + i`; the inverse of `paged_kv_append` with the same arguments.

    `dtype` is the result's type for a float8_e4m3fn cache (bfloat16 by default).  `out=(key, value)` receives the rows
    and keeps what it holds behind the last sequence; new tensors hold zeros there.
    """
    c, r = KvCache(), KvRows()
    heads, dim, _ = _pack_cache(c, key_cache, value_cache, page_table, lengths, query_starts, key_scale, value_scale)
    _check_heads(heads)
    if rows < 0:
        raise ValueError("rows must not be negative")
    if dtype is None:
        dtype = out[0].dtype if out is not None else torch.bfloat16 if key_cache.dtype == _E4M3 else key_cache.dtype
    device = key_cache.device
    with _On(device):
        if out is None:
            key = torch.empty((rows, heads, dim), device=device, dtype=dtype)
            value = torch.empty((rows, heads, dim), device=device, dtype=dtype)
        else:
            key, value = out
        code = _check_rows(key, "key" if out is None else "out[0]", rows, heads, dim, key_cache)
        _check_rows(value, "value" if out is None else "out[1]", rows, heads, dim, key_cache)
        if key.dtype != dtype or value.dtype != dtype:
            raise ValueError(f"out must have dtype {dtype}")
        _check_written(key, value, "out")
        if out is not None and (_overlap(key, value) or any(_overlap(a, b) for a in out for b in (key_cache, value_cache))):
            raise ValueError("out must not overlap the cache, nor its two tensors each other")
        _pack_rows(r, key, value, code, query_starts, out is None)
        _lib.check(_lib.load().fk_kv_gather(C.byref(c), C.byref(r), _stream(device)), "fk_kv_gather")
    return key, value


def paged_attention(query: Any, key_cache: Any, value_cache: Any, page_table: Any, lengths: Any, query_starts: Any = None, *,
                    scale: Optional[float] = None, window: int = 0, sinks: int = 0, key_scale: Any = None, value_scale: Any = None,
                    max_query: int = 0, out: Any = None, flags: int = 0):
    """softmax(scale * query . key) value for `query` `[rows, q_heads, head_dim]` over the cached keys and values.

    Row `query_starts[s] + i` is the token at position `p = lengths[s] - n_s + i` of sequence `s` (its own key and value are
    in the cache already); it sees positions `j <= p`, with `window > 0` only those with `j > p - window` or `j < sinks`.
    Query head `a` reads key/value head `a // (q_heads // kv_heads)`.  `scale` defaults to `head_dim ** -0.5`.

    Result `[rows, q_heads, head_dim]` in the query's dtype (`out` if given; it must not overlap the query or the cache).
    A row that sees nothing (or only scores of -infinity) gives zeros.  Rows behind the last sequence keep what `out`
    held; in a new tensor they are zero.  What masked positions hold, NaN included, has no influence on a row.
    `max_query`, the largest number of rows of one sequence if the caller knows it, only chooses between kernels.
    Sums and softmax statistics are fp32.  Softmax weights are rounded once before they multiply the values: to the query's
    16-bit type, or to fp16 beside a float8_e4m3fn cache (there times their value's scale, next to the largest such product
    that the row sees: 11 bits down to 2^-19 of it, nothing below 2^-30); float32 queries round nothing.
    """
    call = AttentionCall()
    kv_heads, dim, seqs = _pack_cache(call, key_cache, value_cache, page_table, lengths, query_starts, key_scale, value_scale)
    if query.ndim != 3 or query.shape[1] < 1 or query.shape[1] % kv_heads:
        raise ValueError("query must have shape [rows, q_heads, head_dim] with q_heads a multiple of the cache's kv_heads")
    rows, q_heads, _ = query.shape
    code = _check_rows(query, "query", rows, q_heads, dim, key_cache)
    if query_starts is None and rows > seqs:
        raise ValueError("query has more rows than there are sequences: query_starts is required")
    if window < 0 or sinks < 0 or max_query < 0:
        raise ValueError("window, sinks and max_query must not be negative")
    if sinks and not window:
        raise ValueError("sinks need a window: without one every earlier position is visible")
    if window >= 1 << 31 or sinks >= 1 << 31:
        raise ValueError("window and sinks must be below 2^31")
    if scale is None:
        scale = dim ** -0.5
    elif not abs(scale) * math.log2(math.e) <= _FP32_MAX:
        raise ValueError("scale must be finite, in fp32 and times log2(e)")
    device, fresh = query.device, out is None
    lib = _lib.load()
    with _On(device):
        if fresh:
            out = torch.empty_like(query, memory_format=torch.contiguous_format)
        else:
            if _check_rows(out, "out", rows, q_heads, dim, key_cache) != code:
                raise ValueError("out must have the query's dtype")
            _check_written(out, out, "out")
            if any(_overlap(out, t) for t in (query, key_cache, value_cache)):
                raise ValueError("out must not overlap the query or the cache")
        q0, q1, _ = query.stride()
        o0, o1, _ = out.stride()
        _PACK_CALL.pack_into(call, _CACHE_BYTES, query.data_ptr(), out.data_ptr(), code, rows, q_heads, 1 if query_starts is None else min(max_query, rows),
                             q0, q1, o0, o1, 0 if query_starts is None else query_starts.data_ptr(), scale, window, sinks, fresh, flags, 0, 0, 0)
        ref = C.byref(call)
        need = lib.fk_paged_attention_workspace_bytes(ref)
        if need:
            # a new workspace per call: the allocator orders its reuse with the stream, and gives captured calls their own
            ws = torch.empty(need, device=device, dtype=torch.uint8)
            call.workspace, call.workspace_bytes = ws.data_ptr(), need
        _lib.check(lib.fk_paged_attention(ref, _stream(device)), "fk_paged_attention")
    return out


_PAGES_AT_ONCE = 4096          # entries of the page table in one copy


class PagedKVCache:
    """One layer's paged cache for a fixed number of sequences, with the pages handed out as the sequences grow.

    `append` writes each sequence's new tokens and grows it, `attend` runs their attention, `read` returns whole
    sequences, `release` gives a sequence's pages back.  The lengths live on the host as well, so that growing a sequence
    needs no synchronisation; the page table and the lengths on the device are updated by asynchronous copies out of pinned
    memory on the current stream, in place.  What grows on the host cannot be captured in a graph (a replay would write to the
    same positions again): `append`, `read` and `release` are refused there, `attend` and the three functions are not.
    """

    def __init__(self, pages: int, kv_heads: int, head_dim: int, *, seqs: int = 1, page_size: int = 16,
                 dtype: torch.dtype = torch.bfloat16, device: Any = "cuda"):
        if dtype not in _CACHE_DTYPES:
            raise ValueError(f"the cache must be float32, bfloat16, float16 or float8_e4m3fn, got {dtype}")
        if min(pages, kv_heads, seqs, page_size) < 1 or not 1 <= head_dim <= _lib.MAX_HEAD_DIM:
            raise ValueError(f"pages, kv_heads, seqs and page_size must be positive, head_dim between 1 and {_lib.MAX_HEAD_DIM}")
        if pages * page_size >= (1 << 31) - 1024 or kv_heads > _lib.MAX_KV_HEADS:          # every append would be refused
            raise ValueError(f"the cache must hold less than 2^31 - 1024 positions, with at most {_lib.MAX_KV_HEADS} heads")
        shape = (pages, kv_heads, page_size, head_dim)
        self.key, self.value = (torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype) if dtype == torch.float8_e4m3fn
                                else torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        self.key_scale = self.value_scale = None
        if dtype == torch.float8_e4m3fn:
            self.key_scale, self.value_scale = (torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2))
        self.page_size, self.seqs = page_size, seqs
        self.host_lengths = [0] * seqs
        self._owned: list[list[int]] = [[] for _ in range(seqs)]
        self._free = list(range(pages - 1, -1, -1))
        self.page_table = torch.full((seqs, pages), -1, dtype=torch.int32, device=self.key.device)
        # lengths and starts next to each other: one copy brings both
        self._state = torch.zeros(2 * seqs + 1, dtype=torch.int32, device=self.key.device)
        self.lengths = self._state[:seqs]
        self._starts: Any = None
        self._new = [0] * seqs
        # some 32 appends of 64 pages, and never less than one of the largest copies
        self._ring = torch.zeros(max(32 * (96 + seqs + 1), 2 * _PAGES_AT_ONCE), dtype=torch.int64, pin_memory=self.key.is_cuda)
        self._ring_at, self._copies = 0, deque()

    def _scales(self) -> dict:
        return {"key_scale": self.key_scale, "value_scale": self.value_scale}

    def _to_device(self, values, dtype: torch.dtype, into: Any = None):
        """`values` on the device by a copy on the current stream that the host does not wait for.  They are put down in a ring of
        pinned words made once (pinning more while the device works would wait for it); only if the host is a whole ring ahead it waits for
        the oldest copy."""
        size = (len(values) * dtype.itemsize + 7) // 8
        if self._ring_at + size > self._ring.numel():            # back to the front, behind what the lap before left at the end
            while self._copies and self._copies[0][0] >= self._ring_at:
                self._copies.popleft()[1].synchronize()
            self._ring_at = 0
        first, last = self._ring_at, self._ring_at + size
        while self._copies and first <= self._copies[0][0] < last:
            self._copies.popleft()[1].synchronize()
        pinned = self._ring[first:last].view(dtype)[:len(values)]
        pinned.copy_(torch.tensor(values, dtype=dtype))
        self._ring_at = last
        out = torch.empty(len(values), dtype=dtype, device=self.key.device) if into is None else into
        out.copy_(pinned, non_blocking=True)
        over = torch.cuda.Event()
        over.record()
        self._copies.append((first, over))
        return out

    def _not_captured(self, what: str) -> None:
        if self.key.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"{what} changes or reads lengths on the host and cannot be captured in a graph")

    def _grow(self, new) -> None:
        need = [-(-(n + m) // self.page_size) - len(own) for n, m, own in zip(self.host_lengths, new, self._owned)]
        if sum(max(0, n) for n in need) > len(self._free):
            raise ValueError("the cache has no pages left for these tokens")
        at, pages, width = [], [], self.page_table.shape[1]
        for s, n in enumerate(need):
            if n > 0:
                got = [self._free.pop() for _ in range(n)]
                first = s * width + len(self._owned[s])
                at += range(first, first + n)
                pages += got
                self._owned[s] += got
        for i in range(0, len(pages), _PAGES_AT_ONCE):
            part = slice(i, i + _PAGES_AT_ONCE)
            self.page_table.view(-1).index_copy_(0, self._to_device(at[part], torch.int64), self._to_device(pages[part], torch.int32))
        self.host_lengths = [n + m for n, m in zip(self.host_lengths, new)]
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        self._to_device(self.host_lengths + starts, torch.int32, self._state)
        self._new, self._starts = new, self._state[self.seqs:]

    def append(self, key: Any, value: Any, new=None) -> None:
        """`key`, `value` `[rows, kv_heads, head_dim]`: `new[s]` rows for each sequence in turn (default: one each)."""
        self._not_captured("append")
        new = [1] * self.seqs if new is None else [int(n) for n in new]
        if len(new) != self.seqs or min(new) < 0 or sum(new) != key.shape[0]:
            raise ValueError("new must name each sequence's number of rows, with key's rows as their sum")
        # all refusals before the sequences grow: a refused call leaves the cache as it was
        if not self.key.is_cuda:
            raise ValueError("the cache must be on a CUDA device")
        code = _check_rows(key, "key", key.shape[0], self.key.shape[1], self.key.shape[3], self.key)
        if code != _check_rows(value, "value", key.shape[0], self.key.shape[1], self.key.shape[3], self.key):
            raise ValueError("key and value must have the same dtype")
        with _On(self.key.device):
            self._grow(new)
        paged_kv_append(key, value, self.key, self.value, self.page_table, self.lengths, self._starts, **self._scales())

    def attend(self, query: Any, *, scale: Optional[float] = None, window: int = 0, sinks: int = 0):
        """Attention of the rows that the last `append` wrote, `query` `[rows, q_heads, head_dim]`."""
        if self._starts is None or query.shape[0] != sum(self._new):
            raise ValueError("attend takes the rows of the last append")
        return paged_attention(query, self.key, self.value, self.page_table, self.lengths, self._starts, scale=scale, window=window,
                               sinks=sinks, max_query=max(self._new), **self._scales())

    def read(self, dtype: Optional[torch.dtype] = None):
        """Every sequence whole: `(key, value)` `[sum of lengths, kv_heads, head_dim]`, one sequence after the other."""
        self._not_captured("read")
        starts = [0]
        for n in self.host_lengths:
            starts.append(starts[-1] + n)
        with _On(self.key.device):
            at = self._to_device(starts, torch.int32)
        return paged_kv_gather(self.key, self.value, self.page_table, self.lengths, at, starts[-1], dtype=dtype, **self._scales())

    def release(self, seq: int) -> None:
        """Empty one sequence and give its pages back."""
        self._not_captured("release")
        self._free += reversed(self._owned[seq])
        self._owned[seq] = []
        self.host_lengths[seq] = 0
        self.page_table[seq].fill_(-1)
        self.lengths[seq].zero_()
        self._starts = None
