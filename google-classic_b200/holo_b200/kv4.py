"""A paged KV cache held in 4 bits (include/holo_b200.h, holo_kv4), on torch
tensors.

The reference keeps one contiguous fp32 cache a model (src/ai/llm.c:1165-1177)
and serves one sequence.  Here many sequences share a pool of pages: their
tables name the pages, forks share them, and everything is decided on the
device.  The arithmetic is the library's (csrc/kv4_*.cu); work is enqueued on
torch's current stream.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import load
from .attention import DTYPES, LEGACY_STREAM, _device, _raw_stream, check, row_stride, stream_of

BLOCK = 16   # positions a block of a page
INT = torch.int32
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", None)   # absent from builds of torch without CUDA


class Kv4Desc(C.Structure):
    """holo_kv4."""
    _fields_ = [("n_layers", C.c_int), ("n_kv_heads", C.c_int), ("head_dim", C.c_int), ("page_tokens", C.c_int),
                ("n_pages", C.c_int), ("max_seqs", C.c_int), ("max_pages", C.c_int), ("pool", C.c_void_p),
                ("tables", C.c_void_p), ("lens", C.c_void_p), ("refs", C.c_void_p), ("work", C.c_void_p),
                ("stream", C.c_void_p)]


def _ints(t, what: str, shape):
    """t, an int32 tensor of `shape` (-1: any size)."""
    if (not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or not t.is_contiguous() or t.dim() != len(shape)
            or any(n not in (-1, m) for n, m in zip(shape, t.shape))):
        raise TypeError(f"{what} is a contiguous int32 tensor {tuple(shape)}")
    return t


class Kv4Cache:
    """The cache and its sequences.

    Either made empty, of n_pages pages for max_seqs sequences of up to
    max_pages pages each, or over tensors that the caller has: pool (uint8,
    n_layers x n_pages x n_kv_heads x page_tokens / 16 x 18 * head_dim), tables
    (int32 [max_seqs][max_pages]), lens (int32 [max_seqs]) and, for the calls
    that allocate or move pages, refs (int32 [n_pages]).

    Lists of sequences are int32 vectors on the device; seqs None is the
    first ones in order.  Calls return when they are enqueued.  What a kernel
    found wrong (no free page, an index out of range) is raised by check().

    Each stream has a workspace of its own, made with its first call, so that
    calls of several streams and threads may overlap where the cache's contents
    allow it (attention beside attention; a call that changes what another
    reads is ordered by the caller).  Calls that CUDA graphs capture share one
    more: a graph's calls on a cache follow one another, and so do the replays of
    its graphs."""

    def __init__(self, n_layers: int, n_kv_heads: int, head_dim: int, page_tokens: int = 64, n_pages: int = 0,
                 max_seqs: int = 0, max_pages: int = 0, pool=None, tables=None, lens=None, refs=None, device="cuda"):
        self.lib = load()
        blocks = page_tokens // BLOCK
        if pool is None:
            if tables is not None or lens is not None or refs is not None:
                raise TypeError("Kv4Cache: tables, lens and refs come with a pool")
            pool = torch.zeros(n_layers, n_pages, n_kv_heads, blocks, 18 * head_dim, dtype=torch.uint8, device=device)
            tables = torch.full((max_seqs, max_pages), -1, dtype=torch.int32, device=device)
            lens = torch.zeros(max_seqs, dtype=torch.int32, device=device)
            refs = torch.zeros(n_pages, dtype=torch.int32, device=device)
        if not isinstance(pool, torch.Tensor):
            raise TypeError("Kv4Cache: pool is a tensor")
        if pool.dtype != torch.uint8 or not pool.is_contiguous() or pool.dim() != 5 or (
                tuple(pool.shape[2:]) != (n_kv_heads, blocks, 18 * head_dim)) or pool.shape[0] != n_layers:
            raise TypeError(f"Kv4Cache: pool {tuple(pool.shape)} {pool.dtype}")
        _ints(tables, "Kv4Cache: tables", (-1, -1))
        _ints(lens, "Kv4Cache: lens", tables.shape[:1])
        if refs is not None:
            _ints(refs, "Kv4Cache: refs", (pool.shape[1],))
        for t in (tables, lens, refs):
            if t is not None and t.device != pool.device:
                raise ValueError(f"Kv4Cache: tensors on {pool.device} and {t.device}")
        self.pool, self.tables, self.lens, self.refs = pool, tables, lens, refs
        self.desc = d = Kv4Desc(n_layers, n_kv_heads, head_dim, page_tokens, pool.shape[1], tables.shape[0],
                                tables.shape[1], pool.data_ptr(), tables.data_ptr(), lens.data_ptr(),
                                None if refs is None else refs.data_ptr())
        self._heads = (n_kv_heads, head_dim)
        size = self.lib.cuda_kv4_work_bytes(C.addressof(d))
        if size == 0:
            raise ValueError("Kv4Cache: this shape is not supported (head_dim 64/128/256, page_tokens a multiple of 16)")
        self._index = pool.get_device()
        stream = stream_of(self._index)
        self.work = torch.zeros(2 * size, dtype=torch.uint8, device=pool.device)   # this stream's, and that of captured calls
        d.stream, d.work = stream, self.work.data_ptr()
        # stream: (address of its descriptor, the descriptor, its workspace), of calls that no graph captures
        self._of_stream = {stream: (C.addressof(d), d, self.work)}

    def _descriptor(self, stream: int):
        """(address, descriptor, workspace) for calls on `stream`, the current one."""
        d = Kv4Desc.from_buffer_copy(self.desc)
        d.stream, size = stream, self.work.numel() // 2
        if stream != LEGACY_STREAM and _capturing():
            d.work = self.work.data_ptr() + size
            return C.addressof(d), d, self.work
        work = torch.zeros(size, dtype=torch.uint8, device=self.pool.device)   # on this stream, so before its calls
        d.work = work.data_ptr()
        return self._of_stream.setdefault(stream, (C.addressof(d), d, work))

    def _call(self, what: str, fn, *args):
        index = self._index
        stream = (_raw_stream(index) or LEGACY_STREAM) if index == _device() else stream_of(index)   # (which raises)
        mine = self._of_stream.get(stream)
        if mine is None or (stream != LEGACY_STREAM and _capturing()):   # (the default stream cannot be captured)
            mine = self._descriptor(stream)
        rc = fn(mine[0], *args)
        if rc:
            check(rc, what)

    def _seqs(self, seqs, n=None):
        """(pointer, count) of a list of sequences."""
        if seqs is None:
            return None, self.desc.max_seqs if n is None else n
        if seqs.dtype != torch.int32 or seqs.dim() != 1 or not seqs.is_contiguous() or seqs.get_device() != self._index:
            raise TypeError("Kv4Cache: a list of sequences is a contiguous int32 vector on the cache's device")
        return seqs.data_ptr(), seqs.shape[0]

    def check(self):
        """Waits for the current stream's work and raises what a kernel found wrong."""
        torch.cuda.current_stream(self.pool.device).synchronize()
        check(self.lib.cuda_last_status(), "Kv4Cache")

    def extend(self, counts, seqs=None, start=None):
        """Room for counts[i] more positions of each sequence; returns start,
        their lengths before (-1 where there was no room)."""
        i, n = self._index, counts.numel()
        p, m = (None, n) if seqs is None else self._seqs(seqs)
        if start is None:
            start = torch.empty_like(counts)
        if m != n or start.numel() != n:
            raise ValueError("Kv4Cache.extend: one count and start a sequence")
        if counts.dtype != INT or start.dtype != INT or not counts.is_contiguous() or not start.is_contiguous():
            raise TypeError("Kv4Cache.extend: counts and start are contiguous int32 vectors")
        if counts.get_device() != i or start.get_device() != i:
            raise ValueError("Kv4Cache.extend: a tensor is not on the cache's device")
        self._call("cuda_kv4_extend", self.lib.cuda_kv4_extend, p, counts.data_ptr(), start.data_ptr(), n)
        return start

    def _rows(self, what, k, v, cu_rows, start, seqs):
        shape, n = k.shape, cu_rows.numel() - 1
        p, m = (None, n) if seqs is None else self._seqs(seqs)
        if shape != v.shape or len(shape) != 3 or shape[1:] != self._heads or m != n or start.numel() != n:
            raise ValueError(f"{what}: k {tuple(k.shape)}, v {tuple(v.shape)}, {n} sequences in cu_rows")
        dtype = k.dtype
        if dtype not in DTYPES or v.dtype != dtype:
            raise TypeError(f"{what}: k {k.dtype}, v {v.dtype}")
        if cu_rows.dtype != INT or start.dtype != INT or not cu_rows.is_contiguous() or not start.is_contiguous():
            raise TypeError(f"{what}: cu_rows and start are contiguous int32 vectors")
        i = self._index
        if k.get_device() != i or v.get_device() != i or cu_rows.get_device() != i or start.get_device() != i:
            raise ValueError(f"{what}: a tensor is not on the cache's device")
        k_row = 0 if k.is_contiguous() else row_stride(k, *self._heads, what)
        v_row = 0 if v.is_contiguous() else row_stride(v, *self._heads, what)
        return (k.data_ptr(), v.data_ptr(), DTYPES[dtype], k_row, v_row, shape[0], cu_rows.data_ptr(), start.data_ptr(), p, n)

    def append(self, layer: int, k, v, cu_rows, start, seqs=None):
        """Writes rows cu_rows[i] .. cu_rows[i + 1] of k and v [rows][n_kv_heads]
        [head_dim] (float32, float16 or bfloat16) to the positions from
        start[i] on of each sequence."""
        self._call("cuda_kv4_append", self.lib.cuda_kv4_append, layer,
                   *self._rows("Kv4Cache.append", k, v, cu_rows, start, seqs))

    def read(self, layer: int, cu_rows, start, k, v, seqs=None):
        """The same rows read back into k and v, which are returned."""
        self._call("cuda_kv4_read", self.lib.cuda_kv4_read, layer,
                   *self._rows("Kv4Cache.read", k, v, cu_rows, start, seqs))
        return k, v

    def attention(self, layer: int, q, out=None, seqs=None, scale: float = 0.0):
        """Attention of one query a sequence, q [n][n_heads][head_dim], over
        all the positions that it holds; out like q."""
        shape = q.shape
        n, n_heads, hd = shape
        p, m = (None, n) if seqs is None else self._seqs(seqs)
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        if m != n or hd != self._heads[1] or out.shape != shape:
            raise ValueError(f"Kv4Cache.attention: q {tuple(q.shape)}, out {tuple(out.shape)}, {m} sequences")
        dtype = q.dtype
        if dtype not in DTYPES or out.dtype != dtype:
            raise TypeError(f"Kv4Cache.attention: q {q.dtype}, out {out.dtype}")
        if q.get_device() != self._index or out.get_device() != self._index:
            raise ValueError("Kv4Cache.attention: a tensor is not on the cache's device")
        self._call("cuda_kv4_attention", self.lib.cuda_kv4_attention, layer, out.data_ptr(), q.data_ptr(),
                   DTYPES[dtype], row_stride(q, n_heads, hd, "Kv4Cache.attention: q"),
                   row_stride(out, n_heads, hd, "Kv4Cache.attention: out"), n_heads, scale, p, n)
        return out

    def fork(self, parents, children):
        """children[i], an empty sequence, becomes a copy of parents[i]: full
        pages are shared, a last page with room left is copied."""
        p, n = self._seqs(parents)
        k, m = self._seqs(children)
        if n != m:
            raise ValueError("Kv4Cache.fork: one child a parent")
        self._call("cuda_kv4_fork", self.lib.cuda_kv4_fork, p, k, n)

    def release(self, seqs):
        """Empties sequences; pages that no other one holds become free."""
        self._call("cuda_kv4_release", self.lib.cuda_kv4_release, *self._seqs(seqs))

    def compact(self):
        """Moves the pages in use to the front of the pool."""
        self._call("cuda_kv4_compact", self.lib.cuda_kv4_compact)

    def copy_pages(self, src, dst):
        """Copies pages src[i] to dst[i] in every layer."""
        p, n = self._seqs(src)
        k, m = self._seqs(dst)
        if n != m:
            raise ValueError("Kv4Cache.copy_pages: one target a source")
        self._call("cuda_kv4_copy_pages", self.lib.cuda_kv4_copy_pages, p, k, n)
