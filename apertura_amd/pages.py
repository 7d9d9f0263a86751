"""Torch-tensor front end of include/esda_pages.h: caches in pages, shared between sequences and kept
in order on the device.

The reference keeps one growing buffer per layer (ESKVCache.mm:64-109).  Tensors are torch CUDA (HIP)
tensors; torch is only the allocator and stream provider here.
"""
from __future__ import annotations

import ctypes

import torch

from ._lib import MAX_ENTRIES, MAX_POOLS, PageRowsDesc, Pages, Pool, check, check_int32, lib
from .decode import _same_device, _stream_ptr, _used_on


def _check_pool(name: str, pool: torch.Tensor, num_pages: int, page_rows: int) -> None:
    if pool.dtype != torch.bfloat16:
        raise ValueError(f"{name} must be bf16")
    if pool.dim() != 5 or pool.stride(4) != 1 or pool.stride(3) != pool.shape[4]:
        raise ValueError(f"{name} must be a [planes, pages, kv heads, page rows, head_dim] view with dense rows, got "
                         f"{tuple(pool.shape)} with strides {pool.stride()}")
    if pool.shape[1] != num_pages or pool.shape[3] != page_rows:
        raise ValueError(f"{name} has {pool.shape[1]} pages of {pool.shape[3]} rows; the cache has {num_pages} of {page_rows}")


def _pool(pool: torch.Tensor) -> Pool:
    planes, _, heads, _, dim = pool.shape
    check_int32(planes=planes, num_kv_heads=heads)
    return Pool(pool.data_ptr(), planes, heads, dim, 0, pool.stride(0), pool.stride(1), pool.stride(2))


def _int_list(name: str, t: torch.Tensor, index: int, n: int | None = None) -> int:
    """The entries of a list on device `index`."""
    if t.dtype is not torch.int32 or t.dim() != 1 or not t.is_contiguous() or t.get_device() != index:
        raise ValueError(f"{name} must be a contiguous int32 list on cuda:{index}")
    k = t.numel()
    if k > MAX_ENTRIES:
        raise ValueError(f"{name} names {k} slots; a call names at most {MAX_ENTRIES}")
    if n is not None and k != n:
        raise ValueError(f"{name} has {k} entries, the other lists {n}")
    return k


def _table_stride(table: torch.Tensor) -> int:
    if table.dtype != torch.int32 or table.dim() != 2 or (table.shape[1] > 1 and table.stride(1) != 1):
        raise ValueError("table must be int32 [slots, max_pages] with dense rows")
    return table.stride(0) if table.shape[0] > 1 else table.shape[1]


class CacheCalls:
    """What PagedCache and tree.LinearCache have in common: the description that their calls take, the streams
    they are launched on, and the accepted rows of a step of drafted tokens."""

    def _set_up(self, c: Pages, workspace: torch.Tensor | None) -> None:
        need = ctypes.c_size_t(0)
        L = lib()
        check(L.esda_pages_workspace_size(ctypes.byref(c), ctypes.byref(need)))
        if workspace is None:
            workspace = torch.zeros(need.value, dtype=torch.uint8, device=self.device)
        self.workspace = workspace
        c.workspace, c.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        self._cache, self._ref, self._lib = c, ctypes.byref(c), L
        self._streams = {torch._C._cuda_getCurrentRawStream(self._index)}  # ordered behind what was done here
        self._made = None
        if not torch.cuda.is_current_stream_capturing():
            self._made = torch.cuda.Event()
            self._made.record()

    def _stream(self, stream) -> int:
        """The launch's HIP stream; the cache has to be on the current device."""
        if torch._C._cuda_getDevice() != self._index:
            raise ValueError(f"the cache is on {self.device}; the current device is cuda:{torch.cuda.current_device()}")
        raw = torch._C._cuda_getCurrentRawStream(self._index) if stream is None else int(stream.cuda_stream)
        if raw not in self._streams:
            self._first_call_on(torch.cuda.current_stream() if stream is None else stream, raw)
        return raw

    def _first_call_on(self, stream, raw: int) -> None:
        """(Once a stream: a block of memory remembers the streams it is used on.)"""
        with torch.cuda.stream(stream):
            if torch.cuda.is_current_stream_capturing():
                return
        if self._made is not None:
            stream.wait_event(self._made)
        _used_on(stream, self.workspace, self.length, *self._lists)
        self._streams.add(raw)

    def commit(self, accept: torch.Tensor, count: torch.Tensor, stream=None) -> None:
        """The rows of the accepted nodes accept[s][:count[s]] (rising) of a step of drafted tokens become the
        slots' next rows (esda_tree_commit).  accept [slots, A], count [slots] int32."""
        S, A = accept.shape if accept.dim() == 2 else (-1, 0)
        if accept.dtype is not torch.int32 or S != self.slots or (A > 1 and accept.stride(1) != 1) or \
                accept.get_device() != self._index:
            raise ValueError(f"accept must be int32 [{self.slots}, most accepted] with dense rows on {self.device}")
        if count.dtype is not torch.int32 or count.dim() != 1 or count.numel() != S or not count.is_contiguous() or \
                count.get_device() != self._index:
            raise ValueError(f"count must be contiguous int32 [{self.slots}] on {self.device}")
        rc = self._lib.esda_tree_commit(self._ref, accept.data_ptr(), accept.stride(0) if S > 1 else A, A, count.data_ptr(),
                                        self._stream(stream))
        if rc:
            check(rc)
        _used_on(stream, accept, count)

    def left_out(self, stream=None) -> int:
        """What the calls left out since the last time (waits for the stream)."""
        self._stream(stream)
        return pages_status(self.workspace, stream)


class PagedCache(CacheCalls):
    """K / V rows of many sequences in pages (esda_pages).

    pools: bf16 views [planes, pages, kv heads, page rows, head_dim] that one table serves (a plane is
    the K or the V of a layer; layers of another head shape are another pool).  table [slots, most pages]
    int32 (-1: no page), length [slots] int32, refs [pages] int32: the table entries that hold each page
    (left out: counted here).  The tensors are the caller's and are changed in place; every method is
    launched on the current stream, or ``stream``, and reads nothing back (``left_out`` does).

    A workspace that is not given is cleared here, and references are counted, on the current stream.  The
    first call on another stream goes behind that, and the memory of workspace, table, lengths and
    references is not handed out again before that stream is through.  (A call that is being captured does
    neither: whoever replays the graph orders it and keeps the cache.)"""

    def __init__(self, pools: list[torch.Tensor], table: torch.Tensor, length: torch.Tensor,
                 refs: torch.Tensor | None = None, workspace: torch.Tensor | None = None):
        if not 1 <= len(pools) <= MAX_POOLS:
            raise ValueError(f"a cache has 1 .. {MAX_POOLS} pools")
        first = pools[0]
        if first.dim() != 5:
            raise ValueError("a pool is [planes, pages, kv heads, page rows, head_dim]")
        N, R = first.shape[1], first.shape[3]
        for i, p in enumerate(pools):
            _check_pool(f"pool {i}", p, N, R)
        stride = _table_stride(table)
        S, P = table.shape
        if length.dtype != torch.int32 or length.shape != (S,) or not length.is_contiguous():
            raise ValueError("length must be contiguous int32 [slots]")
        check_int32(num_pages=N, page_rows=R, slots=S, max_pages=P)
        if refs is None:
            _same_device({"table": table})
            held = ((table >= 0) & (table < N)).flatten()
            refs = torch.zeros(N, dtype=torch.int32, device=table.device)
            refs.index_add_(0, table.clamp(0, N - 1).flatten().long(), held.int())
        if refs.dtype != torch.int32 or refs.shape != (N,) or not refs.is_contiguous():
            raise ValueError("refs must be contiguous int32 [pages]")
        _same_device({**{f"pool {i}": p for i, p in enumerate(pools)}, "table": table, "length": length, "refs": refs,
                      "workspace": workspace})
        self.pools, self.table, self.length, self.refs = list(pools), table, length, refs
        self.slots, self.max_pages, self.num_pages, self.page_rows = S, P, N, R
        self.device, self._index = table.device, table.device.index
        c = Pages(num_pages=N, page_rows=R, slots=S, max_pages=P, table_stride=stride, table=table.data_ptr(),
                  refs=refs.data_ptr(), length=length.data_ptr(), num_pools=len(pools))
        for i, p in enumerate(pools):
            c.pools[i] = _pool(p)
        self._lists = (table, refs)
        self._set_up(c, workspace)

    @classmethod
    def empty(cls, pools: list[torch.Tensor], slots: int, max_pages: int) -> "PagedCache":
        """A cache of ``slots`` sequences of no rows over the pools' memory."""
        device = pools[0].device
        return cls(pools, torch.full((slots, max_pages), -1, dtype=torch.int32, device=device),
                   torch.zeros(slots, dtype=torch.int32, device=device))

    def reserve(self, slots: torch.Tensor, rows: torch.Tensor, stream=None) -> None:
        """Pages for rows up to rows[i] (exclusive) of slot slots[i]."""
        n = _int_list("slots", slots, self._index)
        _int_list("rows", rows, self._index, n)
        rc = self._lib.esda_pages_reserve(self._ref, slots.data_ptr(), rows.data_ptr(), n, self._stream(stream))
        if rc:
            check(rc)
        _used_on(stream, slots, rows)

    def free(self, slots: torch.Tensor, stream=None) -> None:
        """The slots give up their pages and hold no rows."""
        n = _int_list("slots", slots, self._index)
        rc = self._lib.esda_pages_free(self._ref, slots.data_ptr(), n, self._stream(stream))
        if rc:
            check(rc)
        _used_on(stream, slots)

    def fork(self, src: torch.Tensor, dst: torch.Tensor, rows: torch.Tensor | None = None, stream=None) -> None:
        """Slot dst[i] becomes the first rows[i] rows of slot src[i] (None: all of them)."""
        n = _int_list("src", src, self._index)
        _int_list("dst", dst, self._index, n)
        if rows is not None:
            _int_list("rows", rows, self._index, n)
        rc = self._lib.esda_pages_fork(self._ref, src.data_ptr(), dst.data_ptr(), None if rows is None else rows.data_ptr(), n,
                                       self._stream(stream))
        if rc:
            check(rc)
        _used_on(stream, src, dst, rows)

    def compact(self, stream=None) -> None:
        """The pages in use move to the front of the pools."""
        rc = self._lib.esda_pages_compact(self._ref, self._stream(stream))
        if rc:
            check(rc)


def pages_status(workspace: torch.Tensor, stream=None) -> int:
    """Reads (synchronously, so not in a capture) and clears the status word of a workspace of esda_pages.h or
    esda_tree.h."""
    n = ctypes.c_int32(0)
    _same_device({"workspace": workspace})
    check(lib().esda_pages_status(workspace.data_ptr(), ctypes.byref(n), _stream_ptr(stream)))
    return int(n.value)


def _rows_desc(pool: torch.Tensor, table: torch.Tensor, row0: torch.Tensor, rows: int, linear: torch.Tensor | None) -> PageRowsDesc:
    if pool.dim() != 5:
        raise ValueError("a pool is [planes, pages, kv heads, page rows, head_dim]")
    planes, N, heads, R, dim = pool.shape
    _check_pool("pool", pool, N, R)
    stride = _table_stride(table)
    B, P = table.shape
    if row0.dtype != torch.int32 or row0.shape != (B,) or not row0.is_contiguous():
        raise ValueError("row0 must be contiguous int32 [batch]")
    check_int32(rows=rows, num_pages=N, page_rows=R, batch=B, max_pages=P)
    if linear is not None:
        if linear.dtype != torch.bfloat16 or linear.shape != (planes, B, heads, rows, dim) or \
                (rows > 1 and linear.stride(3) != dim) or linear.stride(4) != 1:
            raise ValueError(f"linear rows must be bf16 {(planes, B, heads, rows, dim)} with dense rows, got "
                             f"{tuple(linear.shape)} with strides {linear.stride()}")
        s = linear.stride()[:3]
    else:
        s = (B * heads * rows * dim, heads * rows * dim, rows * dim)
    return PageRowsDesc(_pool(pool), N, R, B, P, stride, rows, 0, *s)


def pages_write(pool: torch.Tensor, table: torch.Tensor, row0: torch.Tensor, rows: torch.Tensor, stream=None) -> None:
    """rows [planes, B, kv heads, n, D] become rows row0[b] .. row0[b] + n - 1 of sequence b's pages (table
    [B, most pages]) in every plane of pool [planes, pages, kv heads, page rows, D]; those that lie in no
    page are not written."""
    if rows.dim() != 5:
        raise ValueError("rows must be [planes, batch, kv heads, n, head_dim]")
    d = _rows_desc(pool, table, row0, rows.shape[3], rows)
    _same_device({"pool": pool, "table": table, "row0": row0, "rows": rows})
    if rows.numel() == 0:
        return
    check(lib().esda_pages_write(ctypes.byref(d), table.data_ptr(), row0.data_ptr(), rows.data_ptr(), _stream_ptr(stream)))
    _used_on(stream, table, row0, rows)


def pages_read(pool: torch.Tensor, table: torch.Tensor, row0: torch.Tensor, n: int, out: torch.Tensor | None = None,
               stream=None) -> torch.Tensor:
    """Rows row0[b] .. row0[b] + n - 1 of sequence b's pages, [planes, B, kv heads, n, D] (pages_write's
    reverse); rows that lie in no page are 0."""
    if n < 0:
        raise ValueError("n must not be negative")
    d = _rows_desc(pool, table, row0, n, out)
    _same_device({"pool": pool, "table": table, "row0": row0, "out": out})
    if out is None:
        out = torch.empty((pool.shape[0], table.shape[0], pool.shape[2], n, pool.shape[4]), dtype=pool.dtype, device=pool.device)
    if out.numel() == 0:
        return out
    check(lib().esda_pages_read(ctypes.byref(d), table.data_ptr(), row0.data_ptr(), out.data_ptr(), _stream_ptr(stream)))
    _used_on(stream, table, row0, out)
    return out
