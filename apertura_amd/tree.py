"""Torch-tensor front end of include/esda_tree.h: a step of drafted tokens, one behind another or as a
tree, over a cache in pages or a linear one.  One token a sequence is the decode step over pages.

The reference decodes one token of one sequence a step (ESAttention.mm:110-135).  Tensors are torch
CUDA (HIP) tensors; torch is only the allocator and stream provider here.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from ._lib import MAX_POOLS, Pages, TreeArgs, TreeDesc, check, check_int32, lib
from .decode import _dev_ptr, _on, _same_device, _stream_ptr, _used_on
from .pages import CacheCalls, _check_pool, _pool, _table_stride


@dataclass
class TreeStep:
    """Shapes of a step of drafted tokens (esda_tree_desc).  max_pages 0: linear caches, sequence b in
    page b, page_rows rows each."""

    batch: int
    nodes: int
    num_q_heads: int
    num_kv_heads: int
    head_dim: int
    num_pages: int
    page_rows: int
    max_pages: int = 0
    window: int = 0
    kv_shared: bool = False
    scale: float = 1.0
    split_rows: int = 0
    table_stride: int | None = None
    page_stride: int | None = None
    head_stride: int | None = None

    def desc(self) -> TreeDesc:
        hs = self.head_stride if self.head_stride is not None else self.page_rows * self.head_dim
        ps = self.page_stride if self.page_stride is not None else self.num_kv_heads * hs
        ts = self.table_stride if self.table_stride is not None else self.max_pages
        check_int32(batch=self.batch, nodes=self.nodes, num_q_heads=self.num_q_heads, num_kv_heads=self.num_kv_heads,
                    head_dim=self.head_dim, num_pages=self.num_pages, page_rows=self.page_rows, max_pages=self.max_pages,
                    window=self.window, split_rows=self.split_rows)
        return TreeDesc(self.batch, self.nodes, self.num_q_heads, self.num_kv_heads, self.head_dim, int(bool(self.kv_shared)),
                        self.window, self.num_pages, self.page_rows, self.max_pages, ts, ps, hs, self.split_rows,
                        self.scale)

    @classmethod
    def for_pages(cls, pages: torch.Tensor, table: torch.Tensor, num_q_heads: int, nodes: int, **kw) -> "TreeStep":
        """pages: a plane [pages, Hkv, page rows, D] of a pool; table: [B, most pages] int32."""
        if pages.dim() != 4 or pages.stride(3) != 1 or pages.stride(2) != pages.shape[3]:
            raise ValueError("pages must be a [pages, Hkv, page rows, D] view with dense rows")
        N, Hkv, R, D = pages.shape
        return cls(table.shape[0], nodes, num_q_heads, Hkv, D, N, R, table.shape[1], table_stride=_table_stride(table),
                   page_stride=pages.stride(0), head_stride=pages.stride(1), **kw)

    @classmethod
    def for_cache(cls, cache: torch.Tensor, num_q_heads: int, nodes: int, **kw) -> "TreeStep":
        """cache: linear rows [B, Hkv, cap, D]."""
        if cache.dim() != 4 or cache.stride(3) != 1 or cache.stride(2) != cache.shape[3]:
            raise ValueError("cache must be a [B, Hkv, cap, D] view with dense rows")
        B, Hkv, cap, D = cache.shape
        return cls(B, nodes, num_q_heads, Hkv, D, B, cap, page_stride=cache.stride(0), head_stride=cache.stride(1), **kw)


def tree_workspace_bytes(step: TreeStep) -> int:
    n, d = ctypes.c_size_t(0), step.desc()
    check(lib().esda_tree_workspace_size(ctypes.byref(d), ctypes.byref(n)))
    return int(n.value)


def new_tree_workspace(step: TreeStep, device) -> torch.Tensor:
    """Workspace for ``step``, its status word zeroed (pages_status reads it)."""
    n = tree_workspace_bytes(step)
    workspace = torch.empty(n, dtype=torch.uint8, device=device)
    workspace[:256].zero_()
    return workspace


class TreeCall:
    """A step of drafted tokens with its C-ABI arguments marshalled once (as DecodeCall): refill q, k_new,
    v_new, length, table and parent in place between calls.  Usable under HIP graph capture.

    q [B, nodes, Hq, D], k_new and v_new [B, nodes, Hkv, D]; k_pages, v_pages: planes [pages, Hkv, page
    rows, D] (linear: [B, Hkv, cap, D]); length [B] int32: committed rows; parent [B, nodes] int32 (None: a
    chain): -1 on the committed rows, j < i on node j, anything else no node.  A workspace that is not
    given is cleared here, on the current stream: calls on another one go behind that."""

    def __init__(self, step: TreeStep, q, k_new, v_new, k_pages, v_pages, length, table=None, parent=None, out=None,
                 workspace=None):
        d = step.desc()
        B, T, D = step.batch, step.nodes, step.head_dim
        if q.shape != (B, T, step.num_q_heads, D) or not q.is_contiguous():
            raise ValueError(f"q must be contiguous [B, nodes, Hq, D], got {tuple(q.shape)}")
        if k_new.shape != (B, T, step.num_kv_heads, D) or not k_new.is_contiguous():
            raise ValueError("k_new must be contiguous [B, nodes, Hkv, D]")
        if v_new is None and not step.kv_shared:
            raise ValueError("v_new is needed where V does not alias K")
        if v_new is not None and (v_new.shape != k_new.shape or not v_new.is_contiguous()):
            raise ValueError("v_new must be contiguous [B, nodes, Hkv, D]")
        if length.dtype != torch.int32 or length.shape != (B,) or not length.is_contiguous():
            raise ValueError("length must be contiguous int32 [B]")
        if parent is not None and (parent.dtype != torch.int32 or parent.shape != (B, T) or not parent.is_contiguous()):
            raise ValueError("parent must be contiguous int32 [B, nodes]")
        if (table is None) != (step.max_pages == 0):
            raise ValueError("a table goes with pages, and only with them")
        if table is not None and (table.dtype != torch.int32 or table.shape != (B, step.max_pages) or
                                  _table_stride(table) != d.table_stride):
            raise ValueError(f"table must be int32 {(B, step.max_pages)} with rows {d.table_stride} apart")
        vp = k_pages if (v_pages is None or step.kv_shared) else v_pages
        shape, strides = (step.num_pages, step.num_kv_heads, step.page_rows, D), (d.page_stride, d.head_stride, D, 1)
        for name, t in (("k_pages", k_pages), ("v_pages", vp)):
            if t.shape != shape or any(n > 1 and s != w for n, s, w in zip(shape, t.stride(), strides)):
                raise ValueError(f"{name} is {tuple(t.shape)} with strides {t.stride()}; the step describes {shape} with "
                                 f"strides {strides}")
        if out is None:
            out = torch.empty_like(q)
        if out.shape != q.shape or not out.is_contiguous():
            raise ValueError("out must be contiguous [B, nodes, Hq, D]")
        if workspace is None:
            workspace = new_tree_workspace(step, q.device)
        _same_device({"q": q, "k_new": k_new, "v_new": v_new, "k_pages": k_pages, "v_pages": vp, "length": length,
                      "table": table, "parent": parent, "out": out, "workspace": workspace})
        bf = torch.bfloat16
        self._keep = (q, k_new, v_new, k_pages, v_pages, length, table, parent)
        self.step, self.out, self.workspace = step, out, workspace
        self._desc, self._index = d, q.device.index
        self._args = TreeArgs(_dev_ptr(q, bf), _dev_ptr(k_new, bf), None if step.kv_shared else _dev_ptr(v_new, bf),
                              _dev_ptr(k_pages, bf), _dev_ptr(vp, bf), _dev_ptr(table), _dev_ptr(length), _dev_ptr(parent),
                              _dev_ptr(out, bf), _dev_ptr(workspace), workspace.numel() * workspace.element_size())
        self._fn = lib().esda_tree_decode
        self._pd, self._pa = ctypes.byref(self._desc), ctypes.byref(self._args)

    def __call__(self, stream=None) -> torch.Tensor:
        if torch._C._cuda_getDevice() != self._index:
            raise ValueError(f"the step's tensors are on cuda:{self._index}; the current device is another")
        rc = self._fn(self._pd, self._pa, _stream_ptr(stream))
        if rc:
            check(rc)
        return self.out


def tree_decode(step: TreeStep, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor | None, k_pages: torch.Tensor,
                v_pages: torch.Tensor | None, length: torch.Tensor, table: torch.Tensor | None = None,
                parent: torch.Tensor | None = None, out: torch.Tensor | None = None,
                workspace: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Append the nodes' rows behind the committed ones and attend; out [B, nodes, Hq, D] bf16 (see
    TreeCall).  The lengths stay; PagedCache.commit, or LinearCache.commit, moves them on."""
    if workspace is None:
        with _on(stream):
            workspace = new_tree_workspace(step, q.device)
    call = TreeCall(step, q, k_new, v_new, k_pages, v_pages, length, table, parent, out, workspace)
    out = call(stream)
    _used_on(stream, out, call.workspace)
    return out


class LinearCache(CacheCalls):
    """Linear K / V rows of B sequences, for the accepted rows of steps of drafted tokens (TreeStep.for_cache):
    commit and left_out are as PagedCache's.

    caches: bf16 views [planes, B, Hkv, cap, D] (a plane is the K or the V of a layer; layers of another head
    shape are another entry), length [B] int32: committed rows.  The tensors are the caller's and are changed
    in place.  Streams, and a workspace that is not given, are as PagedCache's."""

    def __init__(self, caches: list[torch.Tensor], length: torch.Tensor, workspace: torch.Tensor | None = None):
        if not 1 <= len(caches) <= MAX_POOLS:
            raise ValueError(f"1 .. {MAX_POOLS} caches of other head shapes")
        if caches[0].dim() != 5:
            raise ValueError("a cache is [planes, B, Hkv, cap, D]")
        B, cap = caches[0].shape[1], caches[0].shape[3]
        for i, x in enumerate(caches):
            _check_pool(f"cache {i}", x, B, cap)
        if length.dtype != torch.int32 or length.shape != (B,) or not length.is_contiguous():
            raise ValueError("length must be contiguous int32 [B]")
        check_int32(num_pages=B, page_rows=cap)
        _same_device({**{f"cache {i}": x for i, x in enumerate(caches)}, "length": length, "workspace": workspace})
        self.caches, self.length, self.slots, self.cap = list(caches), length, B, cap
        self.device, self._index, self._lists = length.device, length.device.index, ()
        c = Pages(num_pages=B, page_rows=cap, slots=B, max_pages=1, length=length.data_ptr(), num_pools=len(caches))
        for i, x in enumerate(caches):
            c.pools[i] = _pool(x)
        self._set_up(c, workspace)
