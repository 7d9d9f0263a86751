"""Torch-tensor front end of include/esda_prefix.h: the decode step of a batch whose sequences
share their first tokens, whose K / V rows are stored and read once.

The reference is batch 1 (ESAttention.mm:188) and keeps such a prefix under a marker
(ESKVCache.mm:123-143).  Tensors are torch CUDA (HIP) tensors; torch is only the allocator and
stream provider here.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from ._lib import DecodeArgs, PrefixArgs, PrefixDesc, check, check_int32, lib
from .decode import DecodeStep, _check_cache, _dev_ptr, _on, _same_device, _stream_ptr, _used_on


@dataclass
class PrefixStep:
    """Shapes of a step over a shared prefix (esda_prefix_desc): ``own`` describes the sequences'
    own caches (linear rows, the row of position p is p - prefix_len)."""

    own: DecodeStep
    prefix_len: int
    prefix_head_stride: int | None = None
    split_keys: int = 0

    def desc(self) -> PrefixDesc:
        hs = self.prefix_head_stride if self.prefix_head_stride is not None else self.prefix_len * self.own.head_dim
        check_int32(prefix_len=self.prefix_len, split_keys=self.split_keys)
        return PrefixDesc(self.own.desc(), self.prefix_len, self.split_keys, hs)

    @classmethod
    def for_caches(cls, prefix_k: torch.Tensor, cache: torch.Tensor, num_q_heads: int, split_keys: int = 0,
                   **kw) -> "PrefixStep":
        """prefix_k: [Hkv, P, D] view with dense rows; cache: [B, Hkv, cap, D] (DecodeStep.for_cache)."""
        own = DecodeStep.for_cache(cache, num_q_heads, **kw)
        Hkv, P, D = prefix_k.shape
        if (Hkv, D) != (own.num_kv_heads, own.head_dim) or prefix_k.stride(2) != 1 or prefix_k.stride(1) != D:
            raise ValueError("prefix_k must be an [Hkv, P, D] view with dense rows")
        return cls(own, P, prefix_k.stride(0) if Hkv > 1 else P * D, split_keys)


def prefix_workspace_bytes(step: PrefixStep) -> int:
    n, d = ctypes.c_size_t(0), step.desc()
    check(lib().esda_prefix_decode_workspace_size(ctypes.byref(d), ctypes.byref(n)))
    return int(n.value)


def new_prefix_workspace(step: PrefixStep, device) -> torch.Tensor:
    """Workspace for ``step``, its status word zeroed (decode_status(step.own, workspace) reads it)."""
    return torch.zeros(prefix_workspace_bytes(step), dtype=torch.uint8, device=device)


class PrefixCall:
    """A decode step over a shared prefix with its C-ABI arguments marshalled once (as
    DecodeCall): refill q, k_new, v_new and pos in place between calls.  Usable under HIP graph
    capture.  pos [B] int32: absolute positions, prefix_len or more.  A workspace that is not given is
    cleared here, on the current stream."""

    def __init__(self, step: PrefixStep, q, k_new, v_new, prefix_k, prefix_v, k_cache, v_cache, pos, out=None,
                 workspace=None):
        own, d = step.own, step.desc()
        shape = (own.batch, own.num_q_heads, own.head_dim)
        if q.shape != shape or not q.is_contiguous():
            raise ValueError(f"q must be contiguous [B, Hq, D], got {tuple(q.shape)}")
        if k_new.shape != (own.batch, own.num_kv_heads, own.head_dim) or not k_new.is_contiguous():
            raise ValueError("k_new must be contiguous [B, Hkv, D]")
        if v_new is not None and (v_new.shape != k_new.shape or not v_new.is_contiguous()):
            raise ValueError("v_new must be contiguous [B, Hkv, D]")
        if pos.dtype != torch.int32 or pos.shape != (own.batch,) or not pos.is_contiguous():
            raise ValueError("pos must be contiguous int32 [B]")
        if out is None:
            out = torch.empty_like(q)
        if out.shape != shape or not out.is_contiguous():
            raise ValueError("out must be contiguous [B, Hq, D]")
        if workspace is None:
            workspace = new_prefix_workspace(step, q.device)
        vc = k_cache if (v_cache is None or own.kv_shared) else v_cache
        pv = prefix_k if (prefix_v is None or own.kv_shared) else prefix_v
        _check_cache(own, k_cache, "k_cache")
        _check_cache(own, vc, "v_cache")
        need = (own.num_kv_heads - 1) * d.prefix_head_stride + step.prefix_len * own.head_dim
        for name, t in (("prefix_k", prefix_k), ("prefix_v", pv)):
            if t.dim() == 3 and (t.shape != (own.num_kv_heads, step.prefix_len, own.head_dim) or t.stride(2) != 1 or
                                 t.stride(1) != own.head_dim or
                                 (own.num_kv_heads > 1 and t.stride(0) != d.prefix_head_stride)):
                raise ValueError(f"{name} is {tuple(t.shape)} with strides {t.stride()}; the step describes "
                                 f"({own.num_kv_heads}, {step.prefix_len}, {own.head_dim}), heads {d.prefix_head_stride} apart")
            if t.dim() != 3 and not t.is_contiguous():
                raise ValueError(f"{name}: pass a contiguous buffer or an [Hkv, P, D] view")
            if t.untyped_storage().nbytes() // 2 - t.storage_offset() < need:
                raise ValueError(f"{name} is smaller than the description's extent")
        _same_device({"q": q, "k_new": k_new, "v_new": v_new, "prefix_k": prefix_k, "prefix_v": pv, "k_cache": k_cache,
                      "v_cache": vc, "pos": pos, "out": out, "workspace": workspace})
        bf = torch.bfloat16
        self._keep = (q, k_new, v_new, prefix_k, prefix_v, k_cache, v_cache, pos)
        self.step, self.out, self.workspace = step, out, workspace
        self._desc = d
        self._args = PrefixArgs(
            DecodeArgs(_dev_ptr(q, bf), _dev_ptr(k_new, bf),
                       _dev_ptr(v_new, bf) if (v_new is not None and not own.kv_shared) else None, _dev_ptr(k_cache, bf),
                       _dev_ptr(vc, bf), _dev_ptr(pos), None, _dev_ptr(out, bf), _dev_ptr(workspace),
                       workspace.numel() * workspace.element_size()),
            _dev_ptr(prefix_k, bf), _dev_ptr(pv, bf))
        self._fn = lib().esda_prefix_decode
        self._pd, self._pa = ctypes.byref(self._desc), ctypes.byref(self._args)

    def __call__(self, stream=None) -> torch.Tensor:
        rc = self._fn(self._pd, self._pa, _stream_ptr(stream))
        if rc:
            check(rc)
        return self.out


def prefix_decode(step: PrefixStep, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor | None,
                  prefix_k: torch.Tensor, prefix_v: torch.Tensor | None, k_cache: torch.Tensor,
                  v_cache: torch.Tensor | None, pos: torch.Tensor, out: torch.Tensor | None = None,
                  workspace: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Append the new rows to the sequences' own caches and attend the shared prefix and them; out
    [B, Hq, D] bf16."""
    if workspace is None:
        with _on(stream):
            workspace = new_prefix_workspace(step, q.device)
    call = PrefixCall(step, q, k_new, v_new, prefix_k, prefix_v, k_cache, v_cache, pos, out, workspace)
    out = call(stream)
    _used_on(stream, out, call.workspace)
    return out
