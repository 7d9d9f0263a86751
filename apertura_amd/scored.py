"""Torch-tensor front end of include/esda_scored.h: the decode step and the prefill chunk with
scores capped by a tanh or biased by distance, and chunks with a document or a prefix mask.

The reference has the plain forms (ESAttention.mm:136-193).  Tensors are torch CUDA (HIP)
tensors; torch is only the allocator and stream provider here.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from ._lib import DecodeArgs, ScoreDesc, ScoredPrefillArgs, check, check_int32, lib
from .decode import (DecodeStep, _check_cache, _check_row_base, _dev_ptr, _on, _same_device, _stream_ptr,
                     _used_on, new_workspace)
from .prefill import PrefillStep


@dataclass
class Score:
    """How scores and masks differ from plain attention (esda_score).

    softcap > 0 caps a score s to softcap * tanh(s / softcap); slopes [Hq] float32 takes
    slopes[h] * distance off it; prefix (prefill) lets every query see the keys at positions
    below it."""

    softcap: float = 0.0
    slopes: torch.Tensor | None = None
    prefix: int = 0

    def desc(self, num_q_heads: int) -> ScoreDesc:
        s = self.slopes
        if s is not None and (s.dtype != torch.float32 or s.shape != (num_q_heads,) or not s.is_contiguous()):
            raise ValueError("slopes must be contiguous float32 [Hq]")
        check_int32(prefix=self.prefix)
        if self.softcap > 0 and ctypes.c_float(self.softcap).value == 0:
            raise ValueError(f"softcap = {self.softcap} is 0 in float32, which is no cap")
        return ScoreDesc(self.softcap, self.prefix, None if s is None else s.data_ptr())


def scored_prefill_workspace_bytes(step: PrefillStep, score: Score) -> int:
    n, d, s = ctypes.c_size_t(0), step.desc(), score.desc(step.num_q_heads)
    check(lib().esda_scored_prefill_workspace_size(ctypes.byref(d), ctypes.byref(s), ctypes.byref(n)))
    return int(n.value)


def scored_prefill(step: PrefillStep, score: Score, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                   q_doc: torch.Tensor | None = None, k_doc: torch.Tensor | None = None,
                   out: torch.Tensor | None = None, workspace: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """O [Sq, Hq, D] bf16 of ``step`` with ``score``'s scores and masks (tensors and strides as in
    ``prefill``).  q_doc [Sq] and k_doc [Sk] int32: a query sees the keys of its own document; a
    negative id belongs to none.  Queries that see no key give 0."""
    bf = torch.bfloat16
    D = step.head_dim
    if out is None:
        out = torch.empty((step.seq_q, step.num_q_heads, D), dtype=bf, device=q.device)
    d, s = step.desc(), score.desc(step.num_q_heads)
    kv = (step.num_kv_heads - 1) * d.kv_head_stride + step.seq_k * D
    for name, t, need in (
            ("q", q, (step.num_q_heads - 1) * d.q_head_stride + (step.seq_q - 1) * d.q_row_stride + D),
            ("k", k, kv), ("v", v, kv),
            ("out", out, (step.seq_q - 1) * d.out_row_stride + (step.num_q_heads - 1) * d.out_head_stride + D)):
        if t.dtype != bf:
            raise ValueError(f"{name} must be a bf16 GPU tensor")
        if t.untyped_storage().nbytes() // 2 - t.storage_offset() < need:
            raise ValueError(f"{name} is smaller than the description's extent")
    if (q_doc is None) != (k_doc is None):
        raise ValueError("q_doc and k_doc go together")
    for name, t, n in (("q_doc", q_doc, step.seq_q), ("k_doc", k_doc, step.seq_k)):
        if t is not None and (t.dtype != torch.int32 or t.shape != (n,) or not t.is_contiguous()):
            raise ValueError(f"{name} must be contiguous int32 [{n}]")
    _same_device({"q": q, "k": k, "v": v, "out": out, "q_doc": q_doc, "k_doc": k_doc, "slopes": score.slopes,
                  "workspace": workspace})
    n = ctypes.c_size_t(0)
    check(lib().esda_scored_prefill_workspace_size(ctypes.byref(d), ctypes.byref(s), ctypes.byref(n)))
    if n.value and (workspace is None or workspace.numel() * workspace.element_size() < n.value):
        workspace = torch.empty(n.value, dtype=torch.uint8, device=q.device)
    a = ScoredPrefillArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                          workspace.data_ptr() if n.value else None, n.value, _dev_ptr(q_doc), _dev_ptr(k_doc))
    check(lib().esda_scored_prefill(ctypes.byref(d), ctypes.byref(s), ctypes.byref(a), _stream_ptr(stream)))
    _used_on(stream, out, workspace)
    return out


class ScoredDecodeCall:
    """A decode step with modified scores, its C-ABI arguments marshalled once (as DecodeCall):
    refill q, k_new, v_new and pos in place between calls.  Usable under HIP graph capture.  A
    workspace that is not given is cleared here, on the current stream."""

    def __init__(self, step: DecodeStep, score: Score, q, k_new, v_new, k_cache, v_cache, pos, row_base=None, out=None,
                 workspace=None):
        shape = (step.batch, step.num_q_heads, step.head_dim)
        if q.shape != shape or not q.is_contiguous():
            raise ValueError(f"q must be contiguous [B, Hq, D], got {tuple(q.shape)}")
        if k_new.shape != (step.batch, step.num_kv_heads, step.head_dim) or not k_new.is_contiguous():
            raise ValueError("k_new must be contiguous [B, Hkv, D]")
        if v_new is not None and (v_new.shape != k_new.shape or not v_new.is_contiguous()):
            raise ValueError("v_new must be contiguous [B, Hkv, D]")
        if pos.dtype != torch.int32 or pos.shape != (step.batch,) or not pos.is_contiguous():
            raise ValueError("pos must be contiguous int32 [B]")
        if out is None:
            out = torch.empty_like(q)
        if out.shape != shape or not out.is_contiguous():
            raise ValueError("out must be contiguous [B, Hq, D]")
        if workspace is None:
            workspace = new_workspace(step, q.device)
        vc = k_cache if (v_cache is None or step.kv_shared) else v_cache
        _check_cache(step, k_cache, "k_cache")
        _check_cache(step, vc, "v_cache")
        _check_row_base(step, row_base)
        _same_device({"q": q, "k_new": k_new, "v_new": v_new, "k_cache": k_cache, "v_cache": vc, "pos": pos,
                      "row_base": row_base, "out": out, "workspace": workspace, "slopes": score.slopes})
        bf = torch.bfloat16
        self._keep = (q, k_new, v_new, k_cache, v_cache, pos, row_base, score.slopes)
        self.step, self.out, self.workspace = step, out, workspace
        self._desc, self._score = step.desc(), score.desc(step.num_q_heads)
        self._args = DecodeArgs(_dev_ptr(q, bf), _dev_ptr(k_new, bf),
                                _dev_ptr(v_new, bf) if (v_new is not None and not step.kv_shared) else None,
                                _dev_ptr(k_cache, bf), _dev_ptr(vc, bf), _dev_ptr(pos), _dev_ptr(row_base),
                                _dev_ptr(out, bf), _dev_ptr(workspace), workspace.numel() * workspace.element_size())
        self._fn = lib().esda_scored_decode
        self._pd, self._ps, self._pa = (ctypes.byref(self._desc), ctypes.byref(self._score), ctypes.byref(self._args))

    def __call__(self, stream=None) -> torch.Tensor:
        rc = self._fn(self._pd, self._ps, self._pa, _stream_ptr(stream))
        if rc:
            check(rc)
        return self.out


def scored_decode(step: DecodeStep, score: Score, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor | None,
                  k_cache: torch.Tensor, v_cache: torch.Tensor | None, pos: torch.Tensor,
                  row_base: torch.Tensor | None = None, out: torch.Tensor | None = None,
                  workspace: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """decode_step with ``score``'s scores: append the new rows and attend; out [B, Hq, D] bf16."""
    if workspace is None:
        with _on(stream):
            workspace = new_workspace(step, q.device)
    call = ScoredDecodeCall(step, score, q, k_new, v_new, k_cache, v_cache, pos, row_base, out, workspace)
    out = call(stream)
    _used_on(stream, out, call.workspace)
    return out
