"""Torch-tensor front end of esda_rope (include/esda_rope.h): rotary positions of the q and k
rows that the attention entry points take.

Replaces the reference's rotation by ops (ESRotaryEmbedding.mm:8-46, ESOps.h:58-62) with one
launch for q and k.  Tensors are torch CUDA (HIP) tensors; torch is only the allocator and
stream provider here.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from ._lib import RopeArgs, RopeDesc, RopeScalingDesc, check, check_int32, lib
from .decode import _same_device, _stream_ptr, _used_on

_KINDS = {"none": 0, "linear": 1, "ntk": 2, "bands": 3, "yarn": 4}


@dataclass
class RopeScaling:
    """How a rotary base is scaled for contexts beyond the trained one (esda_rope_scaling):
    kind "none", "linear", "ntk", "bands" or "yarn"."""

    kind: str = "none"
    factor: float = 1.0
    trained_len: int = 0
    low: float = 1.0
    high: float = 4.0


def rope_frequencies(rot_dim: int, base: float, scaling: RopeScaling | None = None,
                     device=None) -> tuple[torch.Tensor, float]:
    """(inv_freq [rot_dim / 2] float32, attn_factor) of a rotary base; computed on the host."""
    s = scaling or RopeScaling()
    if s.kind not in _KINDS:
        raise ValueError(f"unknown rotary scaling {s.kind!r}")
    check_int32(rot_dim=rot_dim, trained_len=s.trained_len)
    d = RopeScalingDesc(_KINDS[s.kind], s.trained_len, base, s.factor, s.low, s.high)
    inv, factor = (ctypes.c_float * max(1, rot_dim // 2))(), ctypes.c_float(0.0)
    check(lib().esda_rope_frequencies(ctypes.byref(d), rot_dim, inv, ctypes.byref(factor)))
    t = torch.tensor(list(inv), dtype=torch.float32)
    return (t if device is None else t.to(device)), float(factor.value)


class RopeCall:
    """A rotation with its C-ABI arguments marshalled once (as DecodeCall): refill q, k and pos in
    place between calls.  Usable under HIP graph capture.

    q [T, Hq, D] and k [T, Hk, D] are bf16 views with unit inner stride (either may be None),
    pos [T] int32, inv_freq [rot_dim / 2] float32.  q_out / k_out default to new tensors and may
    be the inputs themselves."""

    def __init__(self, q, k, pos: torch.Tensor, inv_freq: torch.Tensor, interleaved: bool = False,
                 inverse: bool = False, attn_factor: float = 1.0, q_out=None, k_out=None):
        if q is None and k is None:
            raise ValueError("give q, k or both")
        if q is not None and q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        if k is not None and k_out is None:
            k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
        first = q if q is not None else k
        if first.dim() != 3:
            raise ValueError("q and k must be [tokens, heads, head_dim] views")
        T, _, D = first.shape
        for name, t, like in (("q", q, q), ("k", k, k), ("q_out", q_out, q), ("k_out", k_out, k)):
            if t is None:
                continue
            if like is None:
                raise ValueError(f"{name} without its input")
            if t.dtype != torch.bfloat16:
                raise ValueError(f"{name} must be bf16")
            if t.dim() != 3 or t.shape != like.shape or t.shape[0] != T or t.shape[2] != D or (D > 1 and t.stride(2) != 1):
                raise ValueError(f"{name} must be a [tokens, heads, head_dim] view with unit inner stride, got "
                                 f"{tuple(t.shape)} with strides {t.stride()}")
        if pos.dtype != torch.int32 or pos.shape != (T,) or not pos.is_contiguous():
            raise ValueError("pos must be contiguous int32 [tokens]")
        if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
            raise ValueError("inv_freq must be contiguous float32 [rot_dim / 2]")
        _same_device({"q": q, "k": k, "q_out": q_out, "k_out": k_out, "pos": pos, "inv_freq": inv_freq})

        def strides(t):
            return (t.stride(0), t.stride(1)) if t is not None else (0, 0)

        def ptr(t):
            return t.data_ptr() if t is not None else None

        check_int32(tokens=T, rot_dim=2 * inv_freq.numel())
        self._keep = (q, k, pos, inv_freq)
        self.q_out, self.k_out = q_out, k_out
        self._desc = RopeDesc(T, q.shape[1] if q is not None else 0, k.shape[1] if k is not None else 0, D,
                              2 * inv_freq.numel(), int(bool(interleaved)), int(bool(inverse)), attn_factor, *strides(q),
                              *strides(k), *strides(q_out), *strides(k_out))
        self._args = RopeArgs(ptr(q), ptr(k), ptr(q_out), ptr(k_out), ptr(pos), ptr(inv_freq))
        self._fn = lib().esda_rope
        self._pd, self._pa = ctypes.byref(self._desc), ctypes.byref(self._args)

    def __call__(self, stream=None):
        rc = self._fn(self._pd, self._pa, _stream_ptr(stream))
        if rc:
            check(rc)
        return self.q_out, self.k_out


def rope(q, k, pos: torch.Tensor, inv_freq: torch.Tensor, interleaved: bool = False, inverse: bool = False,
         attn_factor: float = 1.0, q_out=None, k_out=None, stream=None):
    """(q_out, k_out): the rows of q [T, Hq, D] and k [T, Hk, D] (either may be None) rotated to
    positions pos [T]; see RopeCall."""
    out = RopeCall(q, k, pos, inv_freq, interleaved, inverse, attn_factor, q_out, k_out)(stream)
    _used_on(stream, *out)
    return out
