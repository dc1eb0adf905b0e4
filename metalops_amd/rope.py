"""Norms of queries' and keys' heads and their rotation by positions, on MI355X.

What stands between a layer's projection of q and k and the attention: each head's RMS
norm, where a model has them, and the rotary positions, in one pass over both.  Text has one
axis of positions; images and video have several (time, height, width), to each of which
some of the channel pairs belong.

No counterpart in the reference.  As in the rest of the package a HIP kernel of
``libmcq4.so`` does all of it, on the current stream, without a fallback.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from .quantization import _DTYPE_CODES, _native, _require_device, _stream

__all__ = ["qk_norm_rope"]


def _heads(x: torch.Tensor, name: str, out: Optional[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor]:
    """x with neighbouring channels, and its output."""
    if x.shape[2] > 1 and x.stride(2) != 1:
        x = x.contiguous()
    if out is None:
        return x, torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if out.shape != x.shape or out.dtype != x.dtype:
        raise RuntimeError(f"the output of {name} must be {tuple(x.shape)} {x.dtype}, got {tuple(out.shape)} {out.dtype}")
    if out.shape[2] > 1 and out.stride(2) != 1:
        raise RuntimeError(f"the output of {name} must have neighbouring channels")
    if any(n > 1 and s <= 0 for n, s in zip(out.shape, out.stride())):
        raise RuntimeError(f"the output of {name} must not be broadcast")
    return x, out


def _struct(x: torch.Tensor, y: torch.Tensor, w: Optional[torch.Tensor]) -> _lib.RopeHeadsStruct:
    def strides(t):          # where there is one token or head, its stride is any and not asked for
        return (t.stride(0) if t.shape[0] > 1 else 0), (t.stride(1) if t.shape[1] > 1 else 0)
    return _lib.RopeHeadsStruct(x.data_ptr(), y.data_ptr(), None if w is None else w.data_ptr(), *strides(x), *strides(y),
                                x.shape[1], 0 if w is None else _DTYPE_CODES[w.dtype])


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 sections: Optional[Sequence[int]] = None, interleaved: bool = False,
                 out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``q [T, heads, D]`` and ``k [T, kv_heads, D]`` (fp32, fp16 or bf16), normalized and rotated.

    Where a weight ``[D]`` (any of these types) is given, each head becomes
    ``x * rsqrt(mean(x**2) + eps) * weight``.  Then pair i of its first ``2 * len(inv_freq)``
    channels turns by ``position * inv_freq[i]`` radians: channels i and ``i + len(inv_freq)``,
    or with ``interleaved`` 2i and 2i + 1.  The channels behind them keep what the norm made
    of them.  ``positions`` is int32 ``[T]``, or ``[axes, T]`` with ``sections``, up to four numbers:
    the first ``sections[0]`` pairs turn by axis 0's position, the next ``sections[1]`` by axis 1's,
    and so on.  ``inv_freq`` is fp32, its length a multiple of 4; D is a multiple of 8 up to 512.

    Everything is computed in fp32 (angles in fp64: far positions are exact) and rounded once.  Returns
    new tensors, or ``out``, two tensors that may be q and k themselves but overlap nothing else.
    """
    if isinstance(sections, list):
        sections = tuple(sections)
    if _native is not None and out is None:
        pair = _native.qk_norm_rope(q, k, positions, inv_freq, q_weight, k_weight, eps, sections, interleaved)
        if pair is not None:
            return pair
    for name, x in (("q", q), ("k", k)):
        if x.dim() != 3:
            raise RuntimeError(f"{name} must be [T, heads, D], got shape {tuple(x.shape)}")
        if x.dtype not in _DTYPE_CODES or x.dtype != q.dtype:
            raise RuntimeError(f"q and k must both be float16, bfloat16 or float32, got {q.dtype} and {k.dtype}")
        if x.shape[1] == 0:
            raise RuntimeError(f"{name} must have heads")
    T, _, D = q.shape
    if (k.shape[0], k.shape[2]) != (T, D):
        raise RuntimeError(f"q and k must have one T and D, got {tuple(q.shape)} and {tuple(k.shape)}")
    if D % 8 or not 0 < D <= 512:
        raise RuntimeError(f"head dim must be a multiple of 8 up to 512, got {D}")
    if inv_freq.dim() != 1 or inv_freq.dtype != torch.float32:
        raise RuntimeError(f"inv_freq must be 1-dimensional float32, got {tuple(inv_freq.shape)} {inv_freq.dtype}")
    half = inv_freq.shape[0]
    if half % 4 or not 0 < 2 * half <= D:
        raise RuntimeError(f"inv_freq must have a multiple of 4 elements up to D / 2 ({D // 2}), got {half}")
    sections = (half,) if sections is None else tuple(int(s) for s in sections)
    if not 1 <= len(sections) <= 4 or min(sections) < 0 or sum(sections) != half:
        raise RuntimeError(f"sections must be 1 to 4 numbers that add up to {half}, got {sections}")
    if positions.dtype != torch.int32:
        raise RuntimeError(f"positions must be int32, got {positions.dtype}")
    if tuple(positions.shape) != (len(sections), T) and not (len(sections) == 1 and tuple(positions.shape) == (T,)):
        raise RuntimeError(f"positions must be ({len(sections)}, {T}), got {tuple(positions.shape)}")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (tuple(w.shape) != (D,) or w.dtype not in _DTYPE_CODES):
            raise RuntimeError(f"{name} must be ({D},) float16, bfloat16 or float32, got {tuple(w.shape)} {w.dtype}")
    if out is not None and len(out) != 2:
        raise RuntimeError(f"out must be two tensors, got {len(out)}")
    _require_device(q, k, positions, inv_freq, *[t for t in (q_weight, k_weight, *(out or ())) if t is not None])
    q, q_out = _heads(q, "q", None if out is None else out[0])
    k, k_out = _heads(k, "k", None if out is None else out[1])
    if T:
        positions, inv_freq = positions.contiguous(), inv_freq.contiguous()
        if inv_freq.data_ptr() % 16:
            inv_freq = inv_freq.clone()
        q_weight, k_weight = [None if w is None else w.contiguous() for w in (q_weight, k_weight)]
        st = _lib.RopeStruct(_struct(q, q_out, q_weight), _struct(k, k_out, k_weight), positions.data_ptr(), inv_freq.data_ptr(), T, T,
                             (ctypes.c_int32 * 4)(*sections), len(sections), D, 2 * half, int(bool(interleaved)),
                             _DTYPE_CODES[q.dtype], float(eps))
        with torch.cuda.device(q.device):
            _lib.check(_lib.lib.mcq4_qk_norm_rope(ctypes.byref(st), _stream(q.device)), "mcq4_qk_norm_rope")
    return q_out, k_out
