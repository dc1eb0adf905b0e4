"""Microscaled 4-bit floating point (MXFP4) on MI355X: conversion and products.

The format is that of the OCP Microscaling Formats specification, v1.0: along K,
blocks of 32 values share a power-of-two scale (a byte ``b`` for ``2**(b - 127)``,
255 for NaN), and a value is e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 or a negative.  A
matrix ``[..., K]`` is held as ``packed [..., K/2]`` uint8 (value 2i in the low
nibble of byte i) and ``scales [..., K/32]`` uint8.  A weight is held by outputs,
``[N, K]``, as ``nn.Linear`` does; one held ``[K, N]``, as the q4_0 functions take
it, is converted through its transpose: ``quantize_mxfp4(weight.t())``.

No counterpart in the reference.  As in the rest of the package the HIP kernels
of ``libmcq4.so`` do all of it, on the current stream, without a fallback.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib
from .quantization import _DTYPE_CODES, _native, _require_device, _stream, _workspace

MX_BLOCK = 32

__all__ = ["MX_BLOCK", "quantize_mxfp4", "dequantize_mxfp4", "matmul_mxfp4", "linear_mxfp4", "matmul_mxfp4_mxfp4"]

# mcq4.h's MCQ4_ACT_*.
_ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}


def _aligned16(t: torch.Tensor) -> torch.Tensor:
    """``t`` contiguous at a 16-byte aligned address."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _check_packed(packed: torch.Tensor, scales: torch.Tensor, name: str) -> int:
    """K of a packed matrix."""
    if packed.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise RuntimeError(f"{name} and its scales must be uint8, got {packed.dtype} and {scales.dtype}")
    if packed.dim() < 1:
        raise RuntimeError(f"{name} must be [..., K/2], got a scalar")
    K = 2 * packed.shape[-1]
    assert K % MX_BLOCK == 0, f"K ({K}) must be divisible by {MX_BLOCK}"
    if tuple(scales.shape) != (*packed.shape[:-1], K // MX_BLOCK):
        raise RuntimeError(f"scales of {name} must be {(*packed.shape[:-1], K // MX_BLOCK)}, got {tuple(scales.shape)}")
    return K


def quantize_mxfp4(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``x [..., K]`` to ``(packed [..., K/2], scales [..., K/32])``, both uint8.

    The specification's rule: a block's scale is ``2**(floor(log2(amax)) - 2)``, a
    value ``x / scale`` rounded to the nearest e2m1 value, ties to even, and
    saturated at 6.  A block of zeros has byte 0; one with an infinity or a NaN
    has byte 255, so all of it is NaN.  fp32, fp16 and bf16 run as they are, other
    float types through fp32; a matrix may have any strides.
    """
    if _native is not None:
        out = _native.mx_quantize(x)
        if out is not None:
            return out
    if x.dim() < 1:
        raise RuntimeError("x must have at least one dimension")
    K = x.shape[-1]
    assert K % MX_BLOCK == 0, f"K ({K}) must be divisible by {MX_BLOCK}"
    _require_device(x)
    if not x.dtype.is_floating_point:
        raise RuntimeError(f"x must be a floating point tensor, got {x.dtype}")
    if x.dtype not in _DTYPE_CODES:
        x = x.float()
    packed = torch.empty((*x.shape[:-1], K // 2), dtype=torch.uint8, device=x.device)
    scales = torch.empty((*x.shape[:-1], K // MX_BLOCK), dtype=torch.uint8, device=x.device)
    if x.numel() == 0:
        return packed, scales
    m = x if x.dim() == 2 else x.reshape(-1, K)
    with torch.cuda.device(x.device):
        _lib.check(_lib.lib.mcq4_quantize_mxfp4(m.data_ptr(), _DTYPE_CODES[x.dtype], m.stride(0), m.stride(1), m.shape[0],
                                                K, packed.data_ptr(), scales.data_ptr(), _stream(x.device)),
                   "mcq4_quantize_mxfp4")
    return packed, scales


def dequantize_mxfp4(packed: torch.Tensor, scales: torch.Tensor, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The values ``[..., K]`` in ``dtype`` (default float16): exact in fp32 and bf16
    (down to their normal range), rounded once in other types."""
    if dtype is None:
        dtype = torch.float16
    if _native is not None:
        out = _native.mx_dequantize(packed, scales, dtype)
        if out is not None:
            return out
    K = _check_packed(packed, scales, "packed")
    _require_device(packed, scales)
    kernel_dtype = dtype if dtype in _DTYPE_CODES else torch.float32
    out = torch.empty((*packed.shape[:-1], K), dtype=kernel_dtype, device=packed.device)
    if out.numel():
        p, s = _aligned16(packed), scales.contiguous()
        with torch.cuda.device(out.device):
            _lib.check(_lib.lib.mcq4_dequantize_mxfp4(p.data_ptr(), s.data_ptr(), out.numel() // K, K, out.data_ptr(),
                                                      _DTYPE_CODES[kernel_dtype], _stream(out.device)),
                       "mcq4_dequantize_mxfp4")
    return out if dtype == kernel_dtype else out.to(dtype)


def _check_weight(W_packed: torch.Tensor, W_scales: torch.Tensor) -> Tuple[int, int]:
    K = _check_packed(W_packed, W_scales, "W_packed")
    if W_packed.dim() != 2:
        raise RuntimeError(f"W_packed must be [N, K/2], got shape {tuple(W_packed.shape)}")
    return W_packed.shape[0], K


def _rows16(X: torch.Tensor, K: int) -> Tuple[torch.Tensor, int, int]:
    """``X [..., K]`` as rows at 16-byte aligned addresses, their number and their stride."""
    x = X if X.dim() == 2 else X.reshape(-1, K)
    M = x.shape[0]
    if (x.stride(1) != 1 or x.data_ptr() % 16
            or (M > 1 and (x.stride(0) < K or x.stride(0) * x.element_size() % 16))):
        x = _aligned16(x)
    return x, M, x.stride(0) if M > 1 else K     # one row may carry any stride


def matmul_mxfp4(X: torch.Tensor, W_packed: torch.Tensor, W_scales: torch.Tensor) -> torch.Tensor:
    """``X [..., K] @ dequantize_mxfp4(W [N, K]).T`` in X's type, sums in fp32.

    fp16 and bf16 X multiply the weight in X's type (bf16: exact; fp16: exact for
    scales of 2^-23 to 2^13, rounded once beyond).  fp32 X multiplies the exact
    weight, in three bf16 pieces that add up to X.
    """
    if _native is not None:
        Y = _native.mx_matmul(X, W_packed, W_scales)
        if Y is not None:
            return Y
    N, K = _check_weight(W_packed, W_scales)
    if X.dim() < 1:
        raise RuntimeError("X must be [..., K]")
    assert X.shape[-1] == K, f"X K dim ({X.shape[-1]}) must match weight K ({K})"
    _require_device(X, W_packed, W_scales)
    if X.dtype not in _DTYPE_CODES:
        raise RuntimeError(f"X must be float16, bfloat16 or float32, got {X.dtype}")
    Y = torch.empty((*X.shape[:-1], N), dtype=X.dtype, device=X.device)
    if Y.numel() == 0 or K == 0:
        return Y.zero_()
    x, M, ldx = _rows16(X, K)
    w, s = _aligned16(W_packed), W_scales.contiguous()
    code, stream = _DTYPE_CODES[x.dtype], _stream(X.device)
    need = int(_lib.lib.mcq4_matmul_mxfp4_workspace_bytes(M, K, N, code))
    ws = _workspace.get(X.device, stream, need) if need else None
    with torch.cuda.device(X.device), _workspace.guard(ws, stream):
        _lib.check(_lib.lib.mcq4_matmul_mxfp4(x.data_ptr(), code, ldx, w.data_ptr(), s.data_ptr(), Y.data_ptr(), N,
                                              M, K, N, ws.data_ptr() if need else None, ws.numel() if need else 0, stream),
                   "mcq4_matmul_mxfp4")
    return Y


def _operand(t: Optional[torch.Tensor], name: str, Y: torch.Tensor) -> Tuple[Optional[torch.Tensor], int]:
    """``t``, of Y's shape and type, as rows of neighbouring columns, and their stride."""
    if t is None:
        return None, 0
    if t.shape != Y.shape or t.dtype != Y.dtype:
        raise RuntimeError(f"{name} must be {tuple(Y.shape)} {Y.dtype}, got {tuple(t.shape)} {t.dtype}")
    if not t.numel():
        return None, 0
    N = Y.shape[-1]
    t = t if t.dim() == 2 else t.reshape(-1, N)
    if t.shape[0] > 1 and t.stride(0) < N or t.shape[1] > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, t.stride(0) if t.shape[0] > 1 else N


def linear_mxfp4(X: torch.Tensor, W_packed: torch.Tensor, W_scales: torch.Tensor, bias: Optional[torch.Tensor] = None,
                 activation: Optional[str] = None, multiply: Optional[torch.Tensor] = None,
                 residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``activation(matmul_mxfp4(X, W) + bias) * multiply + residual`` in one launch, or as few
    as the product takes: fp32 from the sums on, rounded once to X's type.

    ``bias [N]`` is in X's type or fp32; ``multiply`` (the other half of a gated layer) and
    ``residual`` have the result's shape and type, their rows any stride.  ``activation`` is None,
    "relu", "silu", "gelu" (``x Phi(x)``) or "gelu_tanh" (its tanh form).
    """
    if _native is not None:
        Y = _native.mx_linear(X, W_packed, W_scales, bias, activation, multiply, residual)
        if Y is not None:
            return Y
    N, K = _check_weight(W_packed, W_scales)
    if X.dim() < 1:
        raise RuntimeError("X must be [..., K]")
    assert X.shape[-1] == K, f"X K dim ({X.shape[-1]}) must match weight K ({K})"
    _require_device(X, W_packed, W_scales, *[t for t in (bias, multiply, residual) if t is not None])
    if X.dtype not in _DTYPE_CODES:
        raise RuntimeError(f"X must be float16, bfloat16 or float32, got {X.dtype}")
    if activation not in _ACTIVATIONS:
        raise RuntimeError(f"activation must be one of {tuple(_ACTIVATIONS)}, got {activation!r}")
    Y = torch.empty((*X.shape[:-1], N), dtype=X.dtype, device=X.device)
    if bias is not None:
        if tuple(bias.shape) != (N,) or bias.dtype not in (X.dtype, torch.float32):
            raise RuntimeError(f"bias must be ({N},) {X.dtype} or float32, got {tuple(bias.shape)} {bias.dtype}")
        bias = bias.contiguous()
    mul, ld_mul = _operand(multiply, "multiply", Y)
    res, ld_res = _operand(residual, "residual", Y)
    if Y.numel() == 0:
        return Y
    if K == 0:
        raise RuntimeError("K must be at least 32")
    x, M, ldx = _rows16(X, K)
    w, s = _aligned16(W_packed), W_scales.contiguous()
    code, stream = _DTYPE_CODES[x.dtype], _stream(X.device)
    epilogue = _lib.EpilogueStruct(*[None if t is None else t.data_ptr() for t in (bias, mul, res)], ld_mul, ld_res,
                                   0 if bias is None else _DTYPE_CODES[bias.dtype], _ACTIVATIONS[activation])
    need = int(_lib.lib.mcq4_matmul_mxfp4_workspace_bytes(M, K, N, code))
    ws = _workspace.get(X.device, stream, need) if need else None
    with torch.cuda.device(X.device), _workspace.guard(ws, stream):
        _lib.check(_lib.lib.mcq4_linear_mxfp4(x.data_ptr(), code, ldx, w.data_ptr(), s.data_ptr(), ctypes.byref(epilogue),
                                              Y.data_ptr(), N, M, K, N, ws.data_ptr() if need else None,
                                              ws.numel() if need else 0, stream),
                   "mcq4_linear_mxfp4")
    return Y


def matmul_mxfp4_mxfp4(X_packed: torch.Tensor, X_scales: torch.Tensor, W_packed: torch.Tensor, W_scales: torch.Tensor,
                       dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``dequantize(X [..., K]) @ dequantize(W [N, K]).T`` of two MXFP4 matrices, in
    ``dtype`` (float16, the default, bfloat16 or float32): exact products, sums in fp32."""
    if dtype is None:
        dtype = torch.float16
    if _native is not None:
        Y = _native.mx_matmul_mx(X_packed, X_scales, W_packed, W_scales, dtype)
        if Y is not None:
            return Y
    N, K = _check_weight(W_packed, W_scales)
    Kx = _check_packed(X_packed, X_scales, "X_packed")
    assert Kx == K, f"X K dim ({Kx}) must match weight K ({K})"
    _require_device(X_packed, X_scales, W_packed, W_scales)
    if dtype not in _DTYPE_CODES:
        raise RuntimeError(f"dtype must be float16, bfloat16 or float32, got {dtype}")
    Y = torch.empty((*X_packed.shape[:-1], N), dtype=dtype, device=X_packed.device)
    if Y.numel() == 0 or K == 0:
        return Y.zero_()
    x, xs, w, s = _aligned16(X_packed), X_scales.contiguous(), _aligned16(W_packed), W_scales.contiguous()
    M, stream = Y.numel() // N, _stream(Y.device)
    need = int(_lib.lib.mcq4_matmul_mxfp4_mxfp4_workspace_bytes(M, K, N))
    ws = _workspace.get(Y.device, stream, need) if need else None
    with torch.cuda.device(Y.device), _workspace.guard(ws, stream):
        _lib.check(_lib.lib.mcq4_matmul_mxfp4_mxfp4(x.data_ptr(), xs.data_ptr(), w.data_ptr(), s.data_ptr(), Y.data_ptr(),
                                                    _DTYPE_CODES[dtype], N, M, K, N, ws.data_ptr() if need else None,
                                                    ws.numel() if need else 0, stream),
                   "mcq4_matmul_mxfp4_mxfp4")
    return Y
