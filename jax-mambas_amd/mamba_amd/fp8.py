"""8-bit serving operators on MI355X (HIP kernels behind the C ABI): activations and weights as
e4m3 floats with block scales, and the projections' product in that form.

The 8-bit form of a matrix is ``(q, scales)``: q float8_e4m3fn in rows along the features, which
start on 16 bytes, and float32 scales for blocks of 128 features; a value stands for
``q * scale``. A scale is the block's largest magnitude / 448 (at least 2^-126), q is rounded to
nearest even.

``quantize_fp8(x) -> (q, scales)`` — x (features, tokens) float32 or bfloat16, any non-negative
strides (channel-major activations, or the ``.t()`` of token-major ones); q (tokens, features),
scales (ceil(features / 128), tokens).

``add_rmsnorm_fp8(h, delta, weight, eps=1e-5) -> (hn, q, scales)`` — ``add_rmsnorm``'s residual
add and norm (mamba/mamba1.py:300-337) with the normalised output in 8-bit form: h (features,
tokens) float32, delta float32, bfloat16 or None, hn = h + delta (h itself when delta is None).

``quantize_fp8_weight(w) -> (q, scales)`` — w (M, K) float32 or bfloat16 with contiguous rows;
q (M, K), scales (ceil(M / 128), ceil(K / 128)), one for each 128 x 128 block.

``fp8_matmul(wq, w_scales, xq, x_scales, out_dtype=torch.bfloat16, token_major=False, out=None)``
— W @ X for a weight and activations in 8-bit form: (M, T), or (T, M) with token_major; each
block of 128 features summed on the matrix cores, scaled and added in float32, rounded to out_dtype
(bfloat16 or float32) once. With out_dtype float32 a block's sum is float32 too. With bfloat16 it may
come from the 8-bit matrix instructions, which drop of each 8 neighbouring products what lies below
2^-13 of the largest: less than the output's rounding, except where large products cancel each other.

A NaN or infinity makes what its block stands for NaN. Inference only (no autograd); there is no
CPU path.
"""
from __future__ import annotations

import torch

from . import _lib
from .selective_scan_hip import _io_tag, _ptr, _require_gpu, _resolved, _stream

__all__ = ["quantize_fp8", "add_rmsnorm_fp8", "quantize_fp8_weight", "fp8_matmul"]

_BLOCK = _lib.MSS_FP8_BLOCK
FP8 = torch.float8_e4m3fn
_F32 = torch.float32
_TAGS = {torch.float32: _lib.MSS_F32, torch.bfloat16: _lib.MSS_BF16}


def _blocks(n):
    return -(-n // _BLOCK)


def _empty_rows(rows, cols, device):
    """An uninitialised (rows, cols) 8-bit matrix whose rows start on 16 bytes."""
    if cols % 16 == 0:
        return torch.empty(rows, cols, dtype=FP8, device=device)
    return torch.empty(rows, -(-cols // 16) * 16, dtype=FP8, device=device)[:, :cols]


def _row_stride(q, rows, cols):
    """The row stride of an 8-bit matrix (one that a single row may have, where it has one row)."""
    return q.stride(0) if rows > 1 else -(-cols // 16) * 16


def _no_grad_needed(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError("the 8-bit operators are for inference: call them under torch.no_grad()")


def quantize_fp8(x):
    if x.dim() != 2:
        raise ValueError("x must be a (features, tokens) matrix")
    io = _TAGS.get(x.dtype)
    if io is None:
        io = _io_tag(x.dtype, "x")  # raises
    _no_grad_needed(x)
    _require_gpu(x)
    if x.is_neg():
        x = _resolved(x)
    f, t = x.shape
    dev = x.device
    q = _empty_rows(t, f, dev)
    scales = torch.empty(_blocks(f), t, dtype=_F32, device=dev)
    if f == 0 or t == 0:
        return q, scales
    sf, st = x.stride()
    a = _lib.QuantFp8Args(f, t, io, sf, st, _row_stride(q, t, f), x.data_ptr(), q.data_ptr(), scales.data_ptr())
    _lib.check(_lib.register_hip_kernel().mss_quant_fp8(a, _stream(x)), "mss_quant_fp8")
    return q, scales


def add_rmsnorm_fp8(h, delta, weight, eps=1e-5):
    if h.dtype != _F32 or h.dim() != 2:
        raise TypeError("h must be a float32 (features, tokens) matrix")
    f, t = h.shape
    if weight.dtype != _F32 or weight.dim() != 1 or weight.shape[0] != f:
        raise ValueError(f"weight must be float32 with shape ({f},)")
    tag = _lib.MSS_F32
    if delta is not None:
        if delta.shape != h.shape:
            raise ValueError("delta must have h's shape")
        tag = _TAGS.get(delta.dtype)
        if tag is None:
            tag = _io_tag(delta.dtype, "delta")  # raises
    if f == 0:
        raise ValueError("h has no features")
    _no_grad_needed(h, delta, weight)
    _require_gpu(h, delta, weight)
    if h.is_neg() or weight.is_neg() or (delta is not None and delta.is_neg()):
        h, delta, weight = _resolved(h), _resolved(delta), _resolved(weight)
    h, weight = h.contiguous(), weight.contiguous()
    dev = h.device
    q = _empty_rows(t, f, dev)
    scales = torch.empty(_blocks(f), t, dtype=_F32, device=dev)
    hn = h
    if delta is not None:
        delta = delta.contiguous()
        hn = torch.empty(f, t, dtype=_F32, device=dev)
    if t == 0:
        return hn, q, scales
    a = _lib.NormFp8Args(f, t, tag, eps, _row_stride(q, t, f), h.data_ptr(), _ptr(delta), weight.data_ptr(),
                         hn.data_ptr(), q.data_ptr(), scales.data_ptr())
    _lib.check(_lib.register_hip_kernel().mss_norm_fp8(a, _stream(h)), "mss_norm_fp8")
    return hn, q, scales


def quantize_fp8_weight(w):
    if w.dim() != 2 or (w.shape[1] > 1 and w.stride(1) != 1):
        raise ValueError("w must be a (M, K) matrix with contiguous rows")
    io = _io_tag(w.dtype, "w")
    _no_grad_needed(w)
    _require_gpu(w)
    w = _resolved(w)
    m, k = w.shape
    q = _empty_rows(m, k, w.device)
    scales = torch.empty(_blocks(m), _blocks(k), dtype=_F32, device=w.device)
    if m == 0 or k == 0:
        return q, scales
    a = _lib.QuantFp8WeightArgs(m, k, io, w.stride(0) if m > 1 else k, _row_stride(q, m, k), w.data_ptr(),
                                q.data_ptr(), scales.data_ptr())
    _lib.check(_lib.register_hip_kernel().mss_quant_fp8_weight(a, _stream(w)), "mss_quant_fp8_weight")
    return q, scales


def _check_rows(name, q, k):
    """Refuses what is not an 8-bit matrix of k columns in the layout the kernels read; its rows and
    their stride."""
    if q.dtype != FP8 or q.dim() != 2:
        raise TypeError(f"{name} must be a float8_e4m3fn matrix")
    rows, cols = q.shape
    if cols != k:
        raise ValueError(f"{name} must have {k} columns, got {cols}")
    ld, step = q.stride()
    if rows and cols and (cols > 1 and step != 1 or rows > 1 and ld % 16 != 0 or q.data_ptr() % 16 != 0):
        raise ValueError(f"{name} must have contiguous rows that start on 16 bytes")
    return rows, ld if rows > 1 else -(-cols // 16) * 16


def _check_scales(name, s, rows, cols):
    if s.dtype != _F32 or s.shape != (rows, cols) or not s.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 tensor of shape {(rows, cols)}")


def fp8_matmul(wq, w_scales, xq, x_scales, out_dtype=torch.bfloat16, token_major=False, out=None):
    k = wq.shape[-1] if wq.dim() else 0
    m, ldw = _check_rows("wq", wq, k)
    t, ldx = _check_rows("xq", xq, k)
    kb = -(-k // _BLOCK)
    _check_scales("w_scales", w_scales, -(-m // _BLOCK), kb)
    _check_scales("x_scales", x_scales, kb, t)
    tag = _TAGS.get(out_dtype)
    if tag is None:
        tag = _io_tag(out_dtype, "out_dtype")  # raises
    rows, cols = (t, m) if token_major else (m, t)
    ldc = cols
    if out is not None:
        if out.shape != (rows, cols) or out.dtype != out_dtype or (cols > 1 and out.stride(1) != 1):
            raise ValueError(f"out must be {out_dtype} of shape {(rows, cols)} with contiguous rows")
        if out.is_neg():
            raise ValueError("out must not be lazily negated")
        if rows > 1:
            ldc = out.stride(0)
    _no_grad_needed(wq, w_scales, xq, x_scales, out)
    _require_gpu(wq, w_scales, xq, x_scales, out)
    if w_scales.is_neg() or x_scales.is_neg():
        w_scales, x_scales = _resolved(w_scales), _resolved(x_scales)
    if out is None:
        out = torch.empty(rows, cols, dtype=out_dtype, device=wq.device)
    if m == 0 or t == 0:
        return out
    if k == 0:
        return out.zero_()
    a = _lib.Fp8MmArgs(m, k, t, tag, 1 if token_major else 0, ldw, ldx, ldc, wq.data_ptr(), w_scales.data_ptr(),
                       xq.data_ptr(), x_scales.data_ptr(), out.data_ptr())
    _lib.check(_lib.register_hip_kernel().mss_fp8_mm(a, _stream(wq)), "mss_fp8_mm")
    return out
