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
block of 128 features summed on the matrix cores and scaled in float32, rounded to out_dtype
(bfloat16 or float32) once.

A NaN or infinity makes what its block stands for NaN. Inference only (no autograd); there is no
CPU path.
"""
from __future__ import annotations

import torch

from . import _lib
from .selective_scan_hip import _io_tag, _ptr, _require_gpu, _stream

__all__ = ["quantize_fp8", "add_rmsnorm_fp8", "quantize_fp8_weight", "fp8_matmul"]

_BLOCK = _lib.MSS_FP8_BLOCK
FP8 = torch.float8_e4m3fn


def _blocks(n):
    return -(-n // _BLOCK)


def _empty_rows(rows, cols, device):
    """An uninitialised (rows, cols) 8-bit matrix whose rows start on 16 bytes."""
    if cols % 16 == 0:
        return torch.empty((rows, cols), dtype=FP8, device=device)
    return torch.empty((rows, -(-cols // 16) * 16), dtype=FP8, device=device)[:, :cols]


def _row_stride(q, cols):
    """The row stride of an 8-bit matrix (one that a single row may have, where it has one row)."""
    return q.stride(0) if q.shape[0] > 1 else -(-cols // 16) * 16


def _no_grad_needed(*tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("the 8-bit operators are for inference: call them under torch.no_grad()")


def quantize_fp8(x):
    if x.ndim != 2:
        raise ValueError("x must be a (features, tokens) matrix")
    io = _io_tag(x.dtype, "x")
    _no_grad_needed(x)
    _require_gpu(x)
    f, t = x.shape
    q = _empty_rows(t, f, x.device)
    scales = torch.empty((_blocks(f), t), dtype=torch.float32, device=x.device)
    if f == 0 or t == 0:
        return q, scales
    sf, st = x.stride()
    a = _lib.QuantFp8Args(features=f, tokens=t, io_dtype=io, stride_f=sf, stride_t=st, ldq=_row_stride(q, f),
                          x=x.data_ptr(), q=q.data_ptr(), scales=scales.data_ptr())
    lib = _lib.register_hip_kernel()
    _lib.check(lib.mss_quant_fp8(a, _stream(x)), "mss_quant_fp8")
    return q, scales


def add_rmsnorm_fp8(h, delta, weight, eps=1e-5):
    if h.dtype != torch.float32 or h.ndim != 2:
        raise TypeError("h must be a float32 (features, tokens) matrix")
    f, t = h.shape
    if weight.dtype != torch.float32 or tuple(weight.shape) != (f,):
        raise ValueError(f"weight must be float32 with shape ({f},)")
    if delta is not None and delta.shape != h.shape:
        raise ValueError("delta must have h's shape")
    tag = _lib.MSS_F32 if delta is None else _io_tag(delta.dtype, "delta")
    if f == 0:
        raise ValueError("h has no features")
    _no_grad_needed(h, delta, weight)
    _require_gpu(h, delta, weight)
    h, weight = h.contiguous(), weight.contiguous()
    delta = None if delta is None else delta.contiguous()
    q = _empty_rows(t, f, h.device)
    scales = torch.empty((_blocks(f), t), dtype=torch.float32, device=h.device)
    hn = h if delta is None else torch.empty_like(h)
    if t == 0:
        return hn, q, scales
    a = _lib.NormFp8Args(features=f, tokens=t, delta_dtype=tag, eps=float(eps), ldq=_row_stride(q, f),
                         h=h.data_ptr(), delta=_ptr(delta), weight=weight.data_ptr(), hn=hn.data_ptr(),
                         q=q.data_ptr(), scales=scales.data_ptr())
    lib = _lib.register_hip_kernel()
    _lib.check(lib.mss_norm_fp8(a, _stream(h)), "mss_norm_fp8")
    return hn, q, scales


def quantize_fp8_weight(w):
    if w.ndim != 2 or (w.shape[1] > 1 and w.stride(1) != 1):
        raise ValueError("w must be a (M, K) matrix with contiguous rows")
    io = _io_tag(w.dtype, "w")
    _no_grad_needed(w)
    _require_gpu(w)
    m, k = w.shape
    q = _empty_rows(m, k, w.device)
    scales = torch.empty((_blocks(m), _blocks(k)), dtype=torch.float32, device=w.device)
    if m == 0 or k == 0:
        return q, scales
    a = _lib.QuantFp8WeightArgs(M=m, K=k, io_dtype=io, ldw=w.stride(0) if m > 1 else k, ldq=_row_stride(q, k),
                                w=w.data_ptr(), q=q.data_ptr(), scales=scales.data_ptr())
    lib = _lib.register_hip_kernel()
    _lib.check(lib.mss_quant_fp8_weight(a, _stream(w)), "mss_quant_fp8_weight")
    return q, scales


def _check_rows(name, q, k=None):
    if q.dtype != FP8 or q.ndim != 2:
        raise TypeError(f"{name} must be a float8_e4m3fn matrix")
    if k is not None and q.shape[1] != k:
        raise ValueError(f"{name} must have {k} columns, got {q.shape[1]}")
    rows, cols = q.shape
    if rows and cols and (cols > 1 and q.stride(1) != 1 or rows > 1 and q.stride(0) % 16 != 0 or q.data_ptr() % 16 != 0):
        raise ValueError(f"{name} must have contiguous rows that start on 16 bytes")


def fp8_matmul(wq, w_scales, xq, x_scales, out_dtype=torch.bfloat16, token_major=False, out=None):
    _check_rows("wq", wq)
    (m, k), t = wq.shape, xq.shape[0]
    _check_rows("xq", xq, k)
    for name, s, shape in (("w_scales", w_scales, (_blocks(m), _blocks(k))), ("x_scales", x_scales, (_blocks(k), t))):
        if s.dtype != torch.float32 or tuple(s.shape) != shape or not s.is_contiguous():
            raise ValueError(f"{name} must be a contiguous float32 tensor of shape {shape}")
    shape = (t, m) if token_major else (m, t)
    if out is None:
        out = torch.empty(shape, dtype=out_dtype, device=wq.device)
    elif tuple(out.shape) != shape or out.dtype != out_dtype or (shape[1] > 1 and out.stride(1) != 1):
        raise ValueError(f"out must be {out_dtype} of shape {shape} with contiguous rows")
    tag = _io_tag(out_dtype, "out_dtype")
    _require_gpu(wq, w_scales, xq, x_scales, out)
    if m == 0 or t == 0:
        return out
    if k == 0:
        return out.zero_()
    a = _lib.Fp8MmArgs(M=m, K=k, T=t, out_dtype=tag, token_major=int(bool(token_major)), ldw=_row_stride(wq, k),
                       ldx=_row_stride(xq, k), ldc=out.stride(0) if shape[0] > 1 else shape[1], W=wq.data_ptr(),
                       w_scales=w_scales.data_ptr(), X=xq.data_ptr(), x_scales=x_scales.data_ptr(), C=out.data_ptr())
    lib = _lib.register_hip_kernel()
    _lib.check(lib.mss_fp8_mm(a, _stream(wq)), "mss_fp8_mm")
    return out
