"""Drawing tokens from logits on MI355X (HIP kernel behind the C ABI).

``sample_tokens(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> tokens`` —
logits (rows, vocab) float32 or bfloat16, any non-negative strides (the decode step's logits
are the transpose of a (vocab, batch) matrix); uniform (rows,) float32 in [0, 1), the random
numbers, so that a draw can be repeated; tokens (rows,) int64.

A word whose logit is -inf is absent. With the words ordered by logit (ties: the lower index
first) and weights ``w = exp((logit - largest) / temperature)``: top_k > 0 keeps the first
top_k; top_p < 1 keeps of those the words before which less than top_p of their weight lies;
min_p keeps of those the words with ``w >= min_p``; the first word always stays. The token is
the lowest index at which the running weight of the words kept, in index order, exceeds
``uniform`` times their whole weight. A temperature of 0 takes the first word. A row without a
word, or with a NaN, gives -1. Each setting is a number, or a tensor with one value a row
(float32; top_k int32).

Weights are float32 and added as integers, or, for top-p over rows of more than 65536 words, in float64
in a fixed order: tokens are the same from run to run. There is no CPU path.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .selective_scan_hip import _io_tag, _ptr, _require_gpu, _resolved, _stream

__all__ = ["sample_tokens"]


_F32, _I32, _I64 = torch.float32, torch.int32, torch.int64


def _setting(name, v, rows, dtype, low, high):
    """(number, None) or (0, checked per-row tensor)."""
    if isinstance(v, torch.Tensor):
        if v.dtype != dtype or v.shape != (rows,):
            raise ValueError(f"{name} must be a number or a {dtype} tensor of shape ({rows},)")
        return 0, _resolved(v).contiguous()
    if not low <= v <= high:  # a NaN too
        raise ValueError(f"{name} must be between {low} and {high}, got {v}")
    return v, None


def sample_tokens(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    if logits.dim() != 2:
        raise ValueError("logits must be a (rows, vocab) matrix")
    io = _io_tag(logits.dtype, "logits")
    rows, vocab = logits.shape
    if vocab == 0:
        raise ValueError("logits have no words")
    if uniform.dtype != _F32 or uniform.shape != (rows,):
        raise ValueError(f"uniform must be float32 with shape ({rows},)")
    temperature, temperatures = _setting("temperature", temperature, rows, _F32, 0.0, math.inf)
    top_k, top_ks = _setting("top_k", top_k, rows, _I32, 0, 2**31 - 1)
    top_p, top_ps = _setting("top_p", top_p, rows, _F32, 0.0, 1.0)
    min_p, min_ps = _setting("min_p", min_p, rows, _F32, 0.0, 1.0)
    _require_gpu(logits, uniform, temperatures, top_ks, top_ps, min_ps)
    tokens = torch.empty(rows, dtype=_I64, device=logits.device)
    if rows == 0:
        return tokens
    if logits.is_neg() or uniform.is_neg():
        logits, uniform = _resolved(logits), _resolved(uniform)
    uniform = uniform.contiguous()
    sr, sv = logits.stride()
    a = _lib.SampleArgs(rows, vocab, io, top_k, temperature, top_p, min_p, sr if rows > 1 else 0,
                        sv if vocab > 1 else 1, logits.data_ptr(), uniform.data_ptr(), _ptr(temperatures),
                        _ptr(top_ks), _ptr(top_ps), _ptr(min_ps), tokens.data_ptr())
    _lib.check(_lib.register_hip_kernel().mss_sample(a, _stream(logits)), "mss_sample")
    return tokens
