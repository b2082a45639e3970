"""Serving a MambaLM with 8-bit projections: prompt, single tokens, and the draw of the next one.

``Fp8LM(model)`` takes a ``mamba1.MambaLM`` (its blocks: mamba/mamba1.py:216-363) and holds its in-, gate- and
out-projections and the tied head in the 8-bit form of ``mamba_amd.fp8``, written once from the
float32 masters; the small S6 projections in bf16; copies of what else it reads (the embedding,
norms, conv and S6 vectors). Every norm writes the 8-bit operand of
the product behind it (``add_rmsnorm_fp8``), the scan's output is quantised for the
out-projection (``quantize_fp8``), and logits are float32.

``prefill(tokens) -> (logits, caches)`` — tokens (B, L) int64, right-aligned; logits (B, vocab) of
the last position, and each block's decode state.

``step(token, caches) -> logits`` — token (B,) int64; caches update in place. A token of -1 (what
``sample_tokens`` gives for a row without a word or with a NaN) makes its row's logits NaN, in this step and
those that follow, so that the row's draws stay -1.

``generate(tokens, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, graph=True) -> drawn`` —
draws uniforms.shape[0] tokens a row after the prompt with ``sample_tokens``: uniforms (n, B)
float32 in [0, 1), settings numbers or one a row; drawn (n, B) int64. With ``graph`` the decode
step and its draw are captured once in a HIP graph and replayed. A row whose draw is -1 stays at -1.

Weights of the model that change afterwards are not seen, none of them, until ``refresh()``, which writes
the held ones where they lie (a graph captured from ``step`` goes on with the new ones). Inference
only; there is no CPU path.
"""
from __future__ import annotations

import copy

import torch
import torch.nn as nn
import torch.nn.functional as F

from .conv1d_hip import causal_conv1d_fn
from .decode import causal_conv1d_update
from .fp8 import add_rmsnorm_fp8, fp8_matmul, quantize_fp8, quantize_fp8_weight
from .mamba1 import MambaLM, ShadowWeights
from .sampling import sample_tokens
from .selective_scan_hip import _require_gpu

__all__ = ["Fp8LM"]


_SHADOWED = ("x_proj", "dt_proj")  # of an S6: held in bf16


class _Block:
    """A block's weights as they are served, but for those _SHADOWED."""

    def __init__(self, blk, A):
        self.norm, self.eps = blk.norm.weight.clone(), blk.norm.eps
        self.in_z = quantize_fp8_weight(torch.cat([blk.in_proj, blk.z_proj]))
        self.out = quantize_fp8_weight(blk.out_proj)
        self.conv_weight, self.conv_bias, self.A = blk.conv_weight.clone(), blk.conv_bias.clone(), A.clone()
        # An S6 with parameters of its own; the projections stay the model's, by which their copies are found.
        self.s6 = copy.copy(blk.s6)
        self.s6._parameters = {k: p if p is None or k in _SHADOWED else nn.Parameter(p.detach().clone(), requires_grad=False)
                               for k, p in blk.s6._parameters.items()}

    def tensors(self):
        return [self.norm, *self.in_z, *self.out, self.conv_weight, self.conv_bias, self.A,
                *(p for k, p in self.s6.named_parameters() if k not in _SHADOWED)]


class Fp8LM:
    def __init__(self, model):
        if not isinstance(model, MambaLM):
            raise TypeError("model must be a MambaLM")
        _require_gpu(model.embedding)
        self.model = model
        self._small = ShadowWeights([getattr(b.s6, w) for b in model.blocks for w in _SHADOWED])
        self._blocks = None
        self.refresh()

    @torch.no_grad()
    def refresh(self):
        """Writes every weight that is held from the model's."""
        m = self.model
        # (the embedding has one row more, of NaN, for the token -1)
        none = torch.full_like(m.embedding[:1], float("nan"))
        new = [torch.cat([m.embedding, none]), *quantize_fp8_weight(m.embedding), m.final_norm.weight.clone()]
        matrices = m.a_matrices()
        if self._blocks is None:
            self._ends = new
            self._blocks = [_Block(b, A) for b, A in zip(m.blocks, matrices)]
        else:
            torch._foreach_copy_(self._ends, new)
            for mine, b, A in zip(self._blocks, m.blocks, matrices):
                torch._foreach_copy_(mine.tensors(), _Block(b, A).tensors())
        # (the masters may have been replaced, or changed behind autograd's version counter)
        for mine, b in zip(self._blocks, m.blocks):
            for k in _SHADOWED:
                mine.s6._parameters[k] = b.s6._parameters[k]
        self._small.rebind([getattr(b.s6, w) for b in m.blocks for w in _SHADOWED])
        self._small.refresh(torch.bfloat16)

    def _logits(self, h, delta):
        _, *head, norm = self._ends
        _, q, s = add_rmsnorm_fp8(h, delta, norm, self.model.final_norm.eps)
        return fp8_matmul(*head, q, s, out_dtype=torch.float32, token_major=True)

    @torch.no_grad()
    def prefill(self, tokens):
        batch, length = tokens.shape
        if length == 0:
            raise ValueError("the prompt has no tokens")
        h = self._ends[0][tokens.reshape(-1)].t().contiguous()  # (d_model, B L)
        delta, caches = None, []
        for blk in self._blocks:
            h, q, s = add_rmsnorm_fp8(h, delta, blk.norm, blk.eps)
            xz = fp8_matmul(*blk.in_z, q, s)
            di, k = blk.conv_weight.shape
            rows = xz.view(2 * di, batch, length).permute(1, 0, 2)
            xin, z = rows[:, :di], xz[di:]
            u = causal_conv1d_fn(xin, blk.conv_weight, blk.conv_bias)
            y = blk.s6(u.permute(1, 0, 2).reshape(di, batch * length), batch, z=z, weights=self._small)
            tail = xin[:, :, max(0, length - (k - 1)):]
            conv = F.pad(tail, (k - 1 - tail.shape[2], 0)).contiguous()
            caches.append({"conv": conv, "ssm": blk.s6.last_state, "A": blk.A})
            blk.s6.last_state = None
            delta = fp8_matmul(*blk.out, *quantize_fp8(y))
        last = slice(length - 1, None, length)
        return self._logits(h[:, last].contiguous(), delta[:, last].contiguous()), caches

    @torch.no_grad()
    def step(self, token, caches):
        h = self._ends[0][token].t().contiguous()  # (d_model, B)
        delta = None
        for blk, cache in zip(self._blocks, caches):
            h, q, s = add_rmsnorm_fp8(h, delta, blk.norm, blk.eps)
            xz = fp8_matmul(*blk.in_z, q, s)
            di = blk.conv_weight.shape[0]
            u = causal_conv1d_update(cache["conv"], xz[:di].t(), blk.conv_weight, blk.conv_bias).t()
            y = blk.s6.step(u, xz[di:], cache["ssm"], self._small, cache["A"])
            delta = fp8_matmul(*blk.out, *quantize_fp8(y))
        return self._logits(h, delta)

    @torch.no_grad()
    def generate(self, tokens, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, graph=True):
        if uniforms.dim() != 2 or uniforms.shape[1] != tokens.shape[0]:
            raise ValueError(f"uniforms must be (steps, {tokens.shape[0]})")
        n = uniforms.shape[0]
        drawn = torch.empty(n, tokens.shape[0], dtype=torch.int64, device=tokens.device)
        if n == 0:
            return drawn
        settings = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        logits, caches = self.prefill(tokens)
        drawn[0] = sample_tokens(logits, uniforms[0], **settings)
        if n <= 2 or not graph:
            for i in range(1, n):
                drawn[i] = sample_tokens(self.step(drawn[i - 1], caches), uniforms[i], **settings)
            return drawn
        # The first step runs eagerly (its launches are what a capture needs warm), the rest as a graph.
        drawn[1] = sample_tokens(self.step(drawn[0], caches), uniforms[1], **settings)
        token, uniform = drawn[1].clone(), uniforms[2].clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            token.copy_(sample_tokens(self.step(token, caches), uniform, **settings))
        for i in range(2, n):
            uniform.copy_(uniforms[i])
            g.replay()
            drawn[i] = token
        return drawn
