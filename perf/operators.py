"""Timed cases of the operators that serve a language model in 8 bits, and draw its tokens.

Four kinds of case, one for each operator:

* ``norm``: ``add_rmsnorm_fp8``, the residual's addition and the root-mean-square norm of a
  channel-major stream, written as 8-bit floats with a scale for each token and 128 features;
* ``quant``: ``quantize_fp8``, the same 8-bit form of any activation matrix;
* ``mm``: ``fp8_matmul``, a projection in that form: activations scaled by token and block of
  128 features, the weight by blocks of 128 x 128;
* ``sample``: ``sample_tokens``, a token for each row of logits from given random numbers,
  after temperature, top-k, top-p and min-p.

``listed()`` names twelve cases, ``draw()`` gives more of the same ranges. ``run`` computes a
case in elementary torch operations, or through the framework where ``own`` is true.
"""
import functools
import math
import os
import sys

import torch

own = False

DEV = "cuda"
BLOCK = 128
FP8_MAX = 448.0
TINY = 2.0 ** -126  # smallest scale, of a block without a value other than zero
MOST_FLOPS = 2 * 5120 * 1280 * 16384
MOST_STREAM = 2560 * 16384
MOST_LOGITS = 256 * 131072
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _mm(name, m, k, t, out="bf16", token_major=False):
    return dict(name=name, kind="mm", m=m, k=k, t=t, out=out, token_major=token_major)


def _norm(name, f, t, delta="bf16"):
    return dict(name=name, kind="norm", f=f, t=t, delta=delta)


def _quant(name, f, t, dtype="bf16"):
    return dict(name=name, kind="quant", f=f, t=t, dtype=dtype)


def _sample(name, rows, vocab, dtype="f32", top_k=0, top_p=1.0, min_p=0.0, per_row=False):
    return dict(name=name, kind="sample", rows=rows, vocab=vocab, dtype=dtype, top_k=top_k, top_p=top_p,
                min_p=min_p, per_row=per_row)


def listed():
    return [
        # One token of one stream through a block's in-projection (d_model 1280, expand 2, the
        # rows of x and z stacked): the weight's bytes, and latency.
        _mm("mm_step", 5120, 1280, 1),
        # The tied head over a decode batch of the 130M shape: logits in float32, a row a token.
        _mm("mm_head", 50280, 768, 8, out="f32", token_major=True),
        # The out-projection of a prompt, at a length as prompts have it: few tiles.
        _mm("mm_prompt", 1280, 2560, 333),
        # The in-projection of a batch of long prompts: the matrix cores' rate.
        _mm("mm_large", 5120, 1280, 16384),
        # The block entry of a decode batch: latency.
        _norm("norm_step", 1280, 8),
        # A prompt whose length and width no tile divides.
        _norm("norm_odd", 1000, 1531),
        # The block entry of a batch of long prompts: memory bandwidth.
        _norm("norm_large", 1280, 16384),
        # The scan's output of a decode batch, on its way into the out-projection.
        _quant("quant_step", 2560, 8),
        # The same of a batch of long prompts: the largest copy of this kind.
        _quant("quant_large", 2560, 16384),
        # One stream's next token, the usual filters on, logits in bf16 as a bf16 head gives them.
        _sample("sample_one", 1, 50280, dtype="bf16", top_k=50, top_p=0.95),
        # A serving batch in which every request has its own settings.
        _sample("sample_batch", 64, 50280, per_row=True),
        # Many requests over a large vocabulary, nucleus sampling.
        _sample("sample_large", 256, 131072, top_p=0.9, min_p=0.001),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["mm", "mm", "norm", "quant", "sample", "sample"])
    if kind == "mm":
        while True:
            m, k, t = _log_int(rng, 64, 50280), _log_int(rng, 64, 5120), _log_int(rng, 1, 16384)
            if rng.random() < 0.6:  # most models have round widths
                m, k = max(64, m // 64 * 64), max(64, k // 64 * 64)
            if 2 * m * k * t <= MOST_FLOPS and m * t <= 5120 * 16384:
                break
        case = _mm("", m, k, t, rng.choice(["bf16", "bf16", "f32"]), rng.random() < 0.3)
    elif kind in ("norm", "quant"):
        most = 1280 * 16384 if kind == "norm" else MOST_STREAM
        while True:
            f, t = _log_int(rng, 64, 5120), _log_int(rng, 1, 16384)
            if rng.random() < 0.5:
                f = max(64, f // 64 * 64)
            if f * t <= most:
                break
        case = (_norm("", f, t, rng.choice(["bf16", "bf16", "f32", "none"])) if kind == "norm"
                else _quant("", f, t, rng.choice(["bf16", "bf16", "f32"])))
    else:
        while True:
            rows, vocab = _log_int(rng, 1, 512), _log_int(rng, 1000, 262144)
            if rows * vocab <= MOST_LOGITS:
                break
        case = _sample("", rows, vocab, rng.choice(["f32", "bf16"]), rng.choice([0, 0, 1, 20, 50, 1000]),
                       rng.choice([1.0, 0.95, 0.8, 0.5]), rng.choice([0.0, 0.0, 0.02]), rng.random() < 0.4)
    del case["name"]
    return case


# ---------------------------------------------------------------------------- inputs
def _spread(x):
    """(rows, k) 8-bit values in rows that start on 16 bytes, as the framework keeps them."""
    rows, k = x.shape
    held = torch.zeros(rows, -(-k // 16) * 16, dtype=torch.float8_e4m3fn, device=x.device)
    held[:, :k] = x
    return held[:, :k]


def _blocks(x, size):
    """x with its last axis cut into blocks of `size`, filled up with zeros."""
    n = -(-x.shape[-1] // size)
    full = torch.zeros(*x.shape[:-1], n * size, dtype=x.dtype, device=x.device)
    full[..., :x.shape[-1]] = x
    return full.view(*x.shape[:-1], n, size)


def _made_operands(g, m, k, t):
    """A weight in 8 bits with a scale for each 128 x 128 block, activations in 8 bits with one
    for each token and 128 features (some channels far larger than the others)."""
    w = torch.randn(m, k, generator=g, device=DEV) / math.sqrt(k)
    wb = _blocks(_blocks(w, BLOCK).permute(1, 2, 0), BLOCK)  # (k blocks, in the block, m blocks, in the block)
    ws = (wb.abs().amax((1, 3)) / FP8_MAX).clamp_min(TINY)
    wq = (wb / ws[:, None, :, None]).flatten(2).permute(2, 0, 1).flatten(1)[:m, :k].to(torch.float8_e4m3fn)
    del w, wb
    x = torch.randn(t, k, generator=g, device=DEV) * torch.exp(torch.randn(k, generator=g, device=DEV))
    xb = _blocks(x, BLOCK)
    xs = (xb.abs().amax(2) / FP8_MAX).clamp_min(TINY)
    xq = (xb / xs[:, :, None]).flatten(1)[:, :k].to(torch.float8_e4m3fn)
    return dict(wq=_spread(wq), ws=ws.t().contiguous(), xq=_spread(xq), xs=xs.t().contiguous())


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind = case["kind"]
    s = dict(case)
    if kind == "mm":
        s.update(_made_operands(g, case["m"], case["k"], case["t"]))
    elif kind == "norm":
        f, t = case["f"], case["t"]
        width = torch.exp(0.7 * torch.randn(f, 1, generator=g, device=DEV))  # a stream's channels differ in size
        s["h"] = torch.randn(f, t, generator=g, device=DEV) * width
        s["delta"] = None if case["delta"] == "none" else (
            0.3 * torch.randn(f, t, generator=g, device=DEV)).to(DTYPES[case["delta"]])
        s["weight"] = 1 + 0.2 * torch.randn(f, generator=g, device=DEV)
        s["eps"] = 1e-5
    elif kind == "quant":
        f, t = case["f"], case["t"]
        x = torch.randn(f, t, generator=g, device=DEV)
        s["x"] = (x * torch.sigmoid(2 * torch.randn(f, t, generator=g, device=DEV))).to(DTYPES[case["dtype"]])
    else:
        rows, vocab = case["rows"], case["vocab"]
        # Logits as a trained head gives them: a broad body and a few words far above it.
        x = 2.5 * torch.randn(rows, vocab, generator=g, device=DEV)
        at = torch.randint(0, vocab, (rows, 12), generator=g, device=DEV)
        s["logits"] = x.scatter_add(1, at, 9 * torch.rand(rows, 12, generator=g, device=DEV)).to(DTYPES[case["dtype"]])
        s["uniform"] = torch.rand(rows, generator=g, device=DEV)
        s["temperature"], s["top_k"], s["top_p"], s["min_p"] = 0.8, case["top_k"], case["top_p"], case["min_p"]
        if case["per_row"]:
            pick = lambda values: torch.tensor(values, device=DEV)[  # noqa: E731
                torch.randint(0, len(values), (rows,), generator=g, device=DEV)]
            s["temperature"] = pick([0.0, 0.6, 0.8, 1.0, 1.3])
            s["top_k"] = pick([0, 0, 1, 40, 200]).to(torch.int32)
            s["top_p"] = pick([1.0, 0.95, 0.9, 0.5])
            s["min_p"] = pick([0.0, 0.0, 0.02, 0.1])
    return s


# ---------------------------------------------------------------------------- plain forms
def _plain_quantise(x):
    """x (features, tokens) float32 as 8-bit floats (tokens, features) and scales (blocks,
    tokens): the largest magnitude of each token and 128 features becomes 448."""
    f = x.shape[0]
    xb = _blocks(x.t(), BLOCK)
    scales = (xb.abs().amax(2) / FP8_MAX).clamp_min(TINY)
    q = (xb / scales[:, :, None]).flatten(1)[:, :f].to(torch.float8_e4m3fn)
    return q, scales.t().contiguous()


def _plain_matmul(s):
    m, k = s["wq"].shape
    w = s["wq"].float() * s["ws"].repeat_interleave(BLOCK, 0)[:m].repeat_interleave(BLOCK, 1)[:, :k]
    x = s["xq"].float() * s["xs"].repeat_interleave(BLOCK, 0)[:k].t()
    y = x @ w.t() if s["token_major"] else w @ x.t()
    return y.to(DTYPES[s["out"]])


def _plain_norm(s):
    hn = s["h"] if s["delta"] is None else s["h"] + s["delta"].float()
    rstd = 1 / torch.sqrt(hn.square().mean(0) + s["eps"])
    return (hn, *_plain_quantise(hn * rstd * s["weight"][:, None]))


def _column(v, dtype):
    return (v if torch.is_tensor(v) else torch.tensor([v], device=DEV)).to(dtype)[:, None]


def _plain_sample(s):
    x = s["logits"].float()
    rows, vocab = x.shape
    temperature, min_p = _column(s["temperature"], torch.float64), _column(s["min_p"], torch.float64)
    top_k, top_p = _column(s["top_k"], torch.int64), _column(s["top_p"], torch.float64)
    down, order = torch.sort(x, dim=1, descending=True, stable=True)
    weight = torch.exp((down.double() - down[:, :1].double()) / temperature.where(temperature > 0, 1.0))
    rank = torch.arange(vocab, device=x.device)[None]
    weight = weight * ((top_k <= 0) | (rank < top_k))
    mass = weight.cumsum(1)
    keep = ((mass - weight < top_p * mass[:, -1:]) & (weight >= min_p)) | (rank == 0)
    kept = torch.zeros_like(weight).scatter_(1, order, weight * keep)  # in the words' order
    mass = kept.cumsum(1)
    drawn = (mass > s["uniform"].double()[:, None] * mass[:, -1:]).to(torch.uint8).argmax(1)
    return torch.where(temperature[:, 0] > 0, drawn, order[:, 0])


@functools.cache
def _framework():
    sys.path.insert(0, os.path.join(os.getcwd(), "jax-mambas_amd"))
    from mamba_amd.fp8 import add_rmsnorm_fp8, fp8_matmul, quantize_fp8
    from mamba_amd.sampling import sample_tokens

    return add_rmsnorm_fp8, fp8_matmul, quantize_fp8, sample_tokens


def run(s):
    kind = s["kind"]
    if own:
        add_rmsnorm_fp8, fp8_matmul, quantize_fp8, sample_tokens = _framework()
        if kind == "mm":
            return fp8_matmul(s["wq"], s["ws"], s["xq"], s["xs"], out_dtype=DTYPES[s["out"]],
                              token_major=s["token_major"])
        if kind == "norm":
            hn, q, scales = add_rmsnorm_fp8(s["h"], s["delta"], s["weight"], s["eps"])
            return {"hn": hn, "q": q, "scales": scales}
        if kind == "quant":
            q, scales = quantize_fp8(s["x"])
            return {"q": q, "scales": scales}
        return sample_tokens(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"],
                             top_p=s["top_p"], min_p=s["min_p"])
    if kind == "mm":
        return _plain_matmul(s)
    if kind == "norm":
        hn, q, scales = _plain_norm(s)
        return {"hn": hn, "q": q, "scales": scales}
    if kind == "quant":
        q, scales = _plain_quantise(s["x"].float())
        return {"q": q, "scales": scales}
    return _plain_sample(s)


def work(case):
    kind = case["kind"]
    if kind == "mm":
        m, k, t = case["m"], case["k"], case["t"]
        kb, mb = -(-k // BLOCK), -(-m // BLOCK)
        return {"bytes": m * k + t * k + 4 * kb * (t + mb) + m * t * DTYPES[case["out"]].itemsize,
                "flops": 2 * m * k * t}
    if kind == "norm":
        f, t = case["f"], case["t"]
        # The sum is written only where there is a delta: without one it is h itself.
        delta = 0 if case["delta"] == "none" else 4 + DTYPES[case["delta"]].itemsize
        return {"bytes": f * t * (4 + delta + 1) + 4 * f + 4 * -(-f // BLOCK) * t, "flops": 7 * f * t}
    if kind == "quant":
        f, t = case["f"], case["t"]
        return {"bytes": f * t * (DTYPES[case["dtype"]].itemsize + 1) + 4 * -(-f // BLOCK) * t, "flops": 3 * f * t}
    rows, vocab = case["rows"], case["vocab"]
    return {"bytes": rows * vocab * DTYPES[case["dtype"]].itemsize + 12 * rows, "flops": 5 * rows * vocab}


# ---------------------------------------------------------------------------- 64 bits
def _to_fp8(v):
    """float64 values of magnitude at most 448 rounded to the nearest 8-bit float (4 exponent
    and 3 fraction bits, ties to even), as float64."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def _exact_quantise(y):
    f, t = y.shape
    q = torch.empty(t, f, dtype=torch.float64, device=y.device)
    scales = torch.empty(-(-f // BLOCK), t, dtype=torch.float64, device=y.device)
    for b in range(scales.shape[0]):
        part = y[b * BLOCK:(b + 1) * BLOCK]
        scales[b] = (part.abs().max(0).values / FP8_MAX).clamp_min(TINY)
        q[:, b * BLOCK:(b + 1) * BLOCK] = _to_fp8((part / scales[b]).t())
    return q, scales


def _exact_matmul(s):
    m, k = s["wq"].shape
    y = torch.zeros(m, s["xq"].shape[0], dtype=torch.float64, device=DEV)
    for b in range(s["ws"].shape[1]):
        c = slice(b * BLOCK, min(k, (b + 1) * BLOCK))
        rows = s["ws"][:, b].double()[torch.arange(m, device=DEV) // BLOCK]
        y += (s["wq"][:, c].double() * rows[:, None]) @ (s["xq"][:, c].double() * s["xs"][b].double()[:, None]).t()
    return y.t() if s["token_major"] else y


def _exact_sample(s):
    """Row by row: the words from the most likely on, those that the filters leave, the draw."""
    rows = s["logits"].shape[0]
    at = lambda v, r: float(v[r]) if torch.is_tensor(v) else float(torch.tensor(v, dtype=torch.float32).item())  # noqa: E731
    settings = {n: s[n].cpu() if torch.is_tensor(s[n]) else s[n] for n in ("temperature", "top_k", "top_p", "min_p")}
    uniform, tokens = s["uniform"].double().cpu(), []
    for r in range(rows):
        x = s["logits"][r].double()
        temperature, k = at(settings["temperature"], r), int(at(settings["top_k"], r))
        if temperature <= 0:
            tokens.append(int((x == x.max()).nonzero()[0, 0]))
            continue
        p = torch.softmax(x / temperature, 0)
        words = torch.argsort(-x, stable=True)
        words = words[:k] if k > 0 else words
        q = p[words] / p[words].sum()
        before = torch.cat([q.new_zeros(1), q.cumsum(0)[:-1]])
        n = max(1, int((before < at(settings["top_p"], r)).sum()))
        n = max(1, min(n, int((q[:n] >= at(settings["min_p"], r) * q[0]).sum())))
        words = words[:n].sort().values
        q = p[words] / p[words].sum()
        tokens.append(int(words[min(n - 1, int((q.cumsum(0) <= uniform[r]).sum()))]))
    return torch.tensor(tokens, dtype=torch.int64)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "mm":
        return _exact_matmul(s)
    if case["kind"] == "sample":
        return _exact_sample(s)
    if case["kind"] == "quant":
        q, scales = _exact_quantise(s["x"].double())
        return {"q": q, "scales": scales}
    hn = s["h"].double() if s["delta"] is None else s["h"].double() + s["delta"].double()
    y = hn / torch.sqrt(torch.mean(hn * hn, 0) + s["eps"]) * s["weight"].double()[:, None]
    q, scales = _exact_quantise(y)
    return {"hn": hn, "q": q, "scales": scales}
