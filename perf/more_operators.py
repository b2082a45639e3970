"""Timed cases of the losses a language model is trained with, and of their gradients.

Three operators:

* ``ce``: ``linear_cross_entropy``, the tied head's softmax cross-entropy from the final norm's
  output and the head's weight, in pieces of the vocabulary, the logits not kept;
* ``lin_distill``: ``linear_distill_loss``, the same head trained towards a teacher's top logits;
* ``distill``: ``distill_loss``, distillation from a teacher's top logits for logits at hand.

A case with ``grad`` is the loss's mean and its gradients; one without is the loss of each token,
as scoring a text or validating takes it. ``listed()`` names twelve cases, ``draw()`` gives more
of the same ranges. ``run`` computes a case in elementary torch operations, or through the
framework where ``own`` is true.
"""
import functools
import math
import os
import sys

import torch

own = False

DEV = "cuda"
IGNORE = -100
MOST_PRODUCT = 16384 * 768 * 50280
MOST_LOGITS = 16384 * 50280
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _ce(name, tokens, width, vocab, dtype="bf16", grad=True, masked=0.1, token_major=False):
    return dict(name=name, kind="ce", tokens=tokens, width=width, vocab=vocab, dtype=dtype, grad=grad, masked=masked,
                token_major=token_major)


def _lin_distill(name, tokens, width, vocab, top, dtype="bf16", grad=True, temperature=2.0, masked=0.1,
                 token_major=False):
    return dict(name=name, kind="lin_distill", tokens=tokens, width=width, vocab=vocab, top=top, dtype=dtype, grad=grad,
                temperature=temperature, masked=masked, token_major=token_major)


def _distill(name, tokens, vocab, top, dtype="bf16", grad=True, temperature=2.0, masked=0.1):
    return dict(name=name, kind="distill", tokens=tokens, vocab=vocab, top=top, dtype=dtype, grad=grad,
                temperature=temperature, masked=masked)


def listed():
    return [
        # The induction-heads task: 8 rows of 256 tokens, width 64, 16 words. Latency.
        _ce("ce_small", 2048, 64, 16, dtype="f32", masked=0.0),
        # Scoring one prompt with the 130M shape: the weight's bytes and few tiles.
        _ce("ce_score", 333, 768, 50280, grad=False, masked=0.0),
        # A float32 run at sizes that no tile divides.
        _ce("ce_odd", 1531, 1000, 10007, dtype="f32"),
        # Validation at a width of 2560: the matrix cores' rate.
        _ce("ce_eval", 8192, 2560, 50280, grad=False, masked=0.0),
        # The 130M training step's loss and gradients, padded tokens among the targets.
        _ce("ce_train", 16384, 768, 50280),
        # A short micro-batch towards a teacher's top 32.
        _lin_distill("lin_distill_short", 256, 768, 50280, 32),
        # The same in float32 at sizes that no tile divides, token-major activations.
        _lin_distill("lin_distill_odd", 777, 333, 32003, 20, dtype="f32", temperature=1.0, token_major=True),
        # A training batch of 130M-shape distillation.
        _lin_distill("lin_distill_train", 8192, 768, 50280, 64),
        # A few rows of logits: latency.
        _distill("distill_few", 8, 50280, 16, masked=0.0),
        # Validation in float32, rows that no vector divides.
        _distill("distill_odd", 1531, 32003, 100, dtype="f32", grad=False, temperature=1.0),
        # A training batch: the logits read, their gradient written.
        _distill("distill_train", 4096, 50280, 64),
        # The 130M step's logits, a small teacher list.
        _distill("distill_large", 16384, 50280, 8, temperature=1.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["ce", "ce", "lin_distill", "distill"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    grad, masked = rng.random() < 0.7, rng.choice([0.0, 0.1, 0.5, 1.0] if rng.random() < 0.3 else [0.0, 0.1])
    temperature = rng.choice([1.0, 2.0, 4.0, 0.7])
    if kind == "distill":
        while True:
            tokens, vocab = _log_int(rng, 1, 16384), _log_int(rng, 16, 131072)
            if tokens * vocab <= MOST_LOGITS:
                break
        case = _distill("", tokens, vocab, min(_log_int(rng, 1, 256), vocab // 2), dtype, grad, temperature, masked)
    else:
        while True:
            tokens, width, vocab = _log_int(rng, 1, 16384), _log_int(rng, 64, 2560), _log_int(rng, 16, 131072)
            if rng.random() < 0.6:  # most models have round widths
                width = width // 64 * 64
            if tokens * width * vocab <= MOST_PRODUCT / (1 if dtype == "bf16" else 8):
                break
        token_major = rng.random() < 0.3
        if kind == "ce":
            case = _ce("", tokens, width, vocab, dtype, grad, masked, token_major)
        else:
            case = _lin_distill("", tokens, width, vocab, min(_log_int(rng, 1, 256), vocab // 2), dtype, grad,
                                temperature, masked, token_major)
    del case["name"]
    return case


# ---------------------------------------------------------------------------- inputs
def _teacher(g, tokens, vocab, top, masked):
    """A teacher's list for each token: different words, their logits in falling order; some lists
    shorter than others (-1), and the masked tokens' empty. The lists' first words too."""
    first = torch.randint(0, vocab, (tokens, 1), generator=g, device=DEV)
    step = torch.randint(1, max(2, vocab // top), (tokens, 1), generator=g, device=DEV)
    ids = (first + step * torch.arange(top, device=DEV)) % vocab
    held = torch.sort(9 * torch.rand(tokens, top, generator=g, device=DEV), dim=1, descending=True).values
    length = torch.where(torch.rand(tokens, 1, generator=g, device=DEV) < 0.1,
                         torch.randint(1, top + 1, (tokens, 1), generator=g, device=DEV), top)
    length = torch.where(torch.rand(tokens, 1, generator=g, device=DEV) < masked, 0, length)
    ids = torch.where(torch.arange(top, device=DEV) < length, ids, -1)
    return ids, held, first


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case)
    tokens, vocab, dtype = case["tokens"], case["vocab"], DTYPES[case["dtype"]]
    if case["kind"] == "ce":
        words = torch.randint(0, vocab, (tokens, 1), generator=g, device=DEV)
        masked = torch.rand(tokens, generator=g, device=DEV) < case["masked"]
        s["targets"] = torch.where(masked, IGNORE, words[:, 0])
    else:
        s["ids"], s["teacher"], words = _teacher(g, tokens, vocab, case["top"], case["masked"])
    if case["kind"] == "distill":
        # A broad body of logits, and the teacher's first word above it.
        x = 2.5 * torch.randn(tokens, vocab, generator=g, device=DEV)
        x.scatter_add_(1, words, 9 * torch.rand(tokens, 1, generator=g, device=DEV))
        s["logits"] = x.to(dtype).requires_grad_(case["grad"])
        return s
    width = case["width"]
    weight = 2.5 / math.sqrt(width) * torch.randn(vocab, width, generator=g, device=DEV)
    # Normed activations that point, some more than others, towards their word.
    x = torch.randn(tokens, width, generator=g, device=DEV)
    x = x + 1.5 * torch.rand(tokens, 1, generator=g, device=DEV) * weight[words[:, 0]]
    x = x / x.square().mean(1, keepdim=True).sqrt()
    x = x.to(dtype)
    s["x"] = (x.t() if case["token_major"] else x.t().contiguous()).detach().requires_grad_(case["grad"])
    s["weight"] = weight.to(dtype).requires_grad_(case["grad"])
    return s


# ---------------------------------------------------------------------------- plain forms
def _log_sum(z):
    top = z.amax(1, keepdim=True)
    return top[:, 0] + torch.exp(z - top).sum(1).log()


def _plain_ce(logits, targets, grad):
    """The tokens' losses, and where `grad` the logits' gradient of their mean."""
    counts = targets != IGNORE
    at = torch.where(counts, targets, 0)[:, None]
    lse = _log_sum(logits)
    loss = torch.where(counts, lse - logits.gather(1, at)[:, 0], 0.0)
    if not grad:
        return loss, None
    share = counts / counts.sum().clamp_min(1)
    d = torch.exp(logits - lse[:, None])
    d.scatter_add_(1, at, torch.full_like(d[:, :1], -1.0))
    return (loss * share).sum(), d.mul_(share[:, None])


def _plain_distill(logits, ids, teacher, temperature, grad):
    held = ids >= 0
    at = torch.where(held, ids, 0)
    z = logits / temperature
    t = torch.where(held, teacher.float() / temperature, -math.inf)
    counts = held.any(1)
    e = torch.where(held, torch.exp(t - t.amax(1, keepdim=True)), 0.0)
    q = e / e.sum(1, keepdim=True).clamp_min(1e-30)
    lse = _log_sum(z)
    # sum of q (log q - log p), log p = z - lse
    gap = q.clamp_min(1e-37).log() - (z.gather(1, at) - lse[:, None])
    loss = temperature ** 2 * torch.where(held, q * gap, 0.0).sum(1)
    if not grad:
        return loss, None
    share = counts / counts.sum().clamp_min(1)
    d = torch.exp(z - lse[:, None])
    d.scatter_add_(1, at, -q)
    return (loss * share).sum(), d.mul_((temperature * share)[:, None])


def _plain(s):
    grad = s["grad"]
    if s["kind"] == "distill":
        loss, d = _plain_distill(s["logits"].detach().float(), s["ids"], s["teacher"], s["temperature"], grad)
        return {"loss": loss, "dlogits": d.to(s["logits"].dtype)} if grad else loss
    x, w = s["x"].detach().float(), s["weight"].detach().float()
    logits = x.t() @ w.t()
    if s["kind"] == "ce":
        loss, d = _plain_ce(logits, s["targets"], grad)
    else:
        loss, d = _plain_distill(logits, s["ids"], s["teacher"], s["temperature"], grad)
    if not grad:
        return loss
    dtype = s["x"].dtype
    return {"loss": loss, "dx": (w.t() @ d.t()).to(dtype), "dweight": (d.t() @ x.t()).to(dtype)}


@functools.cache
def _framework():
    sys.path.insert(0, os.path.join(os.getcwd(), "jax-mambas_amd"))
    from mamba_amd.losses import distill_loss, linear_cross_entropy, linear_distill_loss

    return linear_cross_entropy, linear_distill_loss, distill_loss


def run(s):
    if not own:
        return _plain(s)
    linear_cross_entropy, linear_distill_loss, distill_loss = _framework()
    reduction = "mean" if s["grad"] else "none"
    if s["kind"] == "ce":
        loss = linear_cross_entropy(s["x"], s["weight"], s["targets"], ignore_index=IGNORE, reduction=reduction)
    elif s["kind"] == "lin_distill":
        loss = linear_distill_loss(s["x"], s["weight"], s["ids"], s["teacher"], temperature=s["temperature"],
                                   reduction=reduction)
    else:
        loss = distill_loss(s["logits"], s["ids"], s["teacher"], temperature=s["temperature"], reduction=reduction)
    if not s["grad"]:
        return loss
    if s["kind"] == "distill":
        (d,) = torch.autograd.grad(loss, (s["logits"],))
        return {"loss": loss.detach(), "dlogits": d}
    dx, dw = torch.autograd.grad(loss, (s["x"], s["weight"]))
    return {"loss": loss.detach(), "dx": dx, "dweight": dw}


def work(case):
    tokens, vocab, size = case["tokens"], case["vocab"], DTYPES[case["dtype"]].itemsize
    both = 2 if case["grad"] else 1  # a gradient has its input's size
    lists = 8 * tokens if case["kind"] == "ce" else 12 * tokens * case["top"]
    out = 4 if case["grad"] else 4 * tokens
    if case["kind"] == "distill":
        return {"bytes": tokens * vocab * size * both + lists + out, "flops": 4 * both * tokens * vocab}
    width = case["width"]
    # Products: the logits, and the two gradients from theirs.
    return {"bytes": (tokens + vocab) * width * size * both + lists + out,
            "flops": (6 if case["grad"] else 2) * tokens * vocab * width + 4 * both * tokens * vocab}


# ---------------------------------------------------------------------------- 64 bits
def _exact_part(s, logits, rows, share):
    """The losses of some rows, in float64, and the gradient of `share` times each."""
    temperature = s.get("temperature", 1.0)
    p = torch.softmax(logits / temperature, 1)
    log_p = torch.log_softmax(logits / temperature, 1)
    wanted = torch.zeros_like(p)
    if s["kind"] == "ce":
        at = s["targets"][rows]
        here = (at != IGNORE).nonzero()[:, 0]
        wanted[here, at[here]] = 1.0
    else:
        ids, t = s["ids"][rows], s["teacher"][rows].double() / temperature
        top = torch.where(ids >= 0, t, -torch.inf).max(1, keepdim=True).values
        for k in range(ids.shape[1]):
            here = (ids[:, k] >= 0).nonzero()[:, 0]
            wanted[here, ids[here, k]] += torch.exp(t[here, k] - top[here, 0])
        wanted /= wanted.sum(1, keepdim=True).clamp_min(1e-300)
    some = wanted.sum(1) > 0
    loss = temperature ** 2 * (torch.xlogy(wanted, wanted) - wanted * log_p).sum(1) * some
    return loss, temperature * (p * some[:, None] - wanted) * share[rows, None]


def exact(case, seed):
    s = prepare(case, seed)
    tokens = case["tokens"]
    some = s["targets"] != IGNORE if case["kind"] == "ce" else (s["ids"] >= 0).any(1)
    share = some.double() / max(1, int(some.sum()))
    losses, dlogits, dx, dw = [], [], [], 0.0
    for first in range(0, tokens, 2048):
        rows = slice(first, min(tokens, first + 2048))
        if case["kind"] == "distill":
            loss, d = _exact_part(s, s["logits"].detach()[rows].double(), rows, share)
            if case["grad"]:
                dlogits.append(d)
        else:
            x, w = s["x"].detach()[:, rows].double(), s["weight"].detach().double()
            loss, d = _exact_part(s, torch.mm(x.t(), w.t()), rows, share)
            if case["grad"]:
                dx.append(torch.mm(d, w).t())
                dw = dw + torch.mm(d.t(), x.t())
        losses.append(loss)
        del d
    loss = torch.cat(losses)
    if not case["grad"]:
        return loss
    mean = (loss * share).sum()
    if case["kind"] == "distill":
        return {"loss": mean, "dlogits": torch.cat(dlogits)}
    return {"loss": mean, "dx": torch.cat(dx, 1), "dweight": dw}
