"""The language model's losses that keep no logits (MambaLM.loss, MambaLM.distill_loss): the whole model in
float32 against the float64 oracle with the losses' definitions, in bfloat16 with float32 masters and their
copies, and as a captured training step.

float32 within the model tests' bounds (1e-4 of a tensor's largest gradient, 1e-5 of the loss); bfloat16
within theirs (2e-2, 2e-3).
"""
import pytest
import torch
import torch.nn.functional as F

from mamba_amd.lm_ops import GradHolder, cross_entropy
from mamba_amd.mamba1 import GraphedTrainStep, MambaLM, _TiedHeadMM
from mamba_amd.optim import AdamW
from oracle import mamba1_torch as ref

VOCAB, WIDTH, LAYERS, RANK, STATES = 97, 64, 2, 4, 16


def _model():
    torch.manual_seed(3)
    m = MambaLM(VOCAB, WIDTH, LAYERS, 2, STATES, RANK, 4, device="cuda")
    with torch.no_grad():
        m.embedding.mul_(20)  # logits of a trained model's size
    return m


def _batch(b=3, length=40, top=6):
    g = torch.Generator().manual_seed(4)
    tokens = torch.randint(0, VOCAB, (b, length), generator=g)
    targets = torch.roll(tokens, -1, 1)
    targets[:, -1] = -100
    targets[1, :20] = -100  # a prompt
    ids = torch.stack([torch.randperm(VOCAB, generator=g)[:top] for _ in range(b * length)]).view(b, length, top)
    ids[0, 3:9] = -1
    ids[:, :, -1] = -1
    return tokens, targets, ids, 2 * torch.randn(b, length, top, generator=g)


def _oracle_distill(logits, ids, teacher, temperature):
    ids, teacher = ids.flatten(0, 1), teacher.flatten(0, 1).double()
    log_p = torch.log_softmax(logits / temperature, 1)
    live = (ids >= 0).any(1)
    total = 0.0
    for r in live.nonzero()[:, 0]:
        at = ids[r] >= 0
        q = torch.softmax(teacher[r][at] / temperature, 0)
        total = total + temperature ** 2 * (q * (q.log() - log_p[r][ids[r][at]])).sum()
    return total / int(live.sum())


class _Gather(torch.autograd.Function):
    """The embedding of embed_cm, with its holder, on the CPU."""

    @staticmethod
    def forward(ctx, table, tokens, holder):
        ctx.save_for_backward(tokens)
        ctx.holder, ctx.shape = holder, table.shape
        return table[tokens].t().contiguous()

    @staticmethod
    def backward(ctx, dh):
        de = ctx.holder.take()
        de = torch.zeros(ctx.shape) if de is None else de
        return de.index_add_(0, ctx.saved_tensors[0], dh.t()), None, None


def test_a_holder_s_gradient_is_of_one_pass():
    """A pass for another parameter's gradient runs the heads and not the embedding: the next one starts anew. Whole numbers,
    whose sums are exact."""
    g = torch.Generator().manual_seed(1)
    table = torch.randint(-4, 5, (11, 6), generator=g).float().requires_grad_(True)
    middle = torch.randint(-2, 3, (6, 6), generator=g).float().requires_grad_(True)
    tokens = torch.randint(0, 11, (9,), generator=g)
    heads = [torch.randint(-2, 3, (9, 11), generator=g).float() for _ in range(2)]

    def losses(held):
        holder = GradHolder()
        h = _Gather.apply(table, tokens, holder) if held else table[tokens].t()
        x = middle @ h
        return [((_TiedHeadMM.apply(x, table, table.detach(), holder) if held else x.t() @ table.t()) * w).sum() for w in heads]

    leaves = (table, middle)
    soft, hard = losses(False)
    want = {"both": torch.autograd.grad(soft + hard, leaves, retain_graph=True),
            "soft": torch.autograd.grad(soft, leaves, retain_graph=True), "hard": torch.autograd.grad(hard, leaves)}
    soft, hard = losses(True)
    loss = {"both": soft + hard, "soft": soft, "hard": hard}
    for name in ("both", "soft", "hard", "both"):
        for other in ("soft", "both"):  # what these leave in the holder is nobody's
            (got,) = torch.autograd.grad(loss[other], (middle,), retain_graph=True)
            assert torch.equal(got, want[other][1])
        for got, exact in zip(torch.autograd.grad(loss[name], leaves, retain_graph=True), want[name]):
            assert torch.equal(got, exact), name


def test_a_holder_keeps_one_gradient_of_passes_that_leave_it():
    """Passes for another parameter's gradient, over and over: what they leave does not pile up."""
    g = torch.Generator().manual_seed(5)
    table, middle = torch.randn(11, 6, generator=g).requires_grad_(True), torch.randn(6, 6, generator=g).requires_grad_(True)
    holder = GradHolder()
    x = middle @ _Gather.apply(table, torch.arange(9), holder)
    loss = sum(_TiedHeadMM.apply(x, table, table.detach(), holder).square().sum() for _ in range(2))
    for _ in range(5):
        torch.autograd.grad(loss, (middle,), retain_graph=True)
        assert len(holder._parts) == 1
    torch.autograd.grad(loss, (table, middle), retain_graph=True)
    assert holder.grad is None


@pytest.mark.parametrize("inside", ["heads", "one head", "gather", "both"])
def test_a_holder_across_the_passes_of_checkpoints(inside):
    """A checkpoint with re-entry runs a pass of its own within the backward pass."""
    from torch.utils.checkpoint import checkpoint
    g = torch.Generator().manual_seed(2)
    table = torch.randint(-4, 5, (11, 6), generator=g).float().requires_grad_(True)
    middle = torch.randint(-2, 3, (6, 6), generator=g).float().requires_grad_(True)
    tokens = torch.randint(0, 11, (9,), generator=g)
    weights = [torch.randint(-2, 3, (9, 11), generator=g).float() for _ in range(2)]
    again = lambda f, *a: checkpoint(f, *a, use_reentrant=True)

    def loss(held):
        holder = GradHolder()
        gather = lambda t: _Gather.apply(t, tokens, holder)
        heads = [lambda x, w=w: (_TiedHeadMM.apply(x, table, table.detach(), holder) * w).sum() for w in weights]
        if not held:
            x = middle @ table[tokens].t()
            return sum(((x.t() @ table.t()) * w).sum() for w in weights)
        if inside == "both":
            return again(lambda m: sum(f(m @ gather(table)) for f in heads), middle)
        x = middle @ (again(gather, table) if inside == "gather" else gather(table))
        if inside == "heads":
            return sum(again(f, x) for f in heads)
        return (again(heads[0], x) if inside == "one head" else heads[0](x)) + heads[1](x)

    def grads(held):
        table.grad = middle.grad = None
        loss(held).backward()
        return table.grad, middle.grad

    want = grads(False)
    for _ in range(2):
        for a, b in zip(grads(True), want):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_model_losses_match_the_oracle(act):
    print(f"case model losses {act}", flush=True)
    tokens, targets, ids, teacher = _batch()
    model = _model()
    adt = torch.float32 if act == "f32" else torch.bfloat16
    dev = [t.cuda() for t in (tokens, targets, ids, teacher)]
    ce = model.loss(dev[0], dev[1], act_dtype=adt)
    kd = model.distill_loss(dev[0], dev[2], dev[3], temperature=2.0, act_dtype=adt)
    (0.5 * ce + 0.25 * kd).backward()
    torch.cuda.synchronize()
    p = {k: v.detach().cpu().double().requires_grad_(True) for k, v in model.state_dict().items()}
    logits = ref.mamba_lm(p, tokens, LAYERS, RANK, STATES, True, seq_scan=True)
    want_ce = F.cross_entropy(logits, targets.reshape(-1), ignore_index=-100)
    want_kd = _oracle_distill(logits, ids, teacher, 2.0)
    (0.5 * want_ce + 0.25 * want_kd).backward()
    lt, gt = (1e-5, 1e-4) if act == "f32" else (2e-3, 2e-2)
    print(f"  {ce.item():.6f} {want_ce.item():.6f} {kd.item():.6f} {want_kd.item():.6f}", flush=True)
    assert abs(ce.item() - want_ce.item()) <= lt * want_ce.item()
    assert abs(kd.item() - want_kd.item()) <= lt * want_kd.item()
    for k, v in model.named_parameters():
        want = p[k].grad
        err, scale = float((v.grad.cpu().double() - want).abs().max()), float(want.abs().max())
        print(f"  grad {k:28s} max|g|={scale:.3e} max_err={err:.3e}", flush=True)
        assert err <= gt * scale + 1e-7, k


@pytest.mark.gpu
def test_model_losses_options():
    """Lengths, losses a token, casts instead of kept copies; no gradients."""
    tokens, targets, ids, teacher = (t.cuda() for t in _batch())
    model = _model()
    lens = torch.tensor([40, 33, 7], dtype=torch.int32, device="cuda")
    past = torch.arange(40, device="cuda")[None] >= lens[:, None]
    t = torch.where(past, -100, targets)
    with torch.no_grad():
        rows = model.loss(tokens, t, seq_lens=lens, reduction="none").view(3, 40)
        assert bool((rows[t == -100] == 0).all()) and bool((rows[t != -100] > 0).all())
        mean = model.loss(tokens, t, seq_lens=lens)
        # the float32 mean of up to 120 values against the kernel's
        assert abs(float(mean) - float(rows.double().sum() / (t != -100).sum())) <= 2.0 ** -23 * float(mean)
        assert torch.equal(model.loss(tokens, t, seq_lens=lens, shadow_weights=False), mean)
        other = model.distill_loss(tokens, ids, teacher, seq_lens=lens, reduction="sum")
        assert torch.equal(other, model.distill_loss(tokens, ids, teacher, seq_lens=lens, reduction="sum", shadow_weights=False))


@pytest.mark.gpu
def test_training_steps_graph_matches_eager():
    """Steps with both losses eagerly, and the captured step of the cross-entropy against eager ones."""
    tokens, targets, ids, teacher = (t.cuda() for t in _batch())
    m = _model()
    o = AdamW(m.parameters(), lr=1e-3, shadows=m.shadow_weights)
    first = None
    for _ in range(3):
        o.zero_grad(set_to_none=True)
        soft, hard = m.distill_loss(tokens, ids, teacher, temperature=2.0, targets=targets)
        loss = hard + 0.5 * soft
        loss.backward()
        if first is None:  # one pass for both against a pass for each: the sums' order apart
            first = {k: v.grad.clone() for k, v in m.named_parameters()}
            m.zero_grad(set_to_none=True)
            (m.loss(tokens, targets) + 0.5 * m.distill_loss(tokens, ids, teacher, temperature=2.0)).backward()
            for k, v in m.named_parameters():
                assert float((v.grad - first[k]).abs().max()) <= 2e-2 * float(v.grad.abs().max()), k
        assert all(v.grad is not None and bool(torch.isfinite(v.grad).all()) for v in m.parameters())
        o.step()
    del loss

    def fresh():
        a = _model()
        return a, AdamW(a.parameters(), lr=1e-3, shadows=a.shadow_weights)

    m_e, o_e = fresh()
    eager = []
    for _ in range(5):
        o_e.zero_grad(set_to_none=True)
        loss = m_e.loss(tokens, targets)
        loss.backward()
        o_e.step()
        eager.append(loss.item())
    del loss
    m_g, o_g = fresh()
    gs = GraphedTrainStep(m_g, o_g, None, tokens, targets, warmup=2)
    torch.cuda.synchronize()
    graph = []
    for _ in range(3):
        graph.append(gs.step().item())
        torch.cuda.synchronize()
        _ = (m_g.embedding.sum() * 0).item()  # eager work between replays
    print("  eager", eager, "graph", graph, flush=True)
    for a, b in zip(eager[2:], graph):
        assert abs(a - b) <= 2e-3 * abs(a), (a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["loss", "pair", "logits"])
def test_gradients_after_a_pass_for_one_parameter(which):
    """Another parameter's gradient alone, then all of them: as without the first pass, to the bit."""
    tokens, targets, ids, teacher = (t.cuda() for t in _batch())
    grads = []
    for first in (False, True):
        m = _model()
        if which == "loss":
            loss = m.loss(tokens, targets)
        elif which == "pair":
            loss = sum(m.distill_loss(tokens, ids, teacher, temperature=2.0, targets=targets))
        else:
            loss = cross_entropy(m(tokens), targets.reshape(-1).clamp_min(0))
        if first:
            name, some = next((k, v) for k, v in m.named_parameters() if "blocks.1" in k)
            (alone,) = torch.autograd.grad(loss, (some,), retain_graph=True)
        loss.backward()
        grads.append({k: v.grad for k, v in m.named_parameters()})
    assert torch.equal(alone, grads[1][name])
    for k in grads[0]:
        assert torch.equal(grads[0][k], grads[1][k]), k


@pytest.mark.gpu
@pytest.mark.parametrize("way", ["cpu", "checkpoint"])
@pytest.mark.parametrize("act", ["f32", "bf16"])
def test_model_losses_with_what_they_save_elsewhere(way, act):
    """Offloaded, or made again by a checkpoint: the gradients of a plain pass, to the bit."""
    from torch.utils.checkpoint import checkpoint
    tokens, targets, ids, teacher = (t.cuda() for t in _batch())
    adt = torch.float32 if act == "f32" else torch.bfloat16
    grads = []
    for elsewhere in (False, True):
        m = _model()
        run = lambda: 0.7 * sum(m.distill_loss(tokens, ids, teacher, temperature=2.0, targets=targets, act_dtype=adt))
        if not elsewhere:
            loss = run()
        elif way == "checkpoint":
            loss = checkpoint(run, use_reentrant=False)
        else:
            with torch.autograd.graph.save_on_cpu():
                loss = run()
        loss.backward()
        grads.append((loss.detach(), {k: v.grad for k, v in m.named_parameters()}))
    assert torch.equal(grads[0][0], grads[1][0])
    for k in grads[0][1]:
        assert torch.equal(grads[0][1][k], grads[1][1][k]), k
