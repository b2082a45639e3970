"""The language model's losses that keep no logits (MambaLM.loss, MambaLM.distill_loss): the whole model in
float32 against the float64 oracle with the losses' definitions, in bfloat16 with float32 masters and their
copies, and as a captured training step.

float32 within the model tests' bounds (1e-4 of a tensor's largest gradient, 1e-5 of the loss); bfloat16
within theirs (2e-2, 2e-3).
"""
import pytest
import torch
import torch.nn.functional as F

from mamba_amd.mamba1 import GraphedTrainStep, MambaLM
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
