"""Serving a MambaLM with 8-bit projections (serve.Fp8LM): prompt, steps and draws together
(mamba/mamba1.py:300-363 with 8-bit products).

CPU: refusals. GPU: the pieces against the same calls made by hand (bit for bit), a step against
a longer prompt, and the whole against the model in float32. An 8-bit operand differs from its
value by at most 2^-4 of it, so a product of two, whose errors have random signs, by at most
sqrt(2) 2^-4 of its size; the stream takes one such error from each of a block's two products
and the logits one more: for two blocks 5 x 0.089 = 0.44 of the logits' size.
"""
import pytest
import torch

from mamba_amd.fp8 import add_rmsnorm_fp8, fp8_matmul, quantize_fp8, quantize_fp8_weight
from mamba_amd.mamba1 import MambaLM
from mamba_amd.sampling import sample_tokens
from mamba_amd.serve import Fp8LM

VOCAB, DIM, LAYERS = 1000, 192, 2


def lm(seed=0, **kw):
    torch.manual_seed(seed)
    return MambaLM(VOCAB, DIM, LAYERS, device="cuda", **kw)


def prompt(batch, length, seed=1):
    return torch.randint(0, VOCAB, (batch, length), generator=torch.Generator().manual_seed(seed)).cuda()


def test_refusals():
    with pytest.raises(TypeError):
        Fp8LM(torch.nn.Linear(2, 2))
    with pytest.raises(RuntimeError):  # no CPU path
        Fp8LM(MambaLM(10, 16, 1))


@pytest.mark.gpu
def test_gpu_refusals():
    m = Fp8LM(lm())
    with pytest.raises(ValueError):
        m.prefill(prompt(2, 0))
    with pytest.raises(ValueError):
        m.generate(prompt(2, 4), torch.rand(5, 3, device="cuda"))
    with pytest.raises(ValueError):
        m.generate(prompt(2, 4), torch.rand(5, 2, device="cuda"), top_p=2.0)
    assert m.generate(prompt(2, 4), torch.rand(0, 2, device="cuda")).shape == (0, 2)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,length", [(1, 1), (2, 2), (3, 37), (1, 300)])
def test_prefill_is_close_to_float32(batch, length):
    model = lm()
    tokens = prompt(batch, length)
    logits, caches = Fp8LM(model).prefill(tokens)
    with torch.no_grad():
        want = model(tokens, act_dtype=torch.float32).view(batch, length, -1)[:, -1]
    assert logits.dtype == torch.float32 and logits.shape == (batch, VOCAB) and logits.is_contiguous()
    assert len(caches) == LAYERS and caches[0]["ssm"].shape == (batch, 2 * DIM, 16)
    err = float((logits - want).norm() / want.norm())
    print("relative error", err, flush=True)
    assert err < 0.44


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [1, 3, 8])
def test_step_is_the_pieces_together(batch):
    """One block's step by hand, and the logits, bit for bit."""
    model = lm(2)
    m = Fp8LM(model)
    _, caches = m.prefill(prompt(batch, 9))
    mine = [{k: v.clone() for k, v in c.items()} for c in caches]
    token = prompt(batch, 1, seed=3)[:, 0]
    got = m.step(token, caches)
    from mamba_amd.decode import causal_conv1d_update

    with torch.no_grad():
        h, delta = model.embedding[token].t().contiguous(), None
        for blk, c in zip(model.blocks, mine):
            h, q, s = add_rmsnorm_fp8(h, delta, blk.norm.weight, blk.norm.eps)
            xz = fp8_matmul(*quantize_fp8_weight(torch.cat([blk.in_proj, blk.z_proj])), q, s)
            u = causal_conv1d_update(c["conv"], xz[:2 * DIM].t(), blk.conv_weight, blk.conv_bias).t()
            y = blk.s6.step(u, xz[2 * DIM:], c["ssm"], m._small, c["A"])
            delta = fp8_matmul(*quantize_fp8_weight(blk.out_proj), *quantize_fp8(y))
        _, q, s = add_rmsnorm_fp8(h, delta, model.final_norm.weight, model.final_norm.eps)
        want = fp8_matmul(*quantize_fp8_weight(model.embedding), q, s, out_dtype=torch.float32, token_major=True)
    assert torch.equal(got, want)
    for a, b in zip(caches, mine):
        assert torch.equal(a["conv"], b["conv"]) and torch.equal(a["ssm"], b["ssm"])


@pytest.mark.gpu
@pytest.mark.parametrize("batch,length", [(2, 1), (2, 2), (3, 40)])
def test_steps_follow_a_prompt(batch, length):
    """Prompt then three steps against the whole as a prompt: the same function, up to roundings
    to 8 bits that fall differently (as far apart as either may be from float32)."""
    m = Fp8LM(lm(4))
    tokens = prompt(batch, length + 3)
    _, caches = m.prefill(tokens[:, :length])
    for i in range(3):
        logits = m.step(tokens[:, length + i], caches)
    want, _ = m.prefill(tokens)
    err = float((logits - want).norm() / want.norm())
    print("relative error", err, flush=True)
    assert err < 0.44


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(temperature=0.7, top_k=40, top_p=0.95), dict(temperature=0.0),
                                dict(min_p=0.05, by_row=True)], ids=str)
def test_generate(kw):
    """Graph and eager runs give the same tokens, which are the draws made by hand."""
    kw = dict(kw)
    if kw.pop("by_row", False):
        kw["temperature"] = torch.tensor([0.0, 0.8, 1.2], device="cuda")
        kw["top_k"] = torch.tensor([0, 5, 900], dtype=torch.int32, device="cuda")
    m = Fp8LM(lm(5))
    tokens = prompt(3, 11)
    uniforms = torch.rand(7, 3, generator=torch.Generator().manual_seed(6)).cuda()
    eager = m.generate(tokens, uniforms, graph=False, **kw)
    for _ in range(2):
        assert torch.equal(m.generate(tokens, uniforms, **kw), eager)
    logits, caches = m.prefill(tokens)
    for i in range(7):
        token = sample_tokens(logits, uniforms[i], **kw)
        assert torch.equal(token, eager[i])
        logits = m.step(token, caches)


@pytest.mark.gpu
def test_refresh_and_complex_states():
    model = lm(7, complex_ssm=True)
    m = Fp8LM(model)
    tokens = prompt(2, 5)
    before, caches = m.prefill(tokens)
    assert torch.isfinite(m.step(tokens[:, 0], caches)).all()
    with torch.no_grad():
        model.blocks[0].out_proj.mul_(3.0)
    assert torch.equal(m.prefill(tokens)[0], before)
    m.refresh()
    assert not torch.equal(m.prefill(tokens)[0], before)


def changed_in_turn(model):
    """(name, tensor) of every weight of the model, a kind each."""
    blk = model.blocks[1]
    return [("embedding", model.embedding), ("final_norm", model.final_norm.weight), *blk.named_parameters()]


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(), dict(complex_ssm=True)], ids=str)
def test_refresh_is_what_changes_weights(kw):
    """Whatever weight of the model changes, in place or behind autograd's version counter, prompt and
    step give the same until refresh(), and after it what a new Fp8LM of the model gives."""
    model = lm(8, **kw)
    m = Fp8LM(model)
    tokens = prompt(2, 6)

    def out(m):
        logits, caches = m.prefill(tokens)
        return logits, m.step(tokens[:, 3], caches), caches[1]["ssm"]

    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))  # noqa: E731
    held = out(m)
    names = changed_in_turn(model)
    assert len(names) == 13 + len(kw)
    for i, (name, w) in enumerate(names):
        with torch.no_grad():
            (w.data if i % 2 else w).mul_(0.75).add_(0.01)
        assert same(out(m), held), name
        m.refresh()
        now = out(m)
        assert same(now, out(Fp8LM(model))) and not same(now, held), name
        held = now


@pytest.mark.gpu
def test_refresh_reaches_a_captured_step():
    """refresh() writes the weights where they lie: a graph of a step goes on with the new ones."""
    model = lm(9)
    m = Fp8LM(model)
    tokens = prompt(2, 6)
    _, caches = m.prefill(tokens)
    token = tokens[:, 0].clone()
    copies = lambda: [{k: v.clone() for k, v in c.items()} for c in caches]  # noqa: E731
    m.step(token, copies())
    mine = copies()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = m.step(token, mine)
    for scale in (0.5, 1.5, 1.1):
        with torch.no_grad():
            for p in model.parameters():
                p.mul_(scale)
        m.refresh()
        for c, old in zip(mine, caches):
            c["conv"].copy_(old["conv"]), c["ssm"].copy_(old["ssm"])
        # (each cache brings the matrix A of its prompt; a step takes that one)
        eager = copies()
        want = m.step(token, [dict(c, A=g["A"]) for c, g in zip(eager, mine)])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(logits, want)


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("batch", [3, 20])
def test_a_row_without_a_word_stays_without(batch, graph):
    """A row whose draw is -1 draws -1 from then on, greedy or not; the others draw what they draw beside a
    row that is well. So does a loop of steps."""
    m = Fp8LM(lm(10))
    tokens = prompt(batch, 5)
    uniforms = torch.rand(6, batch, generator=torch.Generator().manual_seed(11)).cuda()
    kw = dict(temperature=torch.linspace(0, 1.2, batch, device="cuda"), top_k=30)
    want = m.generate(tokens, uniforms, graph=graph, **kw)
    well = m.prefill

    def prefill(tokens):
        logits, caches = well(tokens)
        logits[1] = float("nan")
        return logits, caches

    m.prefill = prefill
    got = m.generate(tokens, uniforms, graph=graph, **kw)
    assert torch.all(got[:, 1] == -1)
    keep = torch.arange(batch, device="cuda") != 1
    assert torch.equal(got[:, keep], want[:, keep])
    logits, caches = m.prefill(tokens)
    for i in range(3):
        token = sample_tokens(logits, uniforms[i], **kw)
        assert torch.equal(token, got[i])
        logits = m.step(token, caches)
        assert torch.isnan(logits[1]).all() and torch.isfinite(logits[keep]).all()


def e4m3(v):
    """float64 values of magnitude at most 448, rounded to e4m3 (nearest, ties to even)."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def eight_bit(y, rows):
    """What a float64 matrix (.., features) stands for in 8 bits, one scale for `rows` rows and 128 features."""
    out = torch.empty_like(y)
    for i in range(0, y.shape[0], rows):
        for j in range(0, y.shape[1], 128):
            part = y[i:i + rows, j:j + 128]
            scale = (part.abs().max() / 448).clamp_min(2.0 ** -126)
            out[i:i + rows, j:j + 128] = e4m3(part / scale) * scale
    return out


def logits_in_64_bits(model, tokens):
    """Every position's logits of one sequence: the model in float64 with 8-bit products, the S6
    projections' weights in bf16, nothing else rounded."""
    weight = {k: v.detach().double().cpu() for k, v in model.named_parameters()}
    silu, softplus = torch.nn.functional.silu, torch.nn.functional.softplus
    norm = lambda h, w: h / torch.sqrt(h.square().mean(1, keepdim=True) + 1e-5) * w  # noqa: E731
    product = lambda x, w: eight_bit(x, 1) @ eight_bit(w, 128).t()  # noqa: E731
    h = weight["embedding"][tokens.cpu()]
    for i in range(LAYERS):
        p = {k[len(f"blocks.{i}."):]: v for k, v in weight.items() if k.startswith(f"blocks.{i}.")}
        x = norm(h, p["norm.weight"])
        xin, z = product(x, torch.cat([p["in_proj"], p["z_proj"]])).split(2 * DIM, 1)
        k = p["conv_weight"].shape[1]
        wide = torch.cat([xin.new_zeros(k - 1, 2 * DIM), xin])
        u = silu(p["conv_bias"] + sum(p["conv_weight"][:, j] * wide[j:j + len(xin)] for j in range(k)))
        r, n = p["s6.dt_proj"].shape[1], p["s6.A_log"].shape[1]
        dbl = u @ p["s6.x_proj"].bfloat16().double().t()
        dt = softplus(dbl[:, :r] @ p["s6.dt_proj"].bfloat16().double().t() + p["s6.dt_bias"])
        A, state, y = -torch.exp(p["s6.A_log"]), u.new_zeros(2 * DIM, n), []
        for t in range(len(u)):
            state = torch.exp(dt[t][:, None] * A) * state + (dt[t] * u[t])[:, None] * dbl[t, r:r + n]
            y.append(state @ dbl[t, r + n:] + p["s6.D"] * u[t])
        h = h + product(torch.stack(y) * silu(z), p["out_proj"])
    return product(norm(h, weight["final_norm.weight"]), weight["embedding"])


@pytest.mark.gpu
@pytest.mark.parametrize("length", [1, 2, 5, 70, 300])
def test_path_against_64_bits(length):
    """Prompt and three steps against the same model in float64 with the same roundings to 8 bits. The
    path's roundings to bf16 move an 8-bit operand by 2^-8 of itself; that takes it over a border, which
    lie at least 2^-4 of it apart, with a probability of at most 2^-4, and then by a step, at most 2^-3:
    2^-5 in root mean square for each of the five products, together sqrt(5) 2^-5 = 0.07 of the logits'
    size; twice that is allowed."""
    model = lm(12)
    with torch.no_grad():
        for name, p in model.named_parameters():  # norms and D that are not all one
            if name.endswith(("norm.weight", "s6.D")):
                p.mul_(1 + 0.3 * torch.randn_like(p))
    m = Fp8LM(model)
    tokens = prompt(2, length + 3, seed=length)
    want = torch.stack([logits_in_64_bits(model, row) for row in tokens])
    logits, caches = m.prefill(tokens[:, :length])
    for i in range(4):
        err = float((logits.double().cpu() - want[:, length - 1 + i]).norm() / want[:, length - 1 + i].norm())
        print("position", length - 1 + i, "relative error", err, flush=True)
        assert err < 0.14
        if i < 3:
            logits = m.step(tokens[:, length + i], caches)


@pytest.mark.gpu
def test_refresh_after_the_parameters_were_replaced():
    """A state dict assigned to the model puts other Parameter objects in place of those Fp8LM has seen:
    nothing changes until refresh(), and then everything does, a captured step's weights too."""
    model, other = lm(13), lm(14)
    m = Fp8LM(model)
    tokens = prompt(3, 7)
    held, caches = m.prefill(tokens)
    token = tokens[:, 0].clone()
    start = [c["ssm"].clone() for c in caches], [c["conv"].clone() for c in caches]
    graph = torch.cuda.CUDAGraph()
    m.step(token, caches)
    with torch.cuda.graph(graph):
        logits = m.step(token, caches)
    model.load_state_dict(other.state_dict(), assign=True)
    assert torch.equal(m.prefill(tokens)[0], held)
    m.refresh()
    fresh = Fp8LM(other)
    want, new = fresh.prefill(tokens)
    assert torch.equal(m.prefill(tokens)[0], want)
    for _ in range(2):
        for c, n, ssm, conv in zip(caches, new, *start):
            c["ssm"].copy_(ssm), c["conv"].copy_(conv), n["ssm"].copy_(ssm), n["conv"].copy_(conv)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(logits, fresh.step(token, new))
