"""Drawing a token from each row of logits (sample_tokens) after temperature, top-k, top-p, min-p.

CPU: refusals. GPU: against the definition in float64, row by row. Weights are float32 (2^-23
each, and the argument's rounding carried along) and their sums exact, so a running sum is off by
less than 2^-21 of the whole: a token that differs from the definition's is accepted where it is
the definition's at a uniform number or a top_p moved by that much (at borders only).
"""
import math

import numpy as np
import pytest
import torch

from mamba_amd import _lib
from mamba_amd.sampling import sample_tokens


@pytest.fixture(scope="module")
def lib():
    return _lib.register_hip_kernel()


BASE = dict(rows=4, vocab=1000, io_dtype=0, top_k=0, temperature=1.0, top_p=1.0, min_p=0.0, stride_row=1000,
            stride_word=1, logits=1 << 32, uniform=1 << 33, tokens=1 << 34)


@pytest.mark.parametrize("kw,status", [
    (dict(rows=0), 1), (dict(vocab=0), 1), (dict(io_dtype=2), 1), (dict(logits=None), 1), (dict(uniform=None), 1),
    (dict(tokens=None), 1), (dict(stride_row=-1), 1), (dict(stride_word=-1), 1), (dict(tokens=(1 << 32) + 8), 1),
    (dict(tokens=1 << 33), 1), (dict(vocab=(1 << 20) + 1), 2), (dict(stride_row=1 << 50), 2),
])
def test_validation(lib, kw, status):
    assert lib.mss_sample(_lib.SampleArgs(**{**BASE, **kw}), None) == status
    assert lib.mss_sample(None, None) == 1


def test_python_errors():
    x, u = torch.randn(3, 10), torch.rand(3)
    bad = [dict(logits=x.double()), dict(uniform=u.double()), dict(logits=x[0]), dict(uniform=torch.rand(2)),
           dict(logits=x[:, :0]), dict(temperature=-1.0), dict(temperature=math.nan), dict(top_k=-1), dict(top_p=1.5),
           dict(top_p=-0.1), dict(min_p=2.0), dict(top_k=torch.ones(3)), dict(top_p=torch.ones(4)),
           dict(min_p=torch.ones(3, dtype=torch.float64)), dict(temperature=torch.ones(3, 1))]
    for kw in bad:
        with pytest.raises((ValueError, TypeError)):
            sample_tokens(**{**dict(logits=x, uniform=u), **kw})
    with pytest.raises(RuntimeError):
        sample_tokens(x, u)  # no CPU path


# ------------------------------------------------------------------------------------ GPU
def draw(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row by the definition: x float64."""
    if np.isnan(x).any() or not (x > -np.inf).any():
        return -1
    order = np.lexsort((np.arange(len(x)), -x))
    if not temperature > 0:
        return int(order[0])
    order = order[x[order] > -np.inf]
    if top_k > 0:
        order = order[:top_k]
    m = x[order[0]]
    d = np.where(x[order] == m, 0.0, x[order] - m) if np.isinf(m) else x[order] - m
    w = np.exp(d / temperature)
    before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
    n = max(1, int((before < top_p * w.sum()).sum())) if top_p < 1 else len(w)
    n = max(1, int((w[:n] >= min_p).sum())) if min_p > 0 else n
    at = np.sort(order[:n])
    rank = {int(i): k for k, i in enumerate(order)}
    mass = np.cumsum([w[rank[int(i)]] for i in at])
    return int(at[min(n - 1, int((mass <= u * mass[-1]).sum()))])


def check(logits, u, got, **kw):
    x, u, got = logits.double().cpu().numpy(), u.double().cpu().numpy(), got.cpu().numpy()
    row = {k: (lambda r, v=v: float(np.float32(v))) if not torch.is_tensor(v) else (lambda r, v=v.cpu(): float(v[r]))
           for k, v in kw.items()}
    for r in range(len(x)):
        s = {k: f(r) for k, f in row.items()}
        if "top_k" in s:
            s["top_k"] = int(s["top_k"])
        if got[r] == draw(x[r], u[r], **s):
            continue
        near = set()
        for e in (-2.0 ** -21, 0.0, 2.0 ** -21):
            for g in (-2.0 ** -21, 0.0, 2.0 ** -21):
                t = dict(s, top_p=s["top_p"] + g) if s.get("top_p", 1.0) < 1 else s
                near.add(draw(x[r], u[r] + e, **t))
        assert int(got[r]) in near, (r, s, float(u[r]), int(got[r]), near)


def logits_of(rows, vocab, dtype=torch.float32, seed=0, size=2.5):
    g = torch.Generator().manual_seed(seed)
    x = size * torch.randn(rows, vocab, generator=g)
    x.scatter_add_(1, torch.randint(0, vocab, (rows, 4), generator=g), 6 * torch.rand(rows, 4, generator=g))
    return x.to(dtype).to("cuda"), torch.rand(rows, generator=g).to("cuda")


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.7, top_k=1), dict(top_k=5), dict(top_k=50, temperature=0.8),
            dict(top_p=0.9), dict(top_p=0.5, temperature=2.0), dict(top_p=0.0), dict(min_p=0.05), dict(min_p=1.0),
            dict(temperature=0.8, top_k=40, top_p=0.95, min_p=0.01), dict(temperature=1e-4, top_p=0.9),
            dict(temperature=1e4, top_k=300, top_p=0.7), dict(top_k=10**9, top_p=0.3), dict(temperature=math.inf, top_p=0.4)]


@pytest.mark.gpu
@pytest.mark.parametrize("kw", SETTINGS, ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 7), (5, 1000), (2, 8191), (4, 8200), (3, 50280)])
def test_draw(rows, vocab, dtype, kw):
    x, u = logits_of(rows, vocab, dtype, seed=vocab)
    check(x, u, sample_tokens(x, u, **kw), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_vocab(dtype):
    for vocab in (131072, 262143, 1 << 20):
        x, u = logits_of(2, vocab, dtype, seed=vocab)
        for kw in (dict(), dict(top_k=1000, top_p=0.9), dict(top_p=0.99, temperature=1.5)):
            check(x, u, sample_tokens(x, u, **kw), **kw)


@pytest.mark.gpu
def test_settings_by_row():
    rows, vocab = 40, 3001
    x, u = logits_of(rows, vocab)
    g = torch.Generator().manual_seed(1)
    pick = lambda v: torch.tensor(v)[torch.randint(0, len(v), (rows,), generator=g)].to("cuda")  # noqa: E731
    kw = dict(temperature=pick([0.0, 0.5, 1.0, 2.0]), top_k=pick([0, 1, 7, 500, 5000]).int(), top_p=pick([1.0, 0.9, 0.3, 0.0]),
              min_p=pick([0.0, 0.1, 1.0]))
    check(x, u, sample_tokens(x, u, **kw), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["words_apart", "rows_apart", "offset"])
def test_strides(layout, dtype):
    x, u = logits_of(6, 1003, dtype)
    if layout == "words_apart":  # the decode step's (vocab, batch) logits, transposed
        y = x.t().contiguous().t()
    else:
        big = torch.full((6, 1003 + 13), float("nan"), dtype=dtype, device="cuda")
        at = 0 if layout == "rows_apart" else 5
        big[:, at:at + 1003] = x
        y = big[:, at:at + 1003]
    for kw in (dict(), dict(top_k=20, top_p=0.8), dict(temperature=0.0)):
        assert torch.equal(sample_tokens(y, u, **kw), sample_tokens(x, u, **kw))
        check(y, u, sample_tokens(y, u, **kw), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [9, 2000, 40000])
def test_ties(vocab):
    """Words with the same logit: the lower index first, at every filter's border."""
    x = torch.zeros(8, vocab, device="cuda")
    x[1] = -0.0
    x[1, ::2] = 0.0
    x[2, vocab // 2:] = 1.0
    x[3, ::3] = 2.0
    x[4, -1] = 5.0
    x[5] = torch.arange(vocab, device="cuda").remainder(4).float()
    x[6] = torch.arange(vocab, device="cuda").remainder(5).neg().float()
    x[7, : vocab // 2] = -math.inf
    u = torch.tensor([0.0, 0.999, 0.5, 0.3, 0.9, 0.25, 0.7, 0.6], device="cuda")
    for kw in (dict(), dict(top_k=3), dict(top_k=vocab // 2 + 1), dict(top_p=0.37), dict(top_k=6, top_p=0.55),
               dict(min_p=0.3), dict(temperature=0.0), dict(top_k=1), dict(min_p=1.0, top_p=0.2)):
        check(x, u, sample_tokens(x, u, **kw), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [5, 1500, 50280])
def test_rows_at_the_edge(vocab):
    """Rows without a word, with one word, with infinities, with NaN, the type's lowest value,
    and uniform numbers at and past the ends."""
    inf, low = math.inf, torch.finfo(torch.float32).min
    x = torch.randn(10, vocab, device="cuda")
    x[0] = -inf
    x[1] = -inf
    x[1, vocab - 2] = -3.0
    x[2, 3] = math.nan
    x[3, 1] = x[3, 4] = inf
    x[4] = low
    x[5] = low
    x[5, 2] = -low
    x[6] = inf
    x[7] = -inf
    x[7, 2] = low
    u = torch.tensor([0.5, 0.5, 0.5, 0.6, 0.5, 0.99, 0.3, 0.0, -1.0, 1.0], device="cuda")
    for kw in (dict(), dict(top_k=2), dict(top_p=0.6), dict(top_k=3, top_p=0.9, min_p=0.2), dict(temperature=0.0)):
        got = sample_tokens(x, u, **kw)
        check(x[:8], u[:8], got[:8], **kw)
        assert got[0] == -1 and got[1] == vocab - 2 and got[2] == -1 and got[5] == 2 and got[7] == 2
        assert 0 <= int(got[8]) < vocab and 0 <= int(got[9]) < vocab
    first_and_last = sample_tokens(x[8:], u[8:], top_k=3).tolist()
    best = x[8:].topk(3).indices.tolist()
    assert first_and_last == [min(best[0]), max(best[1])]
    nan = torch.full((1,), math.nan, device="cuda")  # a number that is none: the first word kept
    assert int(sample_tokens(x[8:9], nan, top_k=3)) == min(best[0])
    kw = dict(temperature=nan, top_p=nan, min_p=nan)  # settings that are none: greedy, or no filter
    assert int(sample_tokens(x[8:9], u[:1], **kw)) == int(x[8].argmax())
    check(x[8:9], u[:1], sample_tokens(x[8:9], u[:1], top_p=nan, min_p=nan))


@pytest.mark.gpu
def test_frequencies():
    """Many draws of one row follow its probabilities: Pearson's statistic over 12 words stays
    below its 1 - 1e-9 quantile (11 degrees of freedom: 68.6)."""
    p = torch.tensor([0.3, 0.2, 0.1, 0.1, 0.08, 0.06, 0.05, 0.04, 0.03, 0.02, 0.01, 0.01])
    n = 20000
    u = torch.rand(n, generator=torch.Generator().manual_seed(7)).to("cuda")
    got = sample_tokens(p.log().to("cuda").expand(n, 12), u)
    seen = torch.bincount(got.cpu(), minlength=12).double()
    want = p.double() / p.double().sum() * n
    assert float(((seen - want) ** 2 / want).sum()) < 68.6


@pytest.mark.gpu
def test_empty_and_repeated():
    x, u = logits_of(4, 50280)
    assert sample_tokens(x[:0], u[:0]).shape == (0,)
    kw = dict(temperature=0.9, top_k=100, top_p=0.9)
    first = sample_tokens(x, u, **kw)
    for _ in range(5):
        assert torch.equal(first, sample_tokens(x, u, **kw))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sample_tokens(x, u, **kw)
    for seed in (3, 4, 5):
        y, v = logits_of(4, 50280, seed=seed)
        x.copy_(y)
        u.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, sample_tokens(x, u, **kw))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [60000, 70001])
@pytest.mark.parametrize("kw", [dict(top_p=0.95, temperature=3.0), dict(top_k=3000, top_p=0.9), dict(top_k=12000),
                                dict(top_k=40000, top_p=0.5, temperature=2.0), dict(min_p=1e-6, top_p=0.97, temperature=2.0),
                                dict(top_p=0.999), dict(top_k=2870, min_p=0.001), dict(min_p=1e-7),
                                dict(top_p=0.6, temperature=50.0), dict(top_k=300, temperature=20.0)], ids=str)
def test_long_prefixes(vocab, kw, dtype):
    """Prefixes longer than the list holds, and those near its length, in rows that stay in registers
    and rows that do not."""
    x, u = logits_of(3, vocab, dtype, seed=vocab)
    check(x, u, sample_tokens(x, u, **kw), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [50000, 100000])
def test_sorted_and_equal_words(vocab):
    """Words in order of their logits (all of the largest in one place), whole stretches alike."""
    x = torch.empty(6, vocab, device="cuda")
    x[0] = torch.linspace(5, -5, vocab)
    x[1] = torch.linspace(-5, 5, vocab)
    x[2] = 1.0
    x[3] = torch.arange(vocab, device="cuda").div(7, rounding_mode="floor").remainder(11).float()
    x[4] = -3.0
    x[4, 17:400] = 2.0
    x[5] = -math.inf
    x[5, ::2] = 0.25
    u = torch.tensor([0.1, 0.9, 0.5, 0.3, 0.7, 0.999], device="cuda")
    for kw in (dict(), dict(top_k=50), dict(top_k=1000, top_p=0.5), dict(top_p=0.8), dict(min_p=0.1), dict(top_k=200),
               dict(top_p=0.3, min_p=0.5, temperature=0.5)):
        check(x, u, sample_tokens(x, u, **kw), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [65537, 70001, 131072, 262147])
def test_long_rows_whose_beginning_differs(vocab, dtype):
    """Rows too long for registers whose first words say little of the rest: none there, all small or
    large there, the largest at the end, an infinity or a NaN late."""
    x, _ = logits_of(10, vocab, dtype, seed=vocab)
    x[1, :20000] = -math.inf
    x[2, :20000] -= 30
    x[3, :20000] += 12
    x[4, vocab - 1] = x[4].max() + 1
    x[5, vocab - 1] = 90.0
    x[6, :16384] = x[6, :16384].clamp(max=-1.0)
    x[7, 40000:] = -math.inf
    x[8, vocab - 2] = math.inf
    x[9, vocab - 3] = math.nan
    u = torch.linspace(0.02, 0.97, 10, device="cuda")
    for kw in (dict(top_p=0.9, min_p=0.001), dict(top_p=0.9), dict(top_k=50), dict(top_k=700, top_p=0.8), dict(min_p=0.02),
               dict(min_p=1e-6), dict(top_p=0.5, temperature=0.3), dict(top_k=1000, min_p=0.01, temperature=0.05)):
        check(x, u, sample_tokens(x, u, **kw), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("top_k", [127, 128, 129, 130, 200, 255, 256, 257])
def test_lists_around_the_short_ones(top_k):
    """Lists about as long as those that are looked at without bins, in both kinds of rows."""
    for vocab in (700, 50000, 90000):
        x, u = logits_of(5, vocab, torch.float32, seed=top_k)
        for kw in (dict(), dict(top_p=0.9), dict(top_p=0.7, min_p=0.01, temperature=1.4)):
            check(x, u, sample_tokens(x, u, top_k=top_k, **kw), top_k=top_k, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [16000, 50280, 70001])
def test_many_rows_of_long_prefixes(vocab):
    """Every row's prefix outgrows the list, in more rows than there are compute units: what the waves of
    a workgroup share has to be read by all of them before it is cleared."""
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn(300, vocab, generator=g)
    x[::2] *= 0.02  # a bin that outgrows the list too
    x = x.to("cuda")
    u = torch.rand(300, generator=g).to("cuda")
    for kw in (dict(top_p=0.97), dict(top_p=0.95, top_k=vocab - 10, temperature=3.0)):
        got = sample_tokens(x, u, **kw)
        for _ in range(4):
            assert torch.equal(got, sample_tokens(x, u, **kw))
        check(x[::7], u[::7], got[::7], **kw)


@pytest.mark.gpu
def test_lazily_negated():
    """Logits, uniform numbers and settings that torch holds lazily negated give what their values give."""
    x, u = logits_of(6, 1003)
    settings = dict(temperature=torch.linspace(0.5, 1.5, 6, device="cuda"), top_p=torch.linspace(0.5, 1, 6, device="cuda"),
                    min_p=torch.linspace(0, 0.2, 6, device="cuda"))
    want = sample_tokens(x, u, **settings)
    neg = {k: torch._neg_view(-v) for k, v in settings.items()}
    assert all(v.is_neg() for v in neg.values())
    for y in (torch._neg_view(-x), torch.complex(x, -x).conj().imag):
        assert y.is_neg() and torch.equal(y, x)
        assert torch.equal(sample_tokens(y, torch._neg_view(-u), **neg), want)


@pytest.mark.gpu
def test_more_rows_than_one_launch_takes():
    """2^22 rows and some, each with settings of its own: the first word where the temperature is 0, and
    elsewhere the word that holds the uniform number's share of the weight (2^-20 from a border)."""
    rows, vocab = (1 << 22) + 77, 3
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(rows, vocab, generator=g, device="cuda")
    u = torch.rand(rows, generator=g, device="cuda")
    t = torch.rand(rows, generator=g, device="cuda").clamp_min(0.3)
    t[::3] = 0
    k = torch.full((rows,), 2, dtype=torch.int32, device="cuda")
    got = sample_tokens(x, u, temperature=t, top_k=k)
    w = torch.exp((x - x.amax(1, keepdim=True)).double() / t.double().clamp_min(0.3)[:, None])
    w[torch.arange(rows, device="cuda"), x.argmin(1)] = 0
    ends = w.cumsum(1)
    at = u.double() * ends[:, 2]
    inside = (ends - w < at[:, None] + 2.0 ** -20) & (at[:, None] - 2.0 ** -20 < ends) & (w > 0)
    ok = torch.where(t > 0, inside.gather(1, got.clamp(0, 2)[:, None])[:, 0], got == x.argmax(1))
    assert got.min() >= 0 and got.max() <= 2 and torch.all(ok)


@pytest.mark.parametrize("name", ["temperatures", "top_ks", "top_ps", "min_ps"])
def test_tokens_over_settings(lib, name):
    """Tokens written over settings that other rows have yet to read are refused."""
    assert lib.mss_sample(_lib.SampleArgs(**{**BASE, name: (1 << 34) + 8}), None) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [1.0, 0.5])
@pytest.mark.parametrize("base", [0.1, -3.2, -17.3, 50.7, 700.3])
def test_top_p_of_long_rows_whose_beginning_is_far_below(base, temperature):
    """Rows read once whose first words lie about 32 T below the rest, on both sides of a power of two, where
    rounded differences differ most: the whole sum is as exact as the list's. Six thousand words of forty
    logits share the weight, and top_p ends 10^-6 of the sum before and behind a border between two; the
    last word kept is drawn."""
    vocab, rows, grid = 70001, 64, 2.0 ** -5
    rng = np.random.default_rng(int(abs(base) * 10))
    x = np.full((rows, vocab), -np.inf, np.float32)
    first = (base + rng.uniform(-0.1, 0.1, rows)).astype(np.float32)
    top = np.ceil((first.astype(np.float64) + 32 * temperature) / grid) * grid
    words = top[:, None] - grid * np.arange(1, 41)  # exact in float32
    x[:, 5], x[:, 20000], x[:, 30000:36000] = first, top, np.repeat(words, 150, 1)
    w = np.exp((x[:, 20000:36000].astype(np.float64) - top[:, None]) / temperature)
    mass = np.cumsum(w, 1)
    at = 10000 + rng.integers(1000, 5900, rows)
    border = mass[np.arange(rows), at]  # the weight up to a word: the one behind it begins there
    top_p = border / mass[:, -1] + np.where(np.arange(rows) % 2, 1e-6, -1e-6)
    u = torch.full((rows,), 1 - 2.0 ** -24, device="cuda")
    kw = dict(temperature=temperature, top_p=torch.from_numpy(top_p.astype(np.float32)).to("cuda"))
    x = torch.from_numpy(x).to("cuda")
    check(x, u, sample_tokens(x, u, **kw), **kw)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """More than 2^32 logits: the last rows against the same by themselves."""
    rows, vocab = 4200, 1 << 20
    g = torch.Generator(device="cuda").manual_seed(81)
    x = torch.randn(rows, vocab, generator=g, device="cuda", dtype=torch.bfloat16)
    u = torch.rand(rows, generator=g, device="cuda")
    for kw in (dict(top_k=50, top_p=0.9), dict(temperature=0.0), dict()):
        got = sample_tokens(x, u, **kw)
        assert torch.equal(got[-40:], sample_tokens(x[-40:].clone(), u[-40:], **kw))
        check(x[-2:], u[-2:], got[-2:], **kw)
