"""8-bit serving operators: block-scaled e4m3 activations and weights, the residual add + RMSNorm
that writes them (mamba/mamba1.py:300-337), and the product of the two.

CPU: refusals. GPU: against the definitions in float64 on the same inputs.

Tolerances, all per element. An e4m3 rounding moves a value y by at most half a step,
2^(max(floor(log2 |y|), -6) - 4). float32 roundings count 2^-24 each: two between a value and its
quotient by the scale; the norm's sum of F squares at most F of them (halved by the root) and six
more up to the output. For a float32 product the sum of 128 products and the sum over blocks
count one whole step, 2^-23, for each addition, relative to the sum of the magnitudes. For a bf16
product the 8-bit matrix instructions may add the products 8 at a time, of which each loses less
than 2^-13 of the largest: 7 of them, so 2^-10 of the sum of the magnitudes covers the rest too.
"""
import numpy as np
import pytest
import torch

from mamba_amd import _lib
from mamba_amd.fp8 import add_rmsnorm_fp8, fp8_matmul, quantize_fp8, quantize_fp8_weight

BLOCK = 128
FP8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def lib():
    return _lib.register_hip_kernel()


# ------------------------------------------------------------------------------- refusals
QUANT = dict(features=300, tokens=10, io_dtype=0, stride_f=10, stride_t=1, ldq=304, x=1 << 32, q=1 << 36,
             scales=1 << 37)


@pytest.mark.parametrize("kw,status", [
    (dict(features=0), 1), (dict(tokens=-1), 1), (dict(io_dtype=2), 1), (dict(x=None), 1), (dict(q=None), 1),
    (dict(scales=None), 1), (dict(stride_f=-1), 1), (dict(stride_t=-10), 1), (dict(ldq=288), 1), (dict(ldq=305), 1),
    (dict(q=(1 << 36) + 8), 1), (dict(q=1 << 32), 1), (dict(scales=(1 << 32) + 64), 1), (dict(scales=(1 << 36) + 16), 1),
    (dict(stride_f=1 << 50), 2), (dict(features=65536 * 128, ldq=65536 * 128), 2),
])
def test_quant_validation(lib, kw, status):
    assert lib.mss_quant_fp8(_lib.QuantFp8Args(**{**QUANT, **kw}), None) == status
    assert lib.mss_quant_fp8(None, None) == 1


NORM = dict(features=300, tokens=10, delta_dtype=1, eps=1e-5, ldq=304, h=1 << 32, delta=1 << 33, weight=1 << 34,
            hn=1 << 35, q=1 << 36, scales=1 << 37)


@pytest.mark.parametrize("kw,status", [
    (dict(features=0), 1), (dict(tokens=0), 1), (dict(eps=-1.0), 1), (dict(eps=float("nan")), 1), (dict(h=None), 1),
    (dict(weight=None), 1), (dict(hn=None), 1), (dict(q=None), 1), (dict(scales=None), 1), (dict(delta_dtype=3), 1),
    (dict(ldq=302), 1), (dict(q=1 << 32), 1), (dict(hn=(1 << 32) + 16), 1), (dict(hn=1 << 33), 1),
    (dict(scales=(1 << 35) + 64), 1), (dict(q=1 << 34), 1), (dict(features=65536 * 128, ldq=65536 * 128), 2),
])
def test_norm_validation(lib, kw, status):
    assert lib.mss_norm_fp8(_lib.NormFp8Args(**{**NORM, **kw}), None) == status
    assert lib.mss_norm_fp8(None, None) == 1


WEIGHT = dict(M=200, K=300, io_dtype=0, ldw=300, ldq=304, w=1 << 32, q=1 << 36, scales=1 << 37)


@pytest.mark.parametrize("kw,status", [
    (dict(M=0), 1), (dict(K=0), 1), (dict(io_dtype=-1), 1), (dict(ldw=299), 1), (dict(ldq=300), 1), (dict(w=None), 1),
    (dict(q=(1 << 36) + 4), 1), (dict(q=1 << 32), 1), (dict(scales=None), 1), (dict(ldw=1 << 50), 2),
    (dict(M=65536 * 128), 2),
])
def test_weight_validation(lib, kw, status):
    assert lib.mss_quant_fp8_weight(_lib.QuantFp8WeightArgs(**{**WEIGHT, **kw}), None) == status
    assert lib.mss_quant_fp8_weight(None, None) == 1


MM = dict(M=200, K=300, T=10, out_dtype=1, token_major=0, ldw=304, ldx=304, ldc=10, W=1 << 32, w_scales=1 << 33,
          X=1 << 34, x_scales=1 << 35, C=1 << 36)


@pytest.mark.parametrize("kw,status", [
    (dict(M=0), 1), (dict(K=0), 1), (dict(T=0), 1), (dict(out_dtype=7), 1), (dict(ldw=296), 1), (dict(ldx=312), 1),
    (dict(ldc=9), 1), (dict(token_major=1, ldc=199), 1), (dict(W=None), 1), (dict(X=None), 1), (dict(w_scales=None), 1),
    (dict(x_scales=None), 1), (dict(C=None), 1), (dict(W=(1 << 32) + 8), 1), (dict(X=(1 << 34) + 1), 1),
    (dict(C=(1 << 32) + 1024), 1), (dict(C=1 << 34), 1), (dict(C=1 << 35), 1), (dict(C=1 << 33), 1),
    (dict(T=(1 << 19) + 1, ldc=1 << 20), 2), (dict(ldw=1 << 50), 2), (dict(ldc=1 << 50), 2),
])
def test_mm_validation(lib, kw, status):
    assert lib.mss_fp8_mm(_lib.Fp8MmArgs(**{**MM, **kw}), None) == status
    assert lib.mss_fp8_mm(None, None) == 1


def test_python_errors():
    x = torch.randn(8, 4)
    q8 = lambda *s: torch.zeros(*s).to(FP8)  # noqa: E731
    with pytest.raises(TypeError):
        quantize_fp8(x.double())
    with pytest.raises(ValueError):
        quantize_fp8(x[0])
    with pytest.raises(RuntimeError):
        quantize_fp8(x)  # no CPU path
    with pytest.raises(RuntimeError):
        quantize_fp8(x.requires_grad_(True))
    x = torch.randn(8, 4)
    with pytest.raises(TypeError):
        add_rmsnorm_fp8(x.bfloat16(), None, torch.ones(8))
    with pytest.raises(ValueError):
        add_rmsnorm_fp8(x, None, torch.ones(4))
    with pytest.raises(ValueError):
        add_rmsnorm_fp8(x, torch.randn(8, 5), torch.ones(8))
    with pytest.raises(TypeError):
        add_rmsnorm_fp8(x, x.half(), torch.ones(8))
    with pytest.raises(RuntimeError):
        add_rmsnorm_fp8(x, None, torch.ones(8))
    with pytest.raises(ValueError):
        quantize_fp8_weight(torch.randn(8, 4).t())
    with pytest.raises(RuntimeError):
        quantize_fp8_weight(x)
    one, s = torch.ones(1, 1), torch.ones(1, 4)
    with pytest.raises(TypeError):
        fp8_matmul(x, one, q8(4, 16), s)
    with pytest.raises(ValueError):
        fp8_matmul(q8(8, 16), one, q8(4, 32), s)
    with pytest.raises(ValueError):
        fp8_matmul(q8(8, 17), one, q8(4, 17), s)  # rows that do not start on 16 bytes
    with pytest.raises(ValueError):
        fp8_matmul(q8(8, 16), torch.ones(1, 2), q8(4, 16), s)
    with pytest.raises(ValueError):
        fp8_matmul(q8(8, 16), one, q8(4, 16), torch.ones(4, 1))
    with pytest.raises(ValueError):
        fp8_matmul(q8(8, 16), one, q8(4, 16), s, out=torch.zeros(4, 8, dtype=torch.bfloat16))
    with pytest.raises(TypeError):
        fp8_matmul(q8(8, 16), one, q8(4, 16), s, out_dtype=torch.float16)
    with pytest.raises(RuntimeError):
        fp8_matmul(q8(8, 16), one, q8(4, 16), s)


# ------------------------------------------------------------------------------------ GPU
def half_step(y):
    """Half an e4m3 step at float64 y."""
    return 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(np.abs(y), 1e-300))), -6) - 4)


def spread_blocks(scales, n):
    """Scales (blocks, tokens) as one for each of n features: (n, tokens)."""
    return np.repeat(scales, BLOCK, axis=0)[:n]


def check_quantised(y, q, scales, rel):
    """q (tokens, features), scales (blocks, tokens) against y (features, tokens) in float64,
    itself known up to `rel`."""
    f, t = y.shape
    pad = np.zeros((-(-f // BLOCK) * BLOCK, t))
    pad[:f] = np.abs(y)
    want = np.maximum(pad.reshape(-1, BLOCK, t).max(1) / 448.0, 2.0 ** -126)
    s = scales.double().cpu().numpy()
    assert s.shape == want.shape
    assert np.all(np.abs(s - want) <= want * (rel + 2.0 ** -24) * 1.001)
    got = q.float().double().cpu().numpy().T
    assert got.shape == y.shape
    per = spread_blocks(s, f)
    assert np.all(np.abs(got - y / per) <= half_step(y / per) + np.abs(y / per) * (2 * rel + 2.0 ** -22) + 1e-30)


def rand(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * torch.exp(2 * torch.randn(shape[0], 1, generator=g))
    return x.to(dtype).to("cuda")


LAYOUTS = ["channel", "token", "rows_apart", "strided"]


def laid_out(x, layout):
    if layout == "token":
        return x.t().contiguous().t()
    if layout == "rows_apart":
        big = torch.full((x.shape[0], x.shape[1] + 5), float("nan"), dtype=x.dtype, device=x.device)
        big[:, 3:3 + x.shape[1]] = x
        return big[:, 3:3 + x.shape[1]]
    if layout == "strided":
        big = torch.full((2 * x.shape[0], 3 * x.shape[1]), float("nan"), dtype=x.dtype, device=x.device)
        big[::2, ::3] = x
        return big[::2, ::3]
    return x.contiguous()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("f,t", [(1, 1), (5, 3), (128, 64), (129, 65), (1000, 7), (2560, 8), (300, 257), (768, 1031),
                                 (2560, 1)])
def test_quantise(f, t, layout, dtype):
    x = laid_out(rand(f, t, dtype=dtype), layout)
    q, scales = quantize_fp8(x)
    assert q.shape == (t, f) and q.dtype == FP8
    check_quantised(x.double().cpu().numpy(), q, scales, 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [4, 200])
def test_quantise_edges(t):
    """Zeros, subnormals, the largest floats, and values that are not finite, each in a block of
    its own; what they do stays there."""
    x = rand(6 * BLOCK, t)
    x[:BLOCK] = 0
    x[BLOCK:2 * BLOCK] = 1e-42
    x[2 * BLOCK:3 * BLOCK] = 3.4e38
    x[3 * BLOCK + 5, 1] = float("nan")
    x[4 * BLOCK + 9, 2] = float("-inf")
    q, scales = quantize_fp8(x)
    s, v = scales.cpu(), q.float().cpu() * scales.cpu().repeat_interleave(BLOCK, 0).t()
    assert torch.all(s[0] == 2.0 ** -126) and torch.all(v[:, :BLOCK] == 0)
    assert torch.all(s[1] == 2.0 ** -126) and torch.all(v[:, BLOCK:2 * BLOCK].abs() <= 2.0 ** -126 * 2.0 ** -9)
    assert torch.allclose(v[:, 2 * BLOCK:3 * BLOCK], torch.tensor(3.4e38), rtol=2.0 ** -22, atol=0)
    assert torch.isnan(s[3, 1]) and torch.isnan(v[1, 3 * BLOCK:4 * BLOCK]).all()
    assert torch.isinf(s[4, 2]) and torch.isnan(v[2, 4 * BLOCK:5 * BLOCK]).all()
    ok = torch.ones_like(v, dtype=torch.bool)
    ok[1, 3 * BLOCK:4 * BLOCK] = ok[2, 4 * BLOCK:5 * BLOCK] = False
    assert torch.isfinite(v[ok]).all()
    sub = x[5 * BLOCK:].double().cpu().numpy()
    check_quantised(sub, q[:, 5 * BLOCK:], scales[5:], 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,k,ld", [(1, 1, 1), (128, 128, 128), (130, 127, 140), (257, 1001, 1001), (1280, 2560, 2560)])
def test_quantise_weight(m, k, ld, dtype):
    w = rand(m, ld, dtype=dtype)[:, :k]
    q, scales = quantize_fp8_weight(w)
    assert q.shape == (m, k) and scales.shape == (-(-m // BLOCK), -(-k // BLOCK))
    y = w.double().cpu().numpy()
    s = scales.double().cpu().numpy()
    pad = np.zeros((s.shape[0] * BLOCK, s.shape[1] * BLOCK))
    pad[:m, :k] = np.abs(y)
    want = pad.reshape(s.shape[0], BLOCK, s.shape[1], BLOCK).max((1, 3)) / 448.0
    assert np.all(np.abs(s - want) <= want * 2.0 ** -24 * 1.001)
    per = np.repeat(np.repeat(s, BLOCK, 0), BLOCK, 1)[:m, :k]
    got = q.float().double().cpu().numpy()
    assert np.all(np.abs(got - y / per) <= half_step(y / per) + np.abs(y / per) * 2.0 ** -22)


@pytest.mark.gpu
@pytest.mark.parametrize("delta", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("f,t", [(1, 1), (5, 3), (128, 8), (768, 1), (1000, 70), (1280, 300), (129, 1031), (2048, 513),
                                 (2049, 40), (5120, 9), (4100, 515), (640, 4111)])
def test_norm(f, t, delta):
    h = rand(f, t, seed=1)
    d = None if delta is None else rand(f, t, seed=2, dtype=delta)
    w = 1 + 0.3 * torch.randn(f, generator=torch.Generator().manual_seed(3)).to("cuda")
    before = h.clone()
    hn, q, scales = add_rmsnorm_fp8(h, d, w, 1e-5)
    assert torch.equal(h, before)
    if d is None:
        assert hn is h
    else:
        assert torch.equal(hn, h + d.float())
    x = h.double().cpu().numpy()
    if d is not None:
        x = x + d.double().cpu().numpy()
    y = x / np.sqrt((x * x).mean(0) + 1e-5) * w.double().cpu().numpy()[:, None]
    rel = (f / 2 + 6) * 2.0 ** -24
    if d is not None:  # the sum's own rounding, relative to the sum: 2^-24 more
        rel += 2.0 ** -24
    check_quantised(y, q, scales, rel)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [3, 700])
def test_norm_not_finite(t):
    h = rand(300, t, seed=4)
    h[7, 1] = float("nan")
    h[:, 2] = 0
    _, q, scales = add_rmsnorm_fp8(h, None, torch.ones(300, device="cuda"))
    v = q.float() * scales.repeat_interleave(BLOCK, 0)[:300].t()
    assert torch.isnan(v[1]).all() and torch.all(v[2] == 0)
    keep = torch.arange(t, device="cuda") != 1
    assert torch.isfinite(v[keep]).all()


def operands(m, k, t, seed=0):
    w = rand(m, k, seed=seed)
    x = rand(k, t, seed=seed + 1)
    return *quantize_fp8_weight(w), *quantize_fp8(x)


def check_mm(got, wq, ws, xq, xs, token_major, out_dtype, only=slice(None)):
    m, k = wq.shape
    w = wq.float().double().cpu() * ws.double().cpu().repeat_interleave(BLOCK, 0)[:m].repeat_interleave(BLOCK, 1)[:, :k]
    x = (xq.float().double().cpu().t() * xs.double().cpu().repeat_interleave(BLOCK, 0)[:k])[:, only]
    want, size = w @ x, w.abs() @ x.abs()
    got = (got.double().cpu().t() if token_major else got.double().cpu())[:, only]
    bound = size * (min(k, BLOCK) + 3 * xs.shape[0] + 4) * 2.0 ** -23
    if out_dtype == torch.bfloat16:
        bound = size * 2.0 ** -10
    bound += want.abs() * (torch.finfo(out_dtype).eps / 2) * 1.01
    assert got.shape == want.shape
    assert torch.all((got - want).abs() <= bound), float(((got - want).abs() - bound).max())


SHAPES = [(1, 1, 1), (16, 128, 16), (17, 129, 3), (130, 256, 1), (100, 1000, 77), (1280, 2560, 8), (257, 1250, 300),
          (300, 384, 513), (5120, 1280, 1), (1000, 640, 33), (128, 4096, 64), (64, 15, 129), (1280, 2560, 333),
          (515, 143, 1025), (768, 768, 2048)]


@pytest.mark.gpu
@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,k,t", SHAPES)
def test_matmul(m, k, t, out_dtype, token_major):
    a = operands(m, k, t)
    got = fp8_matmul(*a, out_dtype=out_dtype, token_major=token_major)
    assert got.dtype == out_dtype and got.is_contiguous()
    check_mm(got, *a, token_major, out_dtype)
    assert torch.equal(got, fp8_matmul(*a, out_dtype=out_dtype, token_major=token_major))  # the same every time


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,t", [(100, 1000, 5), (300, 200, 140), (520, 384, 600)])
def test_matmul_layouts(m, k, t):
    """Rows apart, an output with rows apart, and what lies between the rows not relied on (NaN
    bytes) nor written."""
    wq, ws, xq, xs = operands(m, k, t)
    wide = lambda q: torch.full((q.shape[0], -(-k // 16) * 16 + 48), 0x7F, dtype=torch.uint8, device="cuda").view(FP8)  # noqa: E731
    w2, x2 = wide(wq), wide(xq)
    w2[:, :k], x2[:, :k] = wq, xq
    for token_major in (False, True):
        rows, cols = (t, m) if token_major else (m, t)
        for dtype in (torch.bfloat16, torch.float32):
            big = torch.full((rows, cols + 3), 7.0, dtype=dtype, device="cuda")
            out = big[:, 1:1 + cols]
            got = fp8_matmul(w2[:, :k], ws, x2[:, :k], xs, out_dtype=dtype, token_major=token_major, out=out)
            assert got is out
            check_mm(got, wq, ws, xq, xs, token_major, dtype)
            assert torch.all(big[:, 0] == 7) and torch.all(big[:, 1 + cols:] == 7)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [4, 40, 300])
def test_matmul_not_finite(t):
    """A token with a NaN, and one with an infinity, give NaN; the other tokens are untouched."""
    m, k = 200, 600
    w, x = rand(m, k), rand(k, t, seed=1)
    clean = operands(m, k, t)
    x[130, 1], x[599, 2] = float("nan"), float("inf")
    q, s = quantize_fp8(x)
    got = fp8_matmul(clean[0], clean[1], q, s)
    keep = [i for i in range(t) if i not in (1, 2)]
    assert torch.isnan(got[:, 1:3]).all()
    assert torch.equal(got[:, keep], fp8_matmul(*clean)[:, keep])


@pytest.mark.gpu
def test_empty():
    z = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    q, s = quantize_fp8(z(300, 0))
    assert q.shape == (0, 300) and s.shape == (3, 0)
    hn, q, s = add_rmsnorm_fp8(z(300, 0), None, z(300))
    assert hn.shape == (300, 0) and q.shape == (0, 300) and s.shape == (3, 0)
    wq, ws = quantize_fp8_weight(torch.randn(8, 300, device="cuda"))
    assert fp8_matmul(wq, ws, q, s).shape == (8, 0)
    wq, ws = quantize_fp8_weight(z(0, 300))
    q, s = quantize_fp8(z(300, 4))
    assert fp8_matmul(wq, ws, q, s, token_major=True).shape == (4, 0)
    wq, ws = quantize_fp8_weight(z(8, 0))
    q, s = quantize_fp8(z(0, 4))
    assert torch.equal(fp8_matmul(wq, ws, q, s), z(8, 4).bfloat16())


@pytest.mark.gpu
def test_side_stream_and_graph():
    """On a stream of its own, and replayed from a graph with new inputs."""
    h, d = rand(640, 9, seed=5), rand(640, 9, seed=6, dtype=torch.bfloat16)
    w, nw = rand(256, 640, seed=7), torch.ones(640, device="cuda")
    wq, ws = quantize_fp8_weight(w)

    def step():
        hn, q, s = add_rmsnorm_fp8(h, d, nw)
        return hn, fp8_matmul(wq, ws, q, s)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (8, 9, 10):
        h.copy_(rand(640, 9, seed=seed))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


# The kernels' other sizes: each side of the numbers at which another kernel takes over.
@pytest.mark.gpu
@pytest.mark.parametrize("delta", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("f,t", [(300, 255), (300, 256), (1000, 2048), (130, 2049), (260, 6144), (129, 6145), (1025, 31),
                                 (2049, 255), (8192, 3), (8193, 5), (8192, 300), (8200, 270)])
def test_norm_sizes(f, t, delta):
    test_norm(f, t, delta)


@pytest.mark.gpu
@pytest.mark.parametrize("f,t", [(300, 31), (300, 32), (129, 63), (1000, 65), (257, 16001)])
def test_quantise_sizes(f, t):
    for dtype in (torch.float32, torch.bfloat16):
        for layout in ("channel", "rows_apart"):
            test_quantise(f, t, layout, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,k,t", [(2100, 200, 2200), (2048, 384, 2048), (3000, 128, 1500), (64, 64, 4000), (5000, 100, 5),
                                   (1000, 2600, 200)])
def test_matmul_sizes(m, k, t, out_dtype, token_major):
    test_matmul(m, k, t, out_dtype, token_major)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [5, 300, 2500, 6200])
def test_norm_blocks_done_from_the_formula(t):
    """Blocks whose maximum before the norm is far from 1, or whose scale is at its lower bound: tiny
    and huge features, weights of zero and far from 1, no epsilon, one infinite feature."""
    f = 700
    h = rand(f, t, seed=11)
    w = torch.ones(f, device="cuda")
    h[:BLOCK] *= 1e-36
    w[BLOCK:2 * BLOCK] = 0
    w[2 * BLOCK:3 * BLOCK] = 1e-33
    w[3 * BLOCK:4 * BLOCK] = 1e-38
    h[:, 1] = 0
    h[:, 2] *= 1e-30  # its squares vanish
    h[:, 3] *= 1e25  # and here overflow: 1 / infinity
    h[130, 4] = float("inf")
    for delta in (None, torch.zeros(f, t, dtype=torch.bfloat16, device="cuda")):
        for eps in (1e-5, 0.0):
            _, q, s = add_rmsnorm_fp8(h, delta, w, eps)
            got = q.double() * s.double().repeat_interleave(BLOCK, 0)[:f].t()
            r = 1 / torch.sqrt(h.square().mean(0) + eps)
            want = (h * r).mul(w[:, None]).double().t()
            per = s.double().repeat_interleave(BLOCK, 0)[:f].t()
            ok = torch.isfinite(want).view(t, f)
            for b in range(s.shape[0]):  # a block with a value that is none stands for none
                part = slice(b * BLOCK, min(f, (b + 1) * BLOCK))
                ok[:, part] &= ok[:, part].all(1, keepdim=True)
            assert torch.equal(torch.isnan(got), ~ok)
            # half a step of the value over its scale, and float32 roundings of value and sum: F / 2 + 8
            ratio = (want / per).abs().clamp_min(2.0 ** -40)
            step = torch.exp2(torch.floor(torch.log2(ratio)).clamp_min(-6) - 4) * per
            bound = step + want.abs() * (f / 2 + 8) * 2.0 ** -23 + 2.0 ** -126 * 2.0 ** -10
            assert ((got - want).abs() <= bound)[ok].all()


@pytest.mark.gpu
@pytest.mark.parametrize("f,t", [(1, 1), (300, 9), (700, 301), (640, 2777), (300, 7001), (9000, 40)])
def test_norm_in_place(lib, f, t):
    """The C entry point with hn = h gives what it gives elsewhere, bit for bit."""
    h, d, w = rand(f, t, seed=12), rand(f, t, seed=13, dtype=torch.bfloat16), torch.rand(f, device="cuda") + 0.5
    hn, q, s = add_rmsnorm_fp8(h, d, w)
    q2, s2 = torch.empty_like(q), torch.empty_like(s)
    ld = -(-f // 16) * 16
    q2 = torch.zeros(t, ld, dtype=torch.uint8, device="cuda").view(FP8)[:, :f]
    a = _lib.NormFp8Args(features=f, tokens=t, delta_dtype=1, eps=1e-5, ldq=ld, h=h.data_ptr(), delta=d.data_ptr(),
                         weight=w.data_ptr(), hn=h.data_ptr(), q=q2.data_ptr(), scales=s2.data_ptr())
    assert lib.mss_norm_fp8(a, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(h, hn) and torch.equal(q2.float(), q.float()) and torch.equal(s2, s)


@pytest.mark.gpu
def test_quantise_borders():
    """Quotients that meet e4m3's borders exactly round to the even neighbour, whatever the scale's
    own rounding: 21 of 448 lies between 20 and 22, 84 between 80 and 88."""
    largest = torch.tensor([2.59375, 2.03125, 2.8125, 7.0, 1.5], device="cuda")
    x = torch.zeros(BLOCK, 5, device="cuda")
    x[0] = largest
    x[1], x[2], x[3] = largest * 3 / 64, -largest * 3 / 16, largest * 9 / 448
    for wide in (1, 20):  # both kernels
        q, _ = quantize_fp8(x.repeat(1, wide).to(torch.bfloat16) if wide == 1 else x.repeat(1, wide))
        v = q.float()[:5]
        assert torch.all(v[:, 0] == 448) and torch.all(v[:, 1] == 20) and torch.all(v[:, 2] == -80) and torch.all(v[:, 3] == 9)


@pytest.mark.gpu
@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,k,t", [(1000, 1024, 200), (500, 1025, 150), (260, 1151, 900), (130, 2688, 700), (1024, 1920, 1024)])
def test_matmul_few_tiles_many_blocks(m, k, t, out_dtype, token_major):
    """Few tiles of C with 8 to 21 blocks of K, even and odd in number, whole and not."""
    test_matmul(m, k, t, out_dtype, token_major)


@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,k,t", [(20000, 300, 7), (17001, 384, 32), (16500, 128, 1), (33000, 640, 33), (40000, 256, 17)])
def test_matmul_many_rows_few_tokens(m, k, t, out_dtype):
    """A head's products: many rows of W, up to 33 tokens, whose logits lie in rows."""
    test_matmul(m, k, t, out_dtype, True)


@pytest.mark.gpu
@pytest.mark.parametrize("delta", [None, torch.bfloat16])
@pytest.mark.parametrize("t", [3, 255, 300])
@pytest.mark.parametrize("f", [1, 130, 700, 1024, 1500, 5000, 9000])
def test_norm_infinite_last_feature(f, t, delta):
    """An infinity in any place, the last feature among them, makes 1 / rms zero: its own block stands for
    NaN, the token's other blocks for zero, and the other tokens are what they are without it."""
    h = rand(f, t, seed=21)
    d = None if delta is None else torch.zeros(f, t, dtype=delta, device="cuda")
    w = torch.ones(f, device="cuda")
    _, q0, s0 = add_rmsnorm_fp8(h, d, w)
    for token, at in enumerate(dict.fromkeys([f - 1, 0, f // 2])):
        x = h.clone()
        x[at, token] = float("-inf")
        _, q, s = add_rmsnorm_fp8(x, d, w)
        v = q.float() * s.repeat_interleave(BLOCK, 0)[:f].t()
        b = at // BLOCK
        own = slice(b * BLOCK, min(f, (b + 1) * BLOCK))
        assert torch.isnan(v[token, own]).all()
        v[token, own] = 0
        assert torch.all(v[token] == 0)
        keep = torch.arange(t, device="cuda") != token
        assert torch.equal(q[keep].float(), q0[keep].float()) and torch.equal(s[:, keep], s0[:, keep])


@pytest.mark.gpu
@pytest.mark.parametrize("wide", [0, 8000])
@pytest.mark.parametrize("t", [4, 300])
def test_norm_borders(t, wide):
    """The norm's bytes are 448 y / max |y| of their block, in which 1 / rms cancels, rounded to the even
    neighbour where that lies on a border: the quantisation's rule."""
    g = torch.Generator().manual_seed(31)
    largest = 1 + torch.randint(0, 128, (300,), generator=g) / 128  # bf16 values
    ratio = torch.tensor([448.0, 21, -84, 9, 5.5, 300, 13, -1.75 / 2, 42, 10.5, 26, -168])
    h = torch.zeros(2 * BLOCK + wide, t)
    for b in range(2):
        m = largest[torch.arange(t) % 150 + 150 * b]
        h[b * BLOCK:b * BLOCK + 12] = (ratio[:, None].double() * m.double() / 448).float()
    h = h.to("cuda")
    exact = h.double()
    for b in range(2):
        part = exact[b * BLOCK:(b + 1) * BLOCK]
        top = part.abs().max(0, keepdim=True).values
        part.mul_(448).div_(top)
    # (products with 448 and quotients on a border are exact in float64 where h is)
    step = torch.exp2(torch.floor(torch.log2(exact.abs().clamp_min(2.0 ** -6))) - 3)
    want = torch.round(exact / step) * step
    for delta in (None, torch.zeros(2 * BLOCK + wide, t, dtype=torch.bfloat16, device="cuda")):
        _, q, _ = add_rmsnorm_fp8(h, delta, torch.ones(2 * BLOCK + wide, device="cuda"))
        assert torch.equal(q.double().t(), want)


def lazily_negated(x, strided=False):
    """x's values as a view that torch has yet to negate: contiguous, or the imaginary part of a conjugate."""
    y = torch.complex(x.float(), -x.float()).conj().imag if strided else torch._neg_view(-x)
    assert y.is_neg() and torch.equal(y, x)
    return y


@pytest.mark.gpu
@pytest.mark.parametrize("t", [5, 300])
def test_lazily_negated(t):
    """Operands that torch holds lazily negated give what their values give."""
    f = 300
    h, d, x = rand(f, t, seed=41), rand(f, t, seed=42, dtype=torch.bfloat16), rand(f, t, seed=43)
    w, weight = rand(200, f, seed=44), torch.rand(f, device="cuda") - 0.5
    same = lambda a, b: all(torch.equal(i.float(), j.float()) for i, j in zip(a, b))  # noqa: E731
    want = quantize_fp8(x)
    assert same(quantize_fp8(lazily_negated(x)), want) and same(quantize_fp8(lazily_negated(x, True)), want)
    want = add_rmsnorm_fp8(h, d, weight)
    for strided in (False, True):
        neg = lambda v: lazily_negated(v, strided)  # noqa: E731
        assert same(add_rmsnorm_fp8(neg(h), lazily_negated(d), neg(weight)), want)
    assert same(add_rmsnorm_fp8(lazily_negated(h), None, weight), add_rmsnorm_fp8(h, None, weight))
    wq, ws = quantize_fp8_weight(w)
    assert same(quantize_fp8_weight(lazily_negated(w)), (wq, ws))
    _, xq, xs = want
    got = fp8_matmul(wq, lazily_negated(ws), xq, lazily_negated(xs))
    assert torch.equal(got, fp8_matmul(wq, ws, xq, xs))
    with pytest.raises(ValueError):
        fp8_matmul(wq, ws, xq, xs, out=lazily_negated(got))


@pytest.mark.parametrize("which", range(5))
def test_matmul_refuses_gradients(which):
    """As the other operators do: a product of operands that ask for a gradient would lose it silently."""
    a = [torch.zeros(8, 16).to(FP8), torch.ones(1, 1), torch.zeros(4, 16).to(FP8), torch.ones(1, 4),
         torch.zeros(8, 4, dtype=torch.bfloat16)]
    a[which].requires_grad_(True)
    with pytest.raises(RuntimeError, match="inference"):
        fp8_matmul(*a[:4], out=a[4])
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):
        fp8_matmul(*a[:4], out=a[4])


@pytest.mark.parametrize("call,base,kw", [
    ("mss_quant_fp8", "QUANT", dict(tokens=(1 << 27) + 1, scales=1 << 40)),
    ("mss_norm_fp8", "NORM", dict(tokens=(1 << 27) + 1, h=1 << 46, delta=1 << 47, hn=1 << 48, scales=1 << 49)),
    ("mss_quant_fp8_weight", "WEIGHT", dict(K=(1 << 30) + 1, ldw=1 << 31, ldq=1 << 31, w=1 << 46, q=1 << 47, scales=1 << 48)),
    ("mss_fp8_mm", "MM", dict(K=(1 << 30) + 1, ldw=1 << 31, ldx=1 << 31, W=1 << 46, X=1 << 47, C=1 << 48)),
])
def test_sizes_past_a_launch(lib, call, base, kw):
    """What a launch's 2^32 threads would not hold is refused."""
    args = {"QUANT": (_lib.QuantFp8Args, QUANT), "NORM": (_lib.NormFp8Args, NORM),
            "WEIGHT": (_lib.QuantFp8WeightArgs, WEIGHT), "MM": (_lib.Fp8MmArgs, MM)}[base]
    assert getattr(lib, call)(args[0](**{**args[1], **kw}), None) == 2


@pytest.mark.gpu
@pytest.mark.parametrize("token_major,out_dtype", [(False, torch.float32), (True, torch.bfloat16)])
def test_matmul_more_rows_than_one_launch_takes(token_major, out_dtype):
    """2^30 rows of W and some, 16 features, one token: each output against its float32 sum."""
    m = (1 << 30) + 200
    g = torch.Generator(device="cuda").manual_seed(51)
    wq = torch.randint(0, 127, (m, 16), generator=g, device="cuda", dtype=torch.uint8).view(FP8)
    ws = torch.rand(-(-m // BLOCK), 1, generator=g, device="cuda") + 0.5
    xq, xs = quantize_fp8(rand(16, 1, seed=52))
    got = fp8_matmul(wq, ws, xq, xs, out_dtype=out_dtype, token_major=token_major).view(m)
    x = xq.float()[0] * xs[0, 0]
    step = 1 << 25
    for r in range(0, m, step):
        w = wq[r:r + step].float()
        s = ws[r // BLOCK:(r + step) // BLOCK, 0].repeat_interleave(BLOCK)[:w.shape[0]]
        want, size = (w * x).sum(1) * s, (w * x.abs()).sum(1) * s
        bound = size * (2.0 ** -10 if out_dtype == torch.bfloat16 else 23 * 2.0 ** -23)
        bound += want.abs() * (torch.finfo(out_dtype).eps / 2) * 1.01
        assert torch.all((got[r:r + step].float() - want).abs() <= bound)


@pytest.mark.gpu
@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("m,k,t", [(16, 128, 16), (40, 256, 5), (130, 1100, 70), (1280, 2560, 333), (20000, 300, 7),
                                   (2100, 200, 2200), (300, 1024, 140)])
def test_matmul_float32_keeps_what_outliers_hide(m, k, t, token_major):
    """Small whole numbers next to large products that cancel within 8 features: every sum is a whole
    number below 2^24 on the way, so a float32 output is exact. A bf16 output is off by its rounding and
    at most 7 of the 8 products' 2^-13 of the largest, in every 8."""
    g = torch.Generator(device="cuda").manual_seed(61)
    w = torch.randint(-4, 5, (m, k), generator=g, device="cuda").float()
    x = torch.randint(-4, 5, (t, k), generator=g, device="cuda").float()
    at = torch.arange(3, k - 1, 128, device="cuda")
    w[:, at], w[:, at + 1], x[:, at], x[:, at + 1] = 448, -448, 448, 448
    want = (w.double().cpu() @ x.double().cpu().t()).cuda()
    rows = lambda v: torch.nn.functional.pad(v, (0, -k % 16)).to(FP8)[:, :k]  # noqa: E731
    one = lambda *s: torch.ones(*s, device="cuda")  # noqa: E731
    kb = -(-k // BLOCK)
    a = rows(w), one(-(-m // BLOCK), kb), rows(x), one(kb, t)
    got = fp8_matmul(*a, out_dtype=torch.float32, token_major=token_major)
    assert torch.equal((got.t() if token_major else got).double(), want)
    got = fp8_matmul(*a, token_major=token_major).double()
    bound = 7 * 2.0 ** -13 * (448 * 448 * len(at) + 16 * (k // 8 + 1))
    assert torch.all(((got.t() if token_major else got) - want).abs() <= bound + (want.abs() + bound) * 2.0 ** -8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("f,t", [(2560, 200), (2560, 208), (2560, 400), (2560, 417), (5120, 129), (5120, 205), (129, 4099),
                                 (64, 8200), (20000, 63), (20000, 64), (9000, 127)])
def test_quantise_both_sides_of_the_tiles(f, t, dtype):
    """Token-contiguous activations about the size from which tiles of 64 tokens take them, whole and not."""
    for layout in ("channel", "rows_apart"):
        test_quantise(f, t, layout, dtype)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """More than 2^32 values in every operand of a kind: the last tokens, and rows, against the same by
    themselves."""
    g = torch.Generator(device="cuda").manual_seed(71)
    f, t = 257, (1 << 24) + 5
    x = torch.randn(f, t, generator=g, device="cuda", dtype=torch.bfloat16)
    same = lambda a, b: all(torch.equal(i.float(), j.float()) for i, j in zip(a, b))  # noqa: E731
    end = slice(t - 100, t)
    q, s = quantize_fp8(x)
    assert same((q[end], s[:, end]), quantize_fp8(x[:, end].contiguous()))
    del q, s
    h = x.float()
    w = torch.ones(f, device="cuda")
    hn, q, s = add_rmsnorm_fp8(h, x, w)
    want = add_rmsnorm_fp8(h[:, end].contiguous(), x[:, end].contiguous(), w)
    assert torch.equal(hn[:, end], want[0])
    # (the kernel for few tokens adds the squares in another order: scales to float32 roundings of f + 6)
    assert torch.equal(q[end].float(), want[1].float())
    assert torch.allclose(s[:, end], want[2], rtol=(f + 12) * 2.0 ** -24, atol=0)
    del x, h, hn, q, s
    m, k, t = 50280, 32, 90001
    wq, ws = quantize_fp8_weight(torch.randn(m, k, generator=g, device="cuda"))
    xq, xs = quantize_fp8(torch.randn(k, t, generator=g, device="cuda"))
    for token_major in (False, True):
        got = fp8_matmul(wq, ws, xq, xs, token_major=token_major)
        if token_major:
            got = got.t()
        part = slice(m // BLOCK * BLOCK, m)
        check_mm(got[part, -300:], wq[part], ws[-1:], xq[-300:], xs[:, -300:].contiguous(), False, torch.bfloat16)
        del got


@pytest.mark.gpu
def test_weight_offsets_past_32_bits():
    m, k = 4000, 1100000
    w = torch.randn(m, k, generator=torch.Generator(device="cuda").manual_seed(72), device="cuda", dtype=torch.bfloat16)
    q, s = quantize_fp8_weight(w)
    end = m // BLOCK * BLOCK
    q1, s1 = quantize_fp8_weight(w[end:].contiguous())
    assert torch.equal(q[end:].float(), q1.float()) and torch.equal(s[-1:], s1)
    x, xs = quantize_fp8(torch.randn(k, 3, device="cuda"))
    for out_dtype in (torch.bfloat16, torch.float32):
        got = fp8_matmul(q, s, x, xs, out_dtype=out_dtype)
        check_mm(got[end:], q1, s1, x, xs, False, out_dtype)
