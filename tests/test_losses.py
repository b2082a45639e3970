"""Losses of a language model: the head's cross-entropy without logits (the reference takes it of its
head's logits, experiments/mamba_inductionheads.py:129-136), distillation from a teacher's top logits,
from the head's operands and from logits.

CPU: refusals. GPU: against the definitions in float64 on the same inputs, gradients against the
formula's and against differences.

Tolerances, per element, in units of U = 2^-24 (half a float32 step). A product's sum of n terms counts a whole
step, 2 U, for each addition, relative to the sum S of the magnitudes, and 16 more for the planes that
a float32 operand is split in and that leave 2^-24 of it: (n + 16) 2 U S. With dz that bound for a
logit, M the largest logarithm to base 2 that a row meets (its largest |logit| / temperature log2 e, and
log2 V), K its words and A = min(V, 128 + V / 512) the longest chain of additions in the sum of the V
exponentials (of a lane, then lanes, waves and tiles): a logarithm, an exponent's argument or their difference is
off by a few M U, the sum by A steps, so that lse / temperature is off by dz / temperature + (8 M + 4 A + 8) U, a
loss by temperature^2 (2 dz / temperature + (16 M + 4 A + 16 + 4 K (M + 1)) U); a word's probability relative
to itself by twice dz / temperature + (16 M + 4 A + 16) U, q by (K + 16) U. g is rounded to bfloat16
(2^-8) where x is, and the gradients to their types.
"""
import numpy as np
import pytest
import torch

from mamba_amd import _lib
from mamba_amd.losses import distill_loss, linear_cross_entropy, linear_distill_loss
from mamba_amd.lm_ops import GradHolder, cross_entropy

U = 2.0 ** -24
BF16, F32 = torch.bfloat16, torch.float32
HALF = {BF16: 2.0 ** -8, F32: U}


@pytest.fixture(scope="module")
def lib():
    return _lib.register_hip_kernel()


# ------------------------------------------------------------------------------- refusals
P = 1 << 32  # addresses far apart, multiples of 256
LINEAR = dict(tokens=20, features=64, vocab=100, top=0, io_dtype=1, teacher_dtype=0, dw_dtype=1, reduction=2, temperature=1.0,
              ignore_index=-100, stride_f=20, stride_t=1, ldw=64, x=P, weight=2 * P, targets=3 * P, ids=4 * P,
              teacher=5 * P, loss=6 * P, mean=7 * P, saved=8 * P, workspace=9 * P, saved_bytes=1 << 40,
              workspace_bytes=1 << 31, grad=10 * P, dx=11 * P, dweight=12 * P)


@pytest.mark.parametrize("kw,status", [
    (dict(tokens=0), 1), (dict(features=0), 1), (dict(vocab=0), 1), (dict(top=-1), 1), (dict(io_dtype=2), 1),
    (dict(reduction=3), 1), (dict(reduction=-1), 1), (dict(temperature=2.0), 1), (dict(stride_f=-1), 1),
    (dict(stride_t=-1), 1), (dict(ldw=63), 1), (dict(x=None), 1), (dict(weight=None), 1), (dict(targets=None), 1),
    (dict(loss=None), 1), (dict(mean=None), 1), (dict(saved=None), 1), (dict(x=P + 1), 1), (dict(weight=2 * P + 1), 1),
    (dict(saved=8 * P + 16), 4), (dict(saved_bytes=100), 4), (dict(workspace=None), 4), (dict(workspace_bytes=10), 4),
    (dict(workspace=9 * P + 8), 4), (dict(loss=P), 1), (dict(mean=2 * P), 1), (dict(saved=3 * P), 1),
    (dict(workspace=P), 1), (dict(loss=7 * P), 1), (dict(tokens=1 << 21), 2), (dict(vocab=1 << 21), 2),
    (dict(features=1 << 17, ldw=1 << 17), 2), (dict(tokens=1 << 19, vocab=1 << 20), 2),
    (dict(top=5, ids=None), 1), (dict(top=5, teacher=None), 1), (dict(top=5, teacher_dtype=4), 1),
    (dict(top=5, temperature=0.0), 1), (dict(top=5, temperature=-1.0), 1), (dict(top=5, temperature=float("nan")), 1),
    (dict(top=5, temperature=float("inf")), 1), (dict(top=5, temperature=1e-39), 1), (dict(top=1025), 2),
    (dict(top=1000, tokens=1 << 18), 2), (dict(top=5, loss=4 * P), 1), (dict(top=5, saved=5 * P), 1),
])
def test_linear_validation(lib, kw, status):
    assert lib.mss_linear_loss_fwd(_lib.LinearLossArgs(**{**LINEAR, **kw}), None) == status


@pytest.mark.parametrize("kw,status", [
    (dict(grad=None), 1), (dict(dx=None, dweight=None), 1), (dict(dw_dtype=5), 1),
    (dict(weight=None), 1), (dict(saved=None), 1), (dict(dx=2 * P), 1), (dict(dweight=8 * P), 1), (dict(dx=12 * P), 1),
    (dict(dx=10 * P), 1), (dict(workspace=2 * P), 1), (dict(workspace_bytes=10), 4), (dict(saved_bytes=10), 4),
])
def test_linear_backward_validation(lib, kw, status):
    assert lib.mss_linear_loss_bwd(_lib.LinearLossArgs(**{**LINEAR, **kw}), None) == status
    assert lib.mss_linear_loss_bwd(None, None) == lib.mss_linear_loss_fwd(None, None) == 1
    assert lib.mss_linear_loss_saved_bytes(None) == lib.mss_linear_loss_workspace_bytes(None, 1) == 0


BIG = dict(LINEAR, tokens=4096, features=1024, vocab=1 << 17, stride_f=4096, ldw=1024, workspace_bytes=1 << 40)


@pytest.mark.parametrize("kw,status", [
    (dict(tokens=4), 2), (dict(io_dtype=0), 2), (dict(reduction=0), 2), (dict(x=None), 1), (dict(weight=None), 1),
    (dict(targets=None), 1), (dict(loss=None), 1), (dict(mean=None), 1), (dict(dx=None), 1), (dict(dweight=None), 1),
    (dict(dw_dtype=3), 1), (dict(workspace_bytes=1 << 20), 4), (dict(saved_bytes=100), 4), (dict(dx=P), 1), (dict(dx=12 * P), 1),
    (dict(dweight=2 * P), 1), (dict(dweight=8 * P), 1), (dict(dx=9 * P), 1), (dict(loss=11 * P), 1),
])
def test_linear_both_validation(lib, kw, status):
    assert lib.mss_linear_loss_fwd_grad(_lib.LinearLossArgs(**{**BIG, **kw}), None) == status
    assert lib.mss_linear_loss_fwd_grad(None, None) == 1


@pytest.mark.parametrize("kw,status", [
    (dict(tokens=4), 2), (dict(io_dtype=0), 2), (dict(reduction=0), 2), (dict(dx=None), 1), (dict(dweight=None), 1), (dict(grad=None), 1),
    (dict(dw_dtype=3), 1), (dict(dx=10 * P), 1), (dict(dweight=11 * P), 1),
])
def test_linear_rescale_validation(lib, kw, status):
    assert lib.mss_linear_loss_rescale(_lib.LinearLossArgs(**{**BIG, **kw}), None) == status
    assert lib.mss_linear_loss_rescale(None, None) == 1


def test_linear_workspaces(lib):
    def sizes(**kw):
        return [lib.mss_linear_loss_workspace_bytes(_lib.LinearLossArgs(**{**BIG, **kw}), i) for i in (-1, 0, 1, 2, 3)]
    none, fwd, bwd, both, none2 = sizes()
    assert none == none2 == 0 and 0 < fwd < bwd < both
    assert sizes(io_dtype=0)[3] == sizes(reduction=0)[3] == sizes(tokens=4)[3] == 0
    # A weight whose rows lie further apart than 32 bits address in a tile is copied.
    saved = [lib.mss_linear_loss_saved_bytes(_lib.LinearLossArgs(**{**LINEAR, "ldw": ldw})) for ldw in (64, 1 << 22, (1 << 22) + 8)]
    assert saved[0] == saved[1] and saved[2] >= saved[1] + 100 * 64 * 2


# Tiles of the gradients' products: rows, columns, stages of the ring, workgroups a CU.
SMALL, LARGE, THIN = (128, 128, 2, 2), (256, 256, 2, 1), (128, 32, 4, 2)


def _parts(tile, rows, cols, k, pairs, dx):
    """Floats of the parts that the product's teams leave: 256 CUs' workgroups in teams of one for each tile of features;
    ranges that are dealt out whole unless some team would then be 8 units longer than an even share, two parts
    a team else."""
    up = lambda a, b: -(-a // b)
    m, n, ring, per_cu = tile
    units = up(up(k, 128) * 2 * pairs, ring)
    size, ranges = (up(rows, m), up(cols, n))[::1 if dx else -1]
    units_all, at_once = ranges * units, max(1, 256 * per_cu // size)
    shares = max(1, min(units_all // 8, at_once))
    whole = up(ranges, at_once) * units <= units_all // shares + 8
    return 0 if whole else 2 * shares * size * m * n


def _backward_plan(t, d, v, planes):
    """The pieces of the vocabulary and, for each, the floats of its gradients' parts."""
    up = lambda a, b: -(-a // b)
    most = max(256, (1 << 30) // (2 * planes * t) // 256 * 256)
    piece = up(up(v, 256), up(up(v, 256) * 256, most)) * 256
    large = lambda r, c: 4 * up(r, 256) * up(c, 256) <= 1.4 * up(r, 128) * up(c, 128)
    tile_x = THIN if t <= 32 else LARGE if t > 384 and large(d, t) else SMALL
    tile_w = LARGE if large(min(piece, v), d) else SMALL
    pairs = 1 if planes == 1 else 3
    words = {min(piece, v - a) for a in range(0, v, piece)}
    return piece, max(max(_parts(tile_x, d, t, n, pairs, True), _parts(tile_w, n, d, t, pairs, False)) for n in words)


def _sweep():
    shapes = [(16384, 1024, 32000), (24576, 2048, 32000), (19037, 2560, 152390), (16384, 896, 128256), (16384, 1024, 128256),
              (32768, 2048, 32000), (1602, 320, 352845), (543, 384, 554631), (1, 64, 1 << 20), (33, 40, 1 << 20)]
    for v in (4096, 10007, 32000, 32768, 50280, 65024, 100352, 128256, 152064, 202048, 256000):
        for d in (64, 320, 512, 640, 768, 896, 1024, 1536, 2048, 2560, 4096):
            shapes += [(t, d, v) for t in range(1024, 32769, 1024)]
    return shapes


def test_linear_workspace_holds_the_parts_of_every_piece(lib):
    """The parts are the workspace's last buffer. Its size has to be what the largest of the vocabulary's pieces leaves:
    the last one has fewer words, and may be shared out where the others are dealt out whole."""
    step = lambda n: -(-n // 256) * 256
    several = 0
    for t, d, v in _sweep():
        for planes in (1, 2):
            for reduction in (0, 2):
                a = _lib.LinearLossArgs(**{**LINEAR, "tokens": t, "features": d, "vocab": v, "ldw": d, "reduction": reduction,
                                           "io_dtype": 2 - planes})
                piece, parts = _backward_plan(t, d, v, planes)
                before = (step(8 * (t + 256)) if reduction == 0 else 0) + 256 + step(2 * planes * t * piece)
                before += step(4 * d * (-(-t // 4) * 4)) if piece < v else 0
                room = lib.mss_linear_loss_workspace_bytes(a, 1) - before
                assert room == step(4 * parts), (t, d, v, planes, room, 4 * parts)
                several += piece < v
    assert several > 1000


def test_linear_workspace_holds_the_parts_of_every_block(lib):
    """The same for both directions at once, in blocks of tokens."""
    step = lambda n: -(-n // 256) * 256
    several = 0
    for t, d, v in _sweep():
        a = _lib.LinearLossArgs(**{**LINEAR, "tokens": t, "features": d, "vocab": v, "ldw": d})
        total = lib.mss_linear_loss_workspace_bytes(a, 2)
        if total == 0:
            continue
        lde = -(-v // 256) * 256
        rows = (1 << 30) // (2 * lde) // 256 * 256
        block = -(--(-t // -(-t // rows)) // 256) * 256
        parts = max(max(_parts(LARGE, d, n, v, 1, True), _parts(LARGE, v, d, n, 1, False))
                    for n in {min(block, t - b) for b in range(0, t, block)})
        rest = total - step(4 * parts)
        # (what else is there: sums of the forward call's tiles, scales, the block's logits, sums of rows and of dw, notes)
        least = step(8 * (t + 256)) + step(2 * block * lde) + step(lde // 256 * 2 * block * 4) + (step(4 * v * d) if block < t else 0)
        sums = rest - least - step(4 * -(-t // block))
        assert sums in [step(8 * t * n) for n in (-(-v // 128) * 2, -(-v // 256) * 2, -(-v // 256) * 4)], (t, d, v)
        several += block < t
    assert several > 1000


DISTILL = dict(rows=20, vocab=100, top=5, io_dtype=1, teacher_dtype=0, reduction=2, temperature=1.0, ld=100, logits=P, ids=2 * P,
               teacher=3 * P, loss=4 * P, mean=5 * P, saved=6 * P, saved_bytes=1 << 31, grad=7 * P, dlogits=8 * P)


@pytest.mark.parametrize("kw,status", [
    (dict(rows=0), 1), (dict(vocab=0), 1), (dict(top=0), 1), (dict(io_dtype=2), 1), (dict(teacher_dtype=-1), 1),
    (dict(reduction=4), 1), (dict(temperature=0.0), 1), (dict(temperature=float("nan")), 1), (dict(ld=99), 1),
    (dict(logits=None), 1), (dict(ids=None), 1), (dict(teacher=None), 1), (dict(loss=None), 1), (dict(mean=None), 1),
    (dict(saved=None), 1), (dict(dlogits=None), 1), (dict(logits=P + 1), 1), (dict(dlogits=8 * P + 1), 1),
    (dict(reduction=0), 1), (dict(saved=6 * P + 4), 4), (dict(saved_bytes=64), 4), (dict(top=1025), 2),
    (dict(rows=1 << 18, top=1000), 2), (dict(rows=(1 << 21) + 1, top=1), 2), (dict(vocab=(1 << 30) + 1, ld=1 << 31), 2), (dict(dlogits=P + 256), 1),
    (dict(loss=P), 1), (dict(saved=2 * P), 1), (dict(mean=4 * P), 1), (dict(dlogits=4 * P), 1), (dict(dlogits=6 * P), 1),
])
def test_distill_validation(lib, kw, status):
    assert lib.mss_distill_fwd_grad(_lib.DistillArgs(**{**DISTILL, **kw}), None) == status
    assert lib.mss_distill_fwd(None, None) == lib.mss_distill_bwd(None, None) == lib.mss_distill_regrad(None, None) == 1
    assert lib.mss_distill_saved_bytes(None) == 0


@pytest.mark.parametrize("kw", [dict(grad=None), dict(dlogits=None), dict(dlogits=7 * P), dict(dlogits=P)])
def test_distill_backward_validation(lib, kw):
    a = _lib.DistillArgs(**{**DISTILL, **kw})
    assert lib.mss_distill_bwd(a, None) == lib.mss_distill_regrad(a, None) == 1


def test_addresses_off_their_type_are_refused(lib):
    """Each address, in the calls that take it."""
    big = {**BIG, "saved_bytes": 1 << 40}
    lists, tgts = dict(big, top=5), dict(big)

    def refused(call, base, kw):
        return call(_lib.LinearLossArgs(**{**base, **kw}) if base is not DISTILL else _lib.DistillArgs(**{**base, **kw}), None) == 1
    for call in (lib.mss_linear_loss_fwd, lib.mss_linear_loss_fwd_grad):
        for kw in (dict(x=P + 1), dict(weight=2 * P + 1), dict(loss=6 * P + 2), dict(mean=7 * P + 1), dict(targets=3 * P + 4)):
            assert refused(call, tgts, kw), kw
        for kw in (dict(ids=4 * P + 4), dict(teacher=5 * P + 2), dict(teacher=5 * P + 1, teacher_dtype=1)):
            assert refused(call, lists, kw), kw
    for call in (lib.mss_linear_loss_bwd, lib.mss_linear_loss_fwd_grad, lib.mss_linear_loss_rescale):
        for kw in (dict(dx=11 * P + 1), dict(dweight=12 * P + 1), dict(dweight=12 * P + 2, dw_dtype=0)):
            assert refused(call, tgts, kw), kw
    for call in (lib.mss_linear_loss_bwd, lib.mss_linear_loss_rescale):
        assert refused(call, tgts, dict(grad=10 * P + 2))
    for call in (lib.mss_distill_fwd, lib.mss_distill_fwd_grad):
        for kw in (dict(ids=2 * P + 4), dict(teacher=3 * P + 2), dict(loss=4 * P + 1), dict(mean=5 * P + 2), dict(logits=P + 1)):
            assert refused(call, DISTILL, kw), kw
    for call in (lib.mss_distill_bwd, lib.mss_distill_regrad):
        for kw in (dict(grad=7 * P + 2), dict(dlogits=8 * P + 1)):
            assert refused(call, DISTILL, kw), kw


def test_struct_layouts_match_the_header(tmp_path):
    import ctypes
    import subprocess
    from pathlib import Path
    structs = {"mss_linear_loss_args": _lib.LinearLossArgs, "mss_distill_args": _lib.DistillArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "mamba_selective_scan.h"', "int main(void) {"]
    for c, cls in structs.items():
        lines.append(f'  printf("%zu\\n", sizeof({c}));')
        lines += [f'  printf("%zu\\n", offsetof({c}, {f}));' for f, _ in cls._fields_]
    (tmp_path / "l.c").write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    root = Path(__file__).resolve().parents[1]
    subprocess.run(["gcc", "-std=c99", "-I", str(root / "include"), str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    seen = [int(v) for v in subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout.split()]
    want = [v for cls in structs.values() for v in (ctypes.sizeof(cls), *(getattr(cls, f).offset for f, _ in cls._fields_))]
    assert seen == want


def test_python_refusals():
    x, w, tg = torch.randn(8, 5), torch.randn(11, 8), torch.zeros(5, dtype=torch.int64)
    ids, te = torch.zeros(5, 3, dtype=torch.int64), torch.randn(5, 3)
    ce, ld, ds = linear_cross_entropy, linear_distill_loss, distill_loss
    z = torch.randn(5, 11)
    for call in (lambda: ce(x, w, tg[:4]), lambda: ce(x, w, tg.int()), lambda: ce(x[0], w, tg), lambda: ce(x, w[:, :7], tg),
                 lambda: ce(x, w, tg, reduction="avg"), lambda: ce(x, w[:0], tg), lambda: ce(x[:0], w[:, :0], tg),
                 lambda: ce(x, w, tg, weight_act=w.bfloat16()), lambda: ce(x, w, tg, weight_act=w[:5]),
                 lambda: ce(x.bfloat16(), w.bfloat16(), tg, holder=GradHolder()),
                 lambda: ld(x, w, ids[:4], te), lambda: ld(x, w, ids.int(), te), lambda: ld(x, w, ids, te[:, :2]),
                 lambda: ld(x, w, ids, te, temperature=0.0), lambda: ld(x, w, ids, te, temperature=float("nan")),
                 lambda: ld(x, w, torch.zeros(5, 1025, dtype=torch.int64), torch.zeros(5, 1025)),
                 lambda: ds(z[0], ids, te), lambda: ds(z, ids, te[:4]), lambda: ds(z, ids, te, temperature=-1),
                 lambda: ds(z[:, :0], ids, te), lambda: ds(z, ids, te, reduction=None)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ce(x.half(), w, tg), lambda: ce(x, w.double(), tg), lambda: ld(x, w, ids, te.half()),
                 lambda: ds(z.double(), ids, te)):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: ce(x, w, tg), lambda: ld(x, w, ids, te), lambda: ds(z, ids, te)):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            call()
    with pytest.raises(RuntimeError, match="detach"):
        ds(z, ids, te.requires_grad_())
    rows = (1 << 21) + 1
    with pytest.raises(ValueError, match="rows"):
        ds(torch.zeros(1, 1).expand(rows, 1), torch.zeros(1, 1, dtype=torch.int64).expand(rows, 1), torch.zeros(1, 1).expand(rows, 1))


class _Hooks:
    """Saved-tensor hooks that keep a copy, as offloading and checkpoints do; `layout` gives the copy its layout."""

    def __init__(self, layout=torch.Tensor.clone):
        self.layout, self.unpacked = layout, []

    def pack(self, t):
        return self.layout(t.detach())

    def unpack(self, t):
        self.unpacked.append(t)
        return t

    def __enter__(self):
        self.context = torch.autograd.graph.saved_tensors_hooks(self.pack, self.unpack)
        return self.context.__enter__()

    def __exit__(self, *e):
        return self.context.__exit__(*e)


class _Calls:
    """The library, its sizes its own, with calls that are noted instead of made."""

    def __init__(self, lib):
        self.lib, self.seen = lib, []

    def __getattr__(self, name):
        if name.endswith("_bytes"):
            return getattr(self.lib, name)

        def call(a, stream):
            self.seen.append((name, type(a).from_buffer_copy(a)))
            return 0
        return call


@pytest.fixture
def calls(lib, monkeypatch):
    import contextlib

    from mamba_amd import losses
    noted = _Calls(lib)
    monkeypatch.setattr(losses._lib, "register_hip_kernel", lambda: noted)
    monkeypatch.setattr(losses, "_stream", lambda t: None)
    monkeypatch.setattr(losses, "_require_gpu", lambda *a: None)
    monkeypatch.setattr(losses, "_guard", lambda t: contextlib.nullcontext())
    return noted


def _off_16(t):
    """A copy whose rows lie off 16 bytes and further apart."""
    if t.dim() != 2:
        return t.clone()
    wide = torch.zeros(t.shape[0], t.shape[1] + 3, dtype=t.dtype)
    wide[:, 1:1 + t.shape[1]] = t
    return wide[:, 1:1 + t.shape[1]]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d,layout,given", [(64, "clone", "plain"), (64, "off", "plain"), (64, "clone", "off"), (64, "t", "plain"),
                                            (40, "clone", "plain"), (40, "off", "plain")])
def test_linear_backward_reads_what_the_hooks_return(calls, lib, dtype, d, layout, given):
    x, w = torch.randn(d, 20).to(dtype).requires_grad_(True), torch.randn(100, d).to(dtype)
    w = (_off_16(w) if given == "off" else w).requires_grad_(True)
    hooks = _Hooks({"clone": lambda t: t.clone(memory_format=torch.contiguous_format), "off": _off_16,
                    "t": lambda t: t.t().contiguous().t() if t.dim() == 2 else t.clone()}[layout])
    with hooks:
        loss = linear_cross_entropy(x, w, torch.zeros(20, dtype=torch.int64))
    torch.autograd.grad(loss, (x, w))
    (_, fwd), (name, a) = calls.seen
    w2, saved = hooks.unpacked
    assert name == "mss_linear_loss_bwd" and a.saved == saved.data_ptr() != fwd.saved and a.saved_bytes == saved.numel()
    assert a.weight != fwd.weight and a.ldw >= d
    assert lib.mss_linear_loss_saved_bytes(a) <= a.saved_bytes  # what the call takes from it is there
    if layout == "clone":
        assert a.weight == w2.data_ptr() and a.ldw == d


@pytest.mark.parametrize("layout", ["clone", "off", "t"])
@pytest.mark.parametrize("reduction,second", [("mean", False), ("none", False), ("sum", True)])
def test_distill_backward_reads_what_the_hooks_return(calls, layout, reduction, second):
    z, ids = torch.randn(20, 100, requires_grad=True), torch.zeros(20, 3, dtype=torch.int64)
    hooks = _Hooks({"clone": torch.Tensor.clone, "off": _off_16, "t": lambda t: t.t().contiguous().t() if t.dim() == 2 else t.clone()}[layout])
    with hooks:
        loss = distill_loss(_off_16(z), ids, torch.zeros(20, 3), reduction=reduction)
    up = torch.ones_like(loss)
    torch.autograd.grad(loss, (z,), up, retain_graph=second)
    if second:
        torch.autograd.grad(loss, (z,), up)
    (_, fwd), (name, a) = calls.seen[0], calls.seen[-1]
    logits, saved = hooks.unpacked[-2:]
    assert name == ("mss_distill_regrad" if reduction == "mean" else "mss_distill_bwd")
    assert a.saved == saved.data_ptr() != fwd.saved and a.saved_bytes == saved.numel() and a.logits != fwd.logits
    if layout == "t":
        assert a.ld == 100
    else:
        assert a.logits == logits.data_ptr() and a.ld == logits.stride(0)


def test_backward_reads_another_layout_at_the_same_address(calls):
    """Memory that was freed and given out again: the address is the forward call's, the rows lie closer."""
    def closer(t):
        return t.as_strided(t.shape, (t.shape[1], 1)) if t.dim() == 2 else t.clone()
    x, targets = torch.randn(64, 20, requires_grad=True), torch.zeros(20, dtype=torch.int64)
    wide = torch.zeros(100, 72)[:, :64].requires_grad_(True)
    with _Hooks(closer):
        loss = linear_cross_entropy(x, wide, targets)
    torch.autograd.grad(loss, (x,))
    fwd, bwd = (a for _, a in calls.seen)
    assert bwd.weight == fwd.weight and (fwd.ldw, bwd.ldw) == (72, 64)
    with _Hooks(closer):
        loss = distill_loss(wide, torch.zeros(100, 3, dtype=torch.int64), torch.zeros(100, 3))
    torch.autograd.grad(loss, (wide,))
    fwd, bwd = (a for _, a in calls.seen[2:])
    assert bwd.logits == fwd.logits and (fwd.ld, bwd.ld) == (72, 64)


def test_operands_on_several_devices_are_refused(calls):
    x, w, tg = torch.randn(8, 5), torch.randn(11, 8), torch.zeros(5, dtype=torch.int64)
    ids, te, z = torch.zeros(5, 3, dtype=torch.int64), torch.randn(5, 3), torch.randn(5, 11)
    for f, operands in ((linear_cross_entropy, (x, w, tg)), (linear_distill_loss, (x, w, ids, te)), (distill_loss, (z, ids, te))):
        f(*operands)
        for i in range(len(operands)):
            with pytest.raises(ValueError, match="devices"):
                f(*(t.to("meta") if j == i else t for j, t in enumerate(operands)))
    with pytest.raises(ValueError, match="devices"):
        linear_cross_entropy(x, w, tg, weight_act=w.to("meta"))
    assert len(calls.seen) == 3


# ------------------------------------------------------------------------------- the definitions
def _wanted_targets(targets, vocab, ignore=-100):
    q = torch.zeros(targets.shape[0], vocab, dtype=torch.float64, device=targets.device)
    live = targets != ignore
    rows = live.nonzero()[:, 0]
    q[rows, targets[rows]] = 1.0
    return q, live


def _wanted_lists(ids, teacher, temperature, vocab):
    q = torch.zeros(ids.shape[0], vocab, dtype=torch.float64, device=ids.device)
    t = teacher.double() / temperature
    for r in range(ids.shape[0]):
        at = ((ids[r] >= 0) & (teacher[r] != -torch.inf)).nonzero()[:, 0]
        if len(at):
            q[r].index_add_(0, ids[r][at], torch.softmax(t[r][at], 0))
    return q, q.sum(1) > 0


class _Bounds:
    """Losses and gradients in float64, with what the module's docstring allows them to be off by. z: logits, dz
    their own bound."""

    def __init__(self, z, dz, q, live, temperature, k, dtype):
        self.live = live
        v = min(z.shape[1], 128 + z.shape[1] / 512)
        s = z / temperature
        lse = torch.logsumexp(s, 1)
        at = torch.where(live, s.masked_fill(s == -torch.inf, 0).abs().amax(1), 0.0)
        m = at * np.log2(np.e) + np.log2(max(2, z.shape[1]))
        dz = dz / temperature
        self.loss = torch.where(live, temperature ** 2 * (torch.special.xlogy(q, q) - torch.where(
            q > 0, q * (s - lse[:, None]), 0.0)).sum(1), 0.0)
        self.loss_tol = temperature ** 2 * (2 * dz + U * (16 * m + 4 * v + 16 + 4 * k * (m + 1))) * live
        p = torch.exp(s - lse[:, None])
        self.g = torch.where(live[:, None], temperature * (p - q), 0.0)
        rel = 2 * dz + U * (16 * m + 4 * v + 16)
        self.g_tol = temperature * torch.where(live[:, None], p * rel[:, None] + q * U * (k + 16), 0.0)
        self.g_tol += (HALF[dtype] + 8 * U) * self.g.abs()

    def reduced(self, reduction, upstream=None):
        """loss and tolerance, and each row's scale of the gradient."""
        n = max(1, int(self.live.sum()))
        up = 1.0 if upstream is None else upstream
        if reduction == "none":
            return self.loss, self.loss_tol, torch.ones_like(self.loss) * up
        by = 1.0 / n if reduction == "mean" else 1.0
        loss = self.loss.sum() * by
        return loss, self.loss_tol.sum() * by + 2 * U * loss.abs(), torch.full_like(self.loss, by) * up


def _check(name, got, want, tol):
    got = got.detach().double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    err = (got - want).abs()
    worst = float((err / tol.clamp_min(1e-300)).nan_to_num(posinf=1e300).max()) if err.numel() else 0.0
    print(f"  {name:8s} max_abs={float(err.max()) if err.numel() else 0:.3e} of tolerance {worst:.3f}", flush=True)
    assert bool(torch.isfinite(got).all()) and bool((err <= tol).all()), name


def _product_tol(a_tol, a, b, terms):
    """Bound of a @ b for a off by a_tol, b exact."""
    return torch.mm(a_tol, b.abs()) + (terms + 16) * 2 * U * torch.mm(a.abs() + a_tol, b.abs())


def _linear_reference(x, w, q, live, temperature, k):
    """x (features, tokens), w as they are read."""
    xd, wd = x.detach().double(), w.detach().double()
    xd = torch.where(live[None], xd, 0.0)  # (what a row that does not count holds is not looked at)
    z = torch.mm(xd.t(), wd.t())
    dz = (x.shape[0] + 16) * 2 * U * torch.mm(xd.abs().t(), wd.abs().t()).amax(1)
    return _Bounds(z, dz, q, live, temperature, k, x.dtype), xd, wd


def _check_linear_grads(ref, xd, wd, scale, x_dtype, w_dtype, dx, dw):
    g, g_tol = ref.g * scale[:, None], ref.g_tol * scale[:, None].abs()
    if dx is not None:
        want = torch.mm(g, wd).t()
        tol = _product_tol(g_tol, g, wd, g.shape[1]).t() + 8 * U * want.abs()
        _check("dx", dx, want, tol * (1 + HALF[x_dtype]) + HALF[x_dtype] * want.abs())
    if dw is not None:
        want = torch.mm(g.t(), xd.t())
        tol = _product_tol(g_tol.t(), g.t(), xd.t(), g.shape[0]) + 8 * U * want.abs()
        _check("dw", dw, want, tol * (1 + HALF[w_dtype]) + HALF[w_dtype] * want.abs())


def _inputs(t, d, v, dtype, seed=0, layout="cm"):
    """x (features, tokens) and a weight, in one of the layouts: channel-major, token-major, rows with gaps and off
    16 bytes."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(t, d, generator=g, device="cuda").to(dtype)
    w = (torch.randn(v, d, generator=g, device="cuda") * (2.0 / d ** 0.5)).to(dtype)
    if layout == "cm":
        return x.t().contiguous(), w
    if layout == "tm":
        return x.t(), w
    xs = torch.full((d, 2 * t + 1), float("nan"), dtype=dtype, device="cuda")
    xs[:, 1::2] = x.t()
    ws = torch.full((v + 1, d + 3), float("nan"), dtype=dtype, device="cuda")
    ws[1:, 1:1 + d] = w
    return xs[:, 1::2], ws[1:, 1:1 + d]


def _targets(t, v, masked, seed=0):
    g = torch.Generator().manual_seed(seed)
    at = torch.randint(0, v, (t,), generator=g)
    return torch.where(torch.rand(t, generator=g) < masked, -100, at).cuda()


def _lists(t, v, top, dtype=F32, seed=0, empty=0.1, again=True):
    """Lists with absent entries (whose logits are NaN or inf), words that stand twice, empty rows."""
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(v, generator=g)[:top] if v >= top else torch.randint(0, v, (top,), generator=g)
                       for _ in range(t)])
    te = (3 * torch.randn(t, top, generator=g)).to(dtype)
    if again and top > 2:
        ids[:, 2] = ids[:, 0]
    absent = torch.rand(t, top, generator=g) < 0.2
    absent[torch.rand(t, generator=g) < empty] = True
    ids = torch.where(absent, -1 - torch.randint(0, 5, (t, top), generator=g), ids)
    te = torch.where(absent, torch.tensor([float("nan"), float("inf"), 1e30])[torch.randint(0, 3, (t, top), generator=g)].to(dtype), te)
    gone = (torch.rand(t, top, generator=g) < 0.1) & ~absent
    te = torch.where(gone, torch.tensor(-float("inf"), dtype=dtype), te)
    return ids.cuda(), te.cuda()


# ------------------------------------------------------------------------------- without logits
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("t,d,v,layout,reduction,masked", [
    (1, 1, 1, "cm", "mean", 0.0), (1, 64, 2, "tm", "sum", 0.0), (3, 7, 17, "gap", "none", 0.3), (5, 64, 129, "cm", "mean", 0.4),
    (32, 96, 300, "tm", "none", 0.2), (33, 128, 255, "cm", "sum", 0.2), (64, 65, 1000, "gap", "mean", 0.1),
    (200, 192, 515, "cm", "none", 0.5), (257, 40, 640, "tm", "mean", 0.1), (130, 320, 16, "cm", "mean", 0.0),
    (1000, 64, 50, "gap", "sum", 0.9), (40, 64, 70000, "cm", "mean", 0.1)])
def test_linear_cross_entropy(dtype, t, d, v, layout, reduction, masked):
    print(f"case linear_cross_entropy {dtype} {t} {d} {v} {layout} {reduction}", flush=True)
    x, w = _inputs(t, d, v, dtype, t + v, layout)
    targets = _targets(t, v, masked, t)
    x = x.clone(memory_format=torch.preserve_format) if layout == "gap" else x
    q, live = _wanted_targets(targets, v)
    if masked:  # nothing that a masked token holds is seen
        x[:, ~live] = float("nan")
        x[:1, ~live] = float("inf")
    x.requires_grad_(True)
    w = w.detach().requires_grad_(True)
    up = torch.linspace(-1.0, 2.0, t, device="cuda") if reduction == "none" else torch.tensor(0.7, device="cuda")
    loss = linear_cross_entropy(x, w, targets, reduction=reduction)
    assert loss.dtype == F32
    dx, dw = torch.autograd.grad(loss, (x, w), up)
    assert dx.dtype == x.dtype and dw.dtype == w.dtype
    ref, xd, wd = _linear_reference(x, w, q, live, 1.0, 1)
    want, tol, scale = ref.reduced(reduction, up.double())
    _check("loss", loss, want, tol)
    _check_linear_grads(ref, xd, wd, scale, dtype, dtype, dx, dw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("t,d,v,top,temperature,reduction,tdtype", [
    (1, 8, 3, 1, 1.0, "mean", F32), (4, 64, 20, 5, 2.0, "none", BF16), (31, 100, 301, 63, 0.5, "sum", F32),
    (70, 64, 257, 64, 4.0, "mean", BF16), (129, 72, 400, 65, 1.0, "none", F32), (20, 128, 1024, 200, 3.0, "mean", F32),
    (10, 64, 1500, 1024, 2.0, "sum", F32), (300, 64, 40, 3, 2.0, "mean", BF16)])
def test_linear_distill_loss(dtype, t, d, v, top, temperature, reduction, tdtype):
    print(f"case linear_distill_loss {dtype} {t} {d} {v} {top} {temperature} {reduction}", flush=True)
    x, w = _inputs(t, d, v, dtype, t + v)
    ids, te = _lists(t, v, top, tdtype, t)
    q, live = _wanted_lists(ids, te, temperature, v)
    x[:, ~live] = float("nan")
    x.requires_grad_(True)
    w.requires_grad_(True)
    up = torch.linspace(-1.0, 2.0, t, device="cuda") if reduction == "none" else torch.tensor(-1.5, device="cuda")
    loss = linear_distill_loss(x, w, ids, te, temperature=temperature, reduction=reduction)
    dx, dw = torch.autograd.grad(loss, (x, w), up)
    ref, xd, wd = _linear_reference(x, w, q, live, temperature, top)
    want, tol, scale = ref.reduced(reduction, up.double())
    _check("loss", loss, want, tol)
    _check_linear_grads(ref, xd, wd, scale, dtype, dtype, dx, dw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,t,d,v", [(BF16, 4096, 64, 4100), (BF16, 4000, 200, 5000), (F32, 4096, 64, 4100), (F32, 8192, 40, 24000),
                                         (BF16, 9000, 64, 61000)])
def test_linear_cross_entropy_many_tiles(dtype, t, d, v):
    """Large tiles; a vocabulary in more than one piece (the last two)."""
    print(f"case many tiles {dtype} {t} {d} {v}", flush=True)
    x, w = _inputs(t, d, v, dtype, 5)
    targets = _targets(t, v, 0.1, 6)
    q, live = _wanted_targets(targets, v)
    x.requires_grad_(True)
    w.requires_grad_(True)
    loss = linear_cross_entropy(x, w, targets)
    dx, dw = torch.autograd.grad(loss, (x, w))
    n = 2048  # the reference in pieces of the tokens
    total, dw_want, dw_tol, losses = 0.0, 0.0, 0.0, 0.0
    by = 1.0 / int(live.sum())
    for a in range(0, t, n):
        part = slice(a, min(t, a + n))
        ref, xd, wd = _linear_reference(x.detach()[:, part], w, q[part], live[part], 1.0, 1)
        total, losses = total + ref.loss.sum() * by, losses + ref.loss_tol.sum() * by
        scale = torch.full_like(ref.loss, by)
        _check_linear_grads(ref, xd, wd, scale, dtype, dtype, dx[:, part], None)
        g, g_tol = ref.g * by, ref.g_tol * by
        dw_want = dw_want + torch.mm(g.t(), xd.t())
        dw_tol = dw_tol + _product_tol(g_tol.t(), g.t(), xd.t(), t)
    _check("loss", loss, total, losses + 2 * U * total)
    half = HALF[dtype]
    _check("dw", dw, dw_want, (dw_tol + 8 * U * dw_want.abs()) * (1 + half) + half * dw_want.abs())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,t,d,v,reduction", [(BF16, 1602, 320, 352845, "none"), (F32, 543, 384, 554631, "mean")])
def test_linear_last_piece_shared_otherwise(dtype, t, d, v, reduction):
    """A last piece of the vocabulary whose ranges the teams share where they take the other pieces' whole."""
    print(f"case last piece {dtype} {t} {d} {v} {reduction}", flush=True)
    piece, parts = _backward_plan(t, d, v, 1 if dtype == BF16 else 2)
    first = _backward_plan(t, d, piece, 1 if dtype == BF16 else 2)
    assert piece < v and first[0] == piece and first[1] < parts
    x, w = _inputs(t, d, v, dtype, 21)
    targets = _targets(t, v, 0.1, 22)
    x.requires_grad_(True)
    w.requires_grad_(True)
    loss = linear_cross_entropy(x, w, targets, reduction=reduction)
    up = torch.linspace(-1.0, 2.0, t, device="cuda") if reduction == "none" else torch.tensor(1.0, device="cuda")
    dx, dw = torch.autograd.grad(loss, (x, w), up)
    by = 1.0 / int((targets != -100).sum()) if reduction == "mean" else 1.0
    total, tol, dw_want, dw_tol = 0.0, 0.0, 0.0, 0.0
    for a in range(0, t, 256):
        part = slice(a, min(t, a + 256))
        ref, xd, wd = _linear_reference(x.detach()[:, part], w, *_wanted_targets(targets[part], v), 1.0, 1)
        scale = up.double()[part] if reduction == "none" else torch.full_like(ref.loss, by)
        if reduction == "none":
            _check("loss", loss[part], ref.loss, ref.loss_tol)
        total, tol = total + ref.loss.sum() * by, tol + ref.loss_tol.sum() * by
        _check_linear_grads(ref, xd, wd, scale, dtype, dtype, dx[:, part], None)
        g, g_tol = ref.g * scale[:, None], ref.g_tol * scale[:, None].abs()
        dw_want = dw_want + torch.mm(g.t(), xd.t())
        dw_tol = dw_tol + _product_tol(g_tol.t(), g.t(), xd.t(), t)
    if reduction == "mean":
        _check("loss", loss, total, tol + 2 * U * total)
    half = HALF[dtype]
    _check("dw", dw, dw_want, (dw_tol + 8 * U * dw_want.abs()) * (1 + half) + half * dw_want.abs())


# Both directions at once: a logit to base 2 is held to half a step of 2^-9, so a probability p is off by (2^(2^-10) - 1) p,
# less than 0.7 2^-10 p, and rounded to bfloat16 after that.
STEP = 2.0 ** -10


def _check_both(x, w, q, live, temperature, k, reduction, up, loss, dx, dw):
    """In pieces of the tokens. An upstream gradient that is not a power of two rounds dx and dw once more."""
    t, n = x.shape[1], 1024
    by = (1.0 / int(live.sum()) if reduction == "mean" else 1.0)
    total, tol, dw_want, dw_tol = 0.0, 0.0, 0.0, 0.0
    more = 0.0 if abs(np.log2(abs(up))) % 1 == 0 else 1.0
    for a in range(0, t, n):
        part = slice(a, min(t, a + n))
        qs = q(part)
        ref, xd, wd = _linear_reference(x.detach()[:, part], w, qs, live[part], temperature, k)
        ref.g_tol += STEP * (ref.g + temperature * qs * live[part, None])
        total, tol = total + ref.loss.sum() * by, tol + ref.loss_tol.sum() * by
        g, g_tol = ref.g * by * up, ref.g_tol * by * abs(up)
        if dx is not None:
            want = torch.mm(g, wd).t()
            bound = _product_tol(g_tol, g, wd, g.shape[1]).t() + 8 * U * want.abs()
            half = HALF[x.dtype] * (1 + more)
            _check("dx", dx[:, part], want, bound * (1 + 2 * half) + half * want.abs())
        if dw is not None:
            dw_want = dw_want + torch.mm(g.t(), xd.t())
            dw_tol = dw_tol + _product_tol(g_tol.t(), g.t(), xd.t(), t)
    _check("loss", loss, total, tol + 2 * U * total.abs())
    if dw is not None:
        half = HALF[dw.dtype] * (1 + more)
        _check("dw", dw, dw_want, (dw_tol + 8 * U * dw_want.abs()) * (1 + 2 * half) + half * dw_want.abs())


@pytest.mark.gpu
@pytest.mark.parametrize("t,d,v,layout,top,temperature,reduction,up,w_dtype", [
    (2048, 640, 53000, "cm", 0, 1.0, "mean", 1.0, BF16), (10500, 640, 53000, "tm", 0, 1.0, "sum", 0.25, F32),
    (1100, 700, 50001, "cm", 5, 2.0, "mean", -0.7, F32), (513, 1300, 66001, "gap", 0, 1.0, "mean", 1.0, BF16),
    (4100, 648, 212345, "tm", 1, 0.5, "sum", 1.0, BF16)])
def test_linear_both_directions_at_once(t, d, v, layout, top, temperature, reduction, up, w_dtype):
    """Large heads, whose gradients come with the loss; tokens in more than one block (the second and the last), and the
    gradients of a second pass, which come without it."""
    print(f"case both {t} {d} {v} {layout} {top} {temperature} {reduction} {up} {w_dtype}", flush=True)
    x, w = _inputs(t, d, v, BF16, t + v, layout)
    x = x.clone(memory_format=torch.preserve_format) if layout == "gap" else x
    if top:
        ids, te = _lists(t, v, top, F32, t) if v < 100000 else (_targets(t, v, 0.1, t)[:, None], torch.randn(t, 1, device="cuda"))
        live = ((ids >= 0) & (te != -torch.inf)).any(1)
        q = lambda part: _wanted_lists(ids[part], te[part], temperature, v)[0]
    else:
        targets = _targets(t, v, 0.1, t)
        live = targets != -100
        q = lambda part: _wanted_targets(targets[part], v)[0]
    x[:, ~live] = float("nan")
    x.requires_grad_(True)
    leaf = w.detach().to(w_dtype).requires_grad_(True)
    run = lambda: (linear_distill_loss(x, leaf, ids, te, temperature, reduction) if top else
                   linear_cross_entropy(x, leaf, targets, reduction=reduction))
    loss = run()
    upstream = torch.tensor(up, device="cuda")
    dx, dw = torch.autograd.grad(loss, (x, leaf), upstream, retain_graph=True)
    assert dw.dtype == w_dtype and dx.shape == x.shape
    _check_both(x, w, q, live, temperature, max(1, top), reduction, up, loss, dx, dw)
    dx2, dw2 = torch.autograd.grad(loss, (x, leaf), upstream)
    assert dx2.data_ptr() != dx.data_ptr() and dw2.data_ptr() != dw.data_ptr()
    _check_both(x, w, q, live, temperature, max(1, top), reduction, up, loss, dx2, dw2)
    (dx3,) = torch.autograd.grad(run(), (x,), upstream)
    assert torch.equal(dx3, dx)


@pytest.mark.gpu
def test_linear_both_directions_far_from_the_target():
    """Tokens whose word is too far below the largest logit: as the two directions apart, to the bit, also where a
    captured run is replayed with such tokens and without."""
    t, d, v = 1024, 640, 53000
    print(f"case far {t} {d} {v}", flush=True)
    near, w = _inputs(t, d, v, BF16, 7)
    w.requires_grad_(True)
    targets = _targets(t, v, 0.1, 8)
    far, broken = near.clone(), near.clone()
    far[:, [5, 700]] *= 32
    broken[3, 9] = float("inf")
    targets[[5, 700, 9]] = 11

    def run(x):
        x = x.detach().requires_grad_(True)
        loss = linear_cross_entropy(x, w, targets)
        return (loss.detach(), *torch.autograd.grad(loss, (x, w)))

    def apart(x):
        x = x.detach().requires_grad_(True)
        loss = linear_cross_entropy(x, w, targets)
        torch.autograd.grad(loss, (x, w), retain_graph=True)
        with torch.no_grad():
            forward = linear_cross_entropy(x, w, targets)
        return (forward, *torch.autograd.grad(loss, (x, w)))

    want = {}
    for name, x in (("far", far), ("near", near), ("broken", broken)):
        got, two = run(x), apart(x)
        if name != "near":
            for a, b in zip(got, two):
                assert torch.equal(a.nan_to_num(12345.0), b.nan_to_num(12345.0)), name
        want[name] = got
    q, live = _wanted_targets(targets, v)
    _check_both(far, w.detach(), lambda part: q[part], live, 1.0, 1, "mean", 1.0, *want["far"])
    assert not torch.isfinite(want["broken"][0])

    x = near.clone().requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loss = linear_cross_entropy(x, w, targets)
        torch.autograd.grad(loss, (x, w))
        del loss
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = linear_cross_entropy(x, w, targets)
        dx, dw = torch.autograd.grad(loss, (x, w))
    for name, given in (("near", near), ("far", far), ("near", near), ("broken", broken), ("far", far), ("near", near)):
        with torch.no_grad():
            x.copy_(given)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((loss.detach(), dx, dw), want[name]):
            assert torch.equal(a.nan_to_num(12345.0), b.nan_to_num(12345.0)), name


@pytest.mark.gpu
def test_linear_both_directions_one_block_far():
    """Such a token in the second of two blocks, none in the first."""
    t, d, v = 3000, 640, 212345
    print(f"case one block far {t} {d} {v}", flush=True)
    x, w = _inputs(t, d, v, BF16, 17)
    x[:, 2900] *= 32
    targets = _targets(t, v, 0.1, 18)
    targets[2900] = 7
    x.requires_grad_(True)
    w.requires_grad_(True)
    loss = linear_cross_entropy(x, w, targets)
    dx, dw = torch.autograd.grad(loss, (x, w))
    _check_both(x, w.detach(), lambda part: _wanted_targets(targets[part], v)[0], targets != -100, 1.0, 1, "mean", 1.0, loss, dx, dw)


@pytest.mark.gpu
def test_weight_rows_far_apart():
    t, d, v = 300, 64, 300
    x, w = _inputs(t, d, v, BF16, 1)
    x.requires_grad_(True)
    w.requires_grad_(True)
    targets = _targets(t, v, 0.1, 1)
    a = linear_cross_entropy(x, w, targets)
    wide = torch.empty_strided((v, d), ((1 << 22) + 8, 1), dtype=BF16, device="cuda")
    wide.copy_(w.detach())
    b = linear_cross_entropy(x, w, targets, weight_act=wide)
    assert torch.equal(a, b)
    for one, two in zip(torch.autograd.grad(a, (x, w)), torch.autograd.grad(b, (x, w))):
        assert torch.equal(one, two)


@pytest.mark.gpu
def test_float32_gradients_of_single_words():
    """A weight of 8 on the diagonal: dx is 8 times the logits' gradient, a word each, whose two planes have to agree in
    every one of two million. A logit has one product, held to 2^-24 and 2^-23 of it (its planes, and their products that
    are dropped), a probability the rounding of the logarithm's argument, 2 M U, of the exponential and the sum of 128
    words, and g its planes and the last rounding: (2 (3 |z| + 2 M) + 160) U p, and 4 U |g|. The planes hold 2^15 g,
    the lower one times 2^-11 in steps of 2^-24 at least: half of 2^-50 of g's own unit, however small it is."""
    t, d = 16384, 128
    g = torch.Generator(device="cuda").manual_seed(12)
    x = (0.4 * torch.randn(d, t, generator=g, device="cuda")).requires_grad_(True)
    w = 8.0 * torch.eye(d, device="cuda")
    targets = _targets(t, d, 0.0, 13)
    (dx,) = torch.autograd.grad(linear_cross_entropy(x, w, targets, reduction="sum"), (x,))
    z = 8.0 * x.detach().double().t()
    p = torch.softmax(z, 1)
    want = p - torch.nn.functional.one_hot(targets, d)
    m = z.abs().amax(1, keepdim=True) * np.log2(np.e) + 7
    tol = (2 * (3 * z.abs().amax(1, keepdim=True) + 2 * m) + 160) * U * p + 4 * U * want.abs() + 2.0 ** -51
    _check("dx / 8", dx.t() / 8, want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("x_exp,w_exp,g_exp", [(0, 0, 0), (60, -60, 0), (-70, 66, 5), (100, -104, -20), (-126, 100, 40), (8, 3, -60)])
def test_float32_of_any_size(x_exp, w_exp, g_exp, reduction):
    """Operands far from 1, elements that differ by 2^24 among themselves, upstream gradients of any size."""
    t, d, v = 70, 72, 300
    x, w = _inputs(t, d, v, F32, 3)
    g = torch.Generator(device="cuda").manual_seed(4)
    x *= torch.exp2(-24.0 * torch.rand(d, 1, generator=g, device="cuda"))
    w *= torch.exp2(-24.0 * torch.rand(v, 1, generator=g, device="cuda"))
    x = torch.ldexp(x, torch.tensor(x_exp, device="cuda")).requires_grad_(True)
    w = torch.ldexp(w, torch.tensor(w_exp, device="cuda")).requires_grad_(True)
    targets = _targets(t, v, 0.2, 5)
    q, live = _wanted_targets(targets, v)
    up = torch.full((t,) if reduction == "none" else (), 2.0 ** g_exp, device="cuda")
    loss = linear_cross_entropy(x, w, targets, reduction=reduction)
    dx, dw = torch.autograd.grad(loss, (x, w), up)
    ref, xd, wd = _linear_reference(x, w, q, live, 1.0, 1)
    # (what is 2^-28 of the largest and less keeps 2^-51 of it, g 2^-52)
    floor = 2.0 ** -50 * d * float(xd.abs().max()) * float(wd.abs().max())
    ref.loss_tol += 2 * floor * live
    ref.g_tol += (2 * floor * (ref.g.abs() + q) + 2.0 ** -50) * live[:, None]
    want, tol, scale = ref.reduced(reduction, up.double())
    _check("loss", loss, want, tol)
    gs, gt = ref.g * scale[:, None], ref.g_tol * scale[:, None]
    small = 2.0 ** -149  # (float32's own end)
    wantx = torch.mm(gs, wd).t()
    tol = _product_tol(gt, gs, wd, v).t() + 2.0 ** -50 * float(wd.abs().max()) * gs.abs().sum(1)
    big = wantx.abs() >= torch.finfo(F32).max * (1 + U)  # what float32 does not hold is rounded to inf
    assert torch.equal(dx[big], torch.sign(wantx[big]).float() * torch.inf)
    _check("dx", dx.masked_fill(big, 0), wantx.masked_fill(big, 0), tol + 16 * U * wantx.abs() + small)
    wantw = torch.mm(gs.t(), xd.t())
    tol = _product_tol(gt.t(), gs.t(), xd.t(), t) + 2.0 ** -50 * float(xd.abs().max()) * gs.abs().sum(0)[:, None]
    _check("dw", dw, wantw, tol + 16 * U * wantw.abs() + small)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("held", [1e30, 3e38, float("inf"), float("nan")])
def test_upstream_gradients_of_rows_that_do_not_count(dtype, held):
    """They reach nothing: the gradients are those of upstream zeros there, to the bit."""
    x, w = _inputs(70, 72, 300, dtype, 3)
    targets, (ids, te) = _targets(70, 300, 0.3, 5), _lists(70, 300, 6, seed=4, empty=0.3)
    z = torch.randn(70, 300, device="cuda").to(dtype).requires_grad_(True)
    x.requires_grad_(True)
    w.requires_grad_(True)
    empty = ~((ids >= 0) & (te != -torch.inf)).any(1)
    for run, leaves, off in ((lambda: linear_cross_entropy(x, w, targets, reduction="none"), (x, w), targets == -100),
                             (lambda: linear_distill_loss(x, w, ids, te, temperature=2.0, reduction="none"), (x, w), empty),
                             (lambda: distill_loss(z, ids, te, temperature=2.0, reduction="none"), (z,), empty)):
        assert bool(off.any()) and not bool(off.all())
        up = torch.linspace(-1.0, 2.0, 70, device="cuda")
        want = torch.autograd.grad(run(), leaves, up.masked_fill(off, 0.0))
        got = torch.autograd.grad(run(), leaves, up.masked_fill(off, held))
        assert all(bool(a.isfinite().all()) and torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_linear_weight_copies_and_holder():
    """A float32 master with and without its bfloat16 copy; the gradient through a holder; one gradient only."""
    t, d, v = 100, 64, 300
    x, w = _inputs(t, d, v, F32, 3)
    x = x.to(BF16).requires_grad_(True)
    w.requires_grad_(True)
    act = w.detach().to(BF16)
    targets = _targets(t, v, 0.2, 4)
    q, live = _wanted_targets(targets, v)
    ref, xd, wd = _linear_reference(x, act, q, live, 1.0, 1)
    want, tol, scale = ref.reduced("mean")
    for kw in (dict(), dict(weight_act=act)):
        loss = linear_cross_entropy(x, w, targets, **kw)
        _check("loss", loss, want, tol)
        dx, dw = torch.autograd.grad(loss, (x, w))
        assert dw.dtype == F32
        _check_linear_grads(ref, xd, wd, scale, BF16, F32, dx, dw)
    holder = GradHolder()
    (dx2,) = torch.autograd.grad(linear_cross_entropy(x, w, targets, holder=holder), (x,))
    holder.take()  # (it adds up what it is given)
    loss = linear_cross_entropy(x, w, targets, weight_act=act, holder=holder)
    loss.backward()
    assert w.grad is None and torch.equal(holder.take(), dw) and torch.equal(x.grad, dx)
    (only,) = torch.autograd.grad(linear_cross_entropy(x.detach(), w, targets), (w,))
    assert torch.equal(only, dw) and torch.equal(dx2, dx)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_nothing_counts_and_no_rows(dtype):
    x, w = _inputs(6, 64, 50, dtype, 1)
    z = torch.randn(6, 50, device="cuda").to(dtype)
    none, no_ids = torch.full((6,), -7, device="cuda"), torch.full((6, 4), -1, device="cuda")
    te = torch.full((6, 4), float("nan"), device="cuda")
    x[:, 0], z[0] = float("nan"), -float("inf")
    for a in (x, w, z):
        a.requires_grad_(True)
    calls = [(lambda r: linear_cross_entropy(x, w, none, ignore_index=-7, reduction=r), (x, w)),
             (lambda r: linear_distill_loss(x, w, no_ids, te, reduction=r), (x, w)),
             (lambda r: distill_loss(z, no_ids, te, reduction=r), (z,)),
             (lambda r: linear_cross_entropy(x[:, :0], w, none[:0], reduction=r), (x, w)),
             (lambda r: linear_distill_loss(x, w, no_ids[:, :0], te[:, :0], reduction=r), (x, w)),
             (lambda r: distill_loss(z[:0], no_ids[:0], te[:0], reduction=r), (z,)),
             (lambda r: distill_loss(z, no_ids[:, :0], te[:, :0], reduction=r), (z,))]
    for f, leaves in calls:
        for r in ("none", "sum", "mean"):
            loss = f(r)
            assert loss.dtype == F32 and bool((loss == 0).all())
            for g in torch.autograd.grad(loss.sum(), leaves):
                assert bool((g == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_words_outside_the_vocabulary_are_nan(dtype):
    x, w = _inputs(40, 64, 50, dtype, 1)
    targets = _targets(40, 50, 0.0, 2)
    targets[3], targets[9], targets[11] = 50, -1, 1 << 40
    loss = linear_cross_entropy(x.requires_grad_(True), w, targets, reduction="none")
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[[3, 9, 11]] = True
    assert torch.equal(loss.isnan(), bad)
    (dx,) = torch.autograd.grad(loss, (x,), torch.ones_like(loss))
    assert torch.equal(dx.isnan().all(0), bad) and torch.equal(dx.isnan().any(0), bad)
    ids, te = _lists(40, 50, 4, seed=3, empty=0.0)
    ids[:, 0], te[:, 0] = 7, 1.0
    ids[3, 0], te[9, 0], te[11, 0] = 50, float("nan"), float("inf")
    z = torch.randn(40, 50, device="cuda").to(dtype).requires_grad_(True)
    for loss, leaf, rows in ((linear_distill_loss(x, w, ids, te, reduction="none"), x, 0),
                             (distill_loss(z, ids, te, reduction="none"), z, 1)):
        assert torch.equal(loss.isnan(), bad)
        (g,) = torch.autograd.grad(loss, (leaf,), torch.ones_like(loss))
        assert torch.equal(g.isnan().all(rows), bad) and torch.equal(g.isnan().any(rows), bad)


# ------------------------------------------------------------------------------- from logits
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("t,v,top,temperature,reduction,tdtype", [
    (1, 1, 1, 1.0, "mean", F32), (7, 2, 2, 2.0, "none", F32), (5, 100, 7, 0.7, "sum", BF16), (9, 4096, 64, 2.0, "mean", F32),
    (6, 4097, 65, 1.0, "none", F32), (4, 16384, 100, 2.0, "sum", F32), (3, 16385, 129, 1.0, "mean", BF16),
    (3, 50280, 32, 2.0, "mean", F32), (2, 65536, 256, 1.0, "none", F32), (2, 65537, 300, 2.0, "mean", F32),
    (2, 131071, 20, 1.0, "sum", F32), (37, 999, 1000, 1.0, "mean", F32)])
def test_distill_loss(dtype, t, v, top, temperature, reduction, tdtype):
    print(f"case distill_loss {dtype} {t} {v} {top} {temperature} {reduction}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(t + v)
    big = (2.5 * torch.randn(t, v + 3, generator=g, device="cuda")).to(dtype)
    z = big[:, 2:2 + v]  # rows off 16 bytes, with gaps
    ids, te = _lists(t, v, top, tdtype, t + 1)
    q, live = _wanted_lists(ids, te, temperature, v)
    # Words of no weight, and rows that do not count, hold anything; a wanted word stays as it is.
    gone = (torch.rand(t, v, generator=g, device="cuda") < 0.2) & (q == 0)
    gone[:, 0] = False
    z[gone] = torch.finfo(dtype).min
    z[gone & (torch.rand(t, v, generator=g, device="cuda") < 0.5)] = -float("inf")
    z[~live] = float("nan")
    z.requires_grad_(True)
    up = torch.linspace(-1.0, 2.0, t, device="cuda") if reduction == "none" else torch.tensor(0.3, device="cuda")
    loss = distill_loss(z, ids, te, temperature=temperature, reduction=reduction)
    zd = torch.where(live[:, None], z.detach().double(), 0.0)
    zd = torch.where(zd == torch.finfo(dtype).min, -torch.inf, zd)  # (their weight is 0 in float64 too)
    ref = _Bounds(zd, torch.zeros(t, dtype=torch.float64, device="cuda"), q, live, temperature, top, dtype)
    want, tol, scale = ref.reduced(reduction, up.double())
    _check("loss", loss, want, tol)
    (dz,) = torch.autograd.grad(loss, (z,), up, retain_graph=True)
    assert dz.dtype == dtype
    gw = ref.g * scale[:, None]
    _check("dz", dz, gw, ref.g_tol * scale[:, None].abs() + 8 * U * gw.abs() + 2.0 ** -149)
    (one,) = torch.autograd.grad(loss, (z,), torch.ones_like(up), retain_graph=True)  # another pass, another upstream
    want, tol, scale = ref.reduced(reduction)
    gw = ref.g * scale[:, None]
    _check("dz at 1", one, gw, ref.g_tol * scale[:, None].abs() + 8 * U * gw.abs() + 2.0 ** -149)
    first = distill_loss(z, ids, te, temperature=temperature, reduction=reduction)  # and the one-reading pass with an upstream of 1
    (again,) = torch.autograd.grad(first, (z,), torch.ones_like(up))
    assert torch.equal(again, one)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_distill_edges_of_the_types(dtype):
    """All words at the type's lowest value are alike; a wanted word of no weight makes the loss inf, its gradient
    stays finite; a row without any word, and one with a NaN, are NaN."""
    lowest = torch.finfo(dtype).min
    z = torch.zeros(4, 70, device="cuda", dtype=dtype)
    z[0], z[1, 5], z[2], z[3, 9] = lowest, -float("inf"), -float("inf"), float("nan")
    ids = torch.tensor([[3], [5], [1], [2]], device="cuda")
    te = torch.zeros(4, 1, device="cuda")
    z.requires_grad_(True)
    loss = distill_loss(z, ids, te, reduction="none")
    (g,) = torch.autograd.grad(loss, (z,), torch.ones_like(loss))
    # log2 70, its product with ln 2 and the exponent: a few steps of 8
    loss = loss.detach()
    assert abs(float(loss[0]) - np.log(70)) <= 32 * U * np.log(70) + 70 * 2 * U
    assert float(loss[1]) == float("inf") and bool(loss[2:].isnan().all())
    want = torch.full((70,), 1 / 70, dtype=torch.float64, device="cuda")
    want[3] -= 1
    _check("lowest", g[0], want, (HALF[dtype] + 200 * U) * want.abs())
    want = torch.full((70,), 1 / 69, dtype=torch.float64, device="cuda")
    want[5] = -1
    _check("absent", g[1], want, (HALF[dtype] + 200 * U) * want.abs())
    assert bool(g[2].isnan().all()) and bool(g[3].isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("v", [3000, 70001, 131072])
@pytest.mark.parametrize("reduction", ["none", "sum"])
def test_distill_a_nan_anywhere_makes_its_row_nan(dtype, v, reduction):
    """Also where what a lane has read before it is words of no weight, and where it reads nothing else."""
    inf = float("inf")
    g = torch.Generator(device="cuda").manual_seed(v)
    z = torch.randn(9, v, generator=g, device="cuda").to(dtype)
    z[0, :16] = float("nan")         # a whole vector, the first of its lane
    z[1, :16], z[1, 3] = -inf, float("nan")
    z[2], z[2, 5], z[2, 100] = -inf, 1.0, float("nan")
    z[3] = float("nan")
    z[4], z[4, v - 1] = -inf, float("nan")
    z[5, v - 1] = float("nan")
    z[6, :2000] = -inf               # and none in these
    z[7] = -inf
    z[7, 5] = 2.0
    z.requires_grad_(True)
    ids = torch.full((9, 1), 5, device="cuda")
    z.data[6, 5] = 1.0
    loss = distill_loss(z, ids, torch.zeros(9, 1, device="cuda"), reduction="none")
    bad = torch.tensor([True] * 6 + [False] * 3, device="cuda")
    assert torch.equal(loss.isnan(), bad) and bool(loss[6:].isfinite().all()) and float(loss[7].detach()) == 0.0
    if reduction == "sum":
        loss = distill_loss(z, ids, torch.zeros(9, 1, device="cuda"), reduction="sum")
        assert bool(loss.isnan())
    (d,) = torch.autograd.grad(loss, (z,), torch.ones_like(loss))
    assert torch.equal(d.isnan().all(1), bad) and torch.equal(d.isnan().any(1), bad)


# ------------------------------------------------------------------------------- both
@pytest.mark.gpu
def test_gradients_against_differences():
    """Central differences along a direction: the loss's own bound over the step, and the step's square times the third
    derivative / 6: the sum of the rows' third central moments of the directional logits over temperature, of which
    each is at most its cubed range / (6 sqrt 3), that of two points' distribution."""
    t, d, v, h = 24, 64, 90, 0.01
    x, w = _inputs(t, d, v, F32, 8)
    ids, te = _lists(t, v, 6, seed=9)
    targets = _targets(t, v, 0.2, 10)
    g = torch.Generator(device="cuda").manual_seed(2)
    along = torch.randn(d, t, generator=g, device="cuda") / d ** 0.5
    for f, temperature, (q, live) in ((lambda a: linear_cross_entropy(a, w, targets, reduction="sum"), 1.0, _wanted_targets(targets, v)),
                                      (lambda a: linear_distill_loss(a, w, ids, te, temperature=2.0, reduction="sum"), 2.0,
                                       _wanted_lists(ids, te, 2.0, v)),
                                      (lambda a: distill_loss(a.t() @ w.t(), ids, te, temperature=2.0, reduction="sum"), 2.0,
                                       _wanted_lists(ids, te, 2.0, v))):
        a = x.clone().requires_grad_(True)
        (dx,) = torch.autograd.grad(f(a), (a,))
        slope = float((dx.double() * along.double()).sum())
        ends = [float(f(x + s * h * along)) for s in (1, -1)]
        ref, xd, wd = _linear_reference(x, w, q, live, temperature, 6)
        dz = torch.mm(along.double().t(), wd.t())
        span = (dz.amax(1) - dz.amin(1))[live] / temperature
        tol = 2 * float(ref.loss_tol.sum()) / (2 * h) + h * h / 6 * temperature ** 2 * float((span ** 3).sum()) / (6 * 3 ** 0.5)
        # (x + h along is rounded to float32: its error moves the loss by the gradient's share of it)
        tol += U * float((dx.abs().double() * (x.abs().double() + h * along.abs().double())).sum()) * 2 / h
        tol += 2 * U * (abs(ends[0]) + abs(ends[1])) / h + 1e-3 * U
        print(f"  slope {slope:.6f} differences {(ends[0] - ends[1]) / (2 * h):.6f} tolerance {tol:.2e}", flush=True)
        assert abs(slope - (ends[0] - ends[1]) / (2 * h)) <= tol


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_runs_are_the_same_and_streams(dtype):
    x, w = _inputs(300, 128, 700, dtype, 3)
    ids, te = _lists(300, 700, 20, seed=4)
    targets = _targets(300, 700, 0.1, 5)
    z = torch.randn(300, 700, device="cuda").to(dtype)
    for a in (x, w, z):
        a.requires_grad_(True)

    def run():
        out = []
        for loss, leaves in ((linear_cross_entropy(x, w, targets), (x, w)), (linear_distill_loss(x, w, ids, te), (x, w)),
                             (distill_loss(z, ids, te), (z,))):
            out += [loss.detach(), *torch.autograd.grad(loss, leaves)]
        return out

    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b, c in zip(first, second, run()):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_graph_replays(dtype):
    """Each replay, on new values of the inputs, against the eager calls; two graphs side by side."""
    t, d, v = 90, 64, 400
    x, w = _inputs(t, d, v, dtype, 3)
    z = torch.randn(t, v, device="cuda").to(dtype)
    ids, te = _lists(t, v, 6, seed=4)
    targets = _targets(t, v, 0.1, 5)
    for a in (x, w, z):
        a.requires_grad_(True)

    def linear():
        loss = linear_cross_entropy(x, w, targets) + 0.5 * linear_distill_loss(x, w, ids, te, temperature=2.0)
        return [loss.detach(), *torch.autograd.grad(loss, (x, w))]

    def logits():
        loss = 2.0 * distill_loss(z, ids, te)
        return [loss.detach(), *torch.autograd.grad(loss, (z,))]

    graphs = []
    for f in (linear, logits):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            f()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = f()
        graphs.append((g, out, f))
    for i in range(4):
        with torch.no_grad():
            x.mul_(0.9)
            w.add_(0.01)
            z.mul_(1.1)
            targets.copy_(torch.roll(targets, 1))
            te.copy_(te.roll(1, 0))
            ids.copy_(ids.roll(1, 0))
        want = [f() for _, _, f in graphs]
        torch.cuda.synchronize()
        for (g, out, _), wanted in zip(graphs, want):
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, wanted)), i


@pytest.mark.gpu
def test_against_the_framework_s_cross_entropy():
    """The two forms of the same loss: from logits rounded to bfloat16 (each off by 2^-8 of itself), and without."""
    t, d, v = 500, 128, 1000
    x, w = _inputs(t, d, v, BF16, 3)
    targets = _targets(t, v, 0.0, 5)
    z = (x.t().contiguous() @ w.t())
    apart = 2 * 2.0 ** -8 * float(z.abs().max()) * 1.1
    assert abs(float(cross_entropy(z, targets)) - float(linear_cross_entropy(x, w, targets))) <= apart


@pytest.mark.gpu
def test_second_backward_and_input_changes():
    x, w = _inputs(50, 64, 90, BF16, 3)
    z = torch.randn(50, 90, device="cuda", requires_grad=True)
    ids, te = _lists(50, 90, 5, seed=1)
    targets = _targets(50, 90, 0.1, 5)
    x.requires_grad_(True)
    w.requires_grad_(True)
    for loss, leaf in ((linear_cross_entropy(x, w, targets), x), (distill_loss(z, ids, te), z)):
        (a,) = torch.autograd.grad(loss, (leaf,), retain_graph=True)
        keep = a.clone()
        a.zero_()
        (b,) = torch.autograd.grad(loss, (leaf,), retain_graph=True)
        assert torch.equal(keep, b)
    # the loss may be written over: nothing of it is read again
    loss = linear_cross_entropy(x, w, targets)
    (a,) = torch.autograd.grad(loss, (x,), retain_graph=True)
    loss.detach().mul_(0.0)
    assert torch.equal(a, torch.autograd.grad(loss, (x,))[0])
    # what the backward pass reads again is watched
    loss = linear_cross_entropy(x, w, targets)
    with torch.no_grad():
        w.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(loss, (x,))


def _saved_elsewhere(run, way):
    """run() with what it saves put elsewhere until the backward pass, and what it had before written over."""
    if way == "checkpoint":
        from torch.utils.checkpoint import checkpoint
        return checkpoint(run, use_reentrant=False)
    with (torch.autograd.graph.save_on_cpu() if way == "cpu" else _Hooks()):
        loss = run()
    torch.cuda.synchronize()
    full = [torch.full((n,), 0x7f, dtype=torch.uint8, device="cuda") for n in (1 << 12, 1 << 16, 1 << 19, 1 << 20, 1 << 22, 1 << 24) for _ in range(8)]
    del full
    return loss


@pytest.mark.gpu
@pytest.mark.parametrize("way", ["clone", "cpu", "checkpoint"])
@pytest.mark.parametrize("dtype,d,layout,reduction", [(BF16, 64, "cm", "none"), (BF16, 64, "gap", "mean"), (F32, 40, "cm", "sum")])
def test_linear_saved_elsewhere(dtype, d, layout, reduction, way):
    x, w = _inputs(90, d, 400, dtype, 3, layout)
    targets, (ids, te) = _targets(90, 400, 0.1, 5), _lists(90, 400, 6, seed=4)
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    up = torch.linspace(-1.0, 2.0, 90, device="cuda") if reduction == "none" else torch.tensor(0.7, device="cuda")
    for run in (lambda: linear_cross_entropy(x, w, targets, reduction=reduction),
                lambda: linear_distill_loss(x, w, ids, te, temperature=2.0, reduction=reduction)):
        want = torch.autograd.grad(run(), (x, w), up)
        got = torch.autograd.grad(_saved_elsewhere(run, way), (x, w), up)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("way", ["clone", "cpu"])
def test_linear_both_directions_saved_elsewhere(way):
    """A head whose gradients come with its loss: the first pass has them, the second one makes its own."""
    x, w = _inputs(1024, 640, 33000, BF16, 3)
    targets = _targets(1024, 33000, 0.1, 5)
    x.requires_grad_(True)
    w.requires_grad_(True)
    run = lambda: linear_cross_entropy(x, w, targets)

    def passes(loss):
        return [torch.autograd.grad(loss, (x, w), retain_graph=keep) for keep in (True, False)]
    for got, want in zip(passes(_saved_elsewhere(run, way)), passes(run())):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("way", ["clone", "cpu", "checkpoint"])
@pytest.mark.parametrize("dtype,reduction", [(BF16, "none"), (BF16, "mean"), (F32, "sum")])
def test_distill_saved_elsewhere(dtype, reduction, way):
    big = torch.randn(90, 405, device="cuda").to(dtype)
    z = big[:, 2:402].detach().requires_grad_(True)  # rows off 16 bytes, with gaps
    ids, te = _lists(90, 400, 6, seed=4)
    up = torch.linspace(-1.0, 2.0, 90, device="cuda") if reduction == "none" else torch.tensor(0.7, device="cuda")
    run = lambda: distill_loss(z, ids, te, temperature=2.0, reduction=reduction)

    def passes(loss):
        return [torch.autograd.grad(loss, (z,), up, retain_graph=keep)[0] for keep in ((True, False) if way != "checkpoint" else (False,))]
    for got, want in zip(passes(_saved_elsewhere(run, way)), passes(run())):
        assert torch.equal(got, want)
