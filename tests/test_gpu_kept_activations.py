"""Activations kept in 8 bits (`checkpoint_activation`, `restore_activation`) and the gated SiLU that keeps its input so
(`silu_gate`, `silu_gate_checkpoint`, `silu_gate_backward`).

What is kept is compared bit for bit.  The activation and its gradient are compared with 64 bits: one rounding of half a step of
the result's type, and in front of it fp32 with a sigmoid of 1e-5 (16-bit types: `__expf` is within 2 + 1.173 |g| ulp, |g| < 40) or
2e-6 (fp32: expf within 2 ulp, a division, five products)."""
from __future__ import annotations

import pytest
import torch

from conftest import gpu_ready
from taac_2026_b200 import ops

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
SHAPES = [(1, 128), (3, 384), (77, 640), (500, 2048), (13, 8192), (20000, 128)]


@pytest.fixture(autouse=True)
def _need_gpu():
    if not gpu_ready():
        pytest.fail("gpu tests need an sm_100 device and a built libtb200.so")


def _data(rows, cols, dtype, seed, scale=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(rows, cols, generator=g, device="cuda") * scale).to(dtype)


def _kept(x):
    """The definition, on the host: smallest power of two with max / s <= 448 over the finite values, NaN for the others."""
    blocks = x.cpu().double().view(x.shape[0], -1, 128)
    finite = blocks.isfinite()
    amax = torch.where(finite, blocks.abs(), 0.0).amax(-1)
    mantissa, exponent = torch.frexp(amax)
    e = (exponent - 9 + (mantissa > 0.875).int()).clamp(-126, 126)
    s = torch.where(amax > 0, torch.exp2(e.double()), 1.0)
    q = torch.where(finite, blocks / s[..., None], float("nan")).float().to(torch.float8_e4m3fn)
    return q.view(x.shape), s.float()


def _same(q, want):
    a, b = q.cpu().view(torch.uint8), want.view(torch.uint8)
    nan = (b & 0x7F) == 0x7F
    assert torch.equal(a[~nan], b[~nan]) and bool(((a[nan] & 0x7F) == 0x7F).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_keep_and_restore(dtype, rows, cols):
    x = _data(rows, cols, dtype, rows + cols)
    x[0, 0], x[-1, -1] = 448.0, -7.0                     # on the border between two powers of two
    q, s = ops.checkpoint_activation(x)
    want_q, want_s = _kept(x)
    assert torch.equal(s.cpu(), want_s)
    _same(q, want_q)
    exact = want_q.double() * want_s.double().repeat_interleave(128, 1)
    for out in (torch.float32, torch.bfloat16):
        back = ops.restore_activation(q, s, out)
        assert back.dtype == out and torch.equal(back.double().cpu(), exact)
    if dtype == torch.float16:
        assert torch.equal(ops.restore_activation(q, s, torch.float16).cpu(), exact.half())


def test_values_at_the_ends_of_the_range():
    x = torch.zeros(6, 128, device="cuda")
    x[1, 3] = 1e-42                                       # subnormal: the scale stops at 2^-126
    x[2, 0], x[2, 1] = 3.4e38, 1.0
    x[3, 0], x[3, 1], x[3, 2] = float("inf"), 2.0, float("nan")
    x[4] = float("-inf")
    x[5, 127] = 2.0 ** -126
    q, s = ops.checkpoint_activation(x)
    want_q, want_s = _kept(x)
    assert torch.equal(s.cpu(), want_s)
    _same(q, want_q)
    back = ops.restore_activation(q, s, torch.float32)
    assert bool(back[3, [0, 2]].isnan().all()) and float(back[3, 1]) == 2.0 and bool(back[4].isnan().all())


def _act(u, gated, gate_first):
    if not gated:
        return u, torch.ones_like(u)
    a, b = u.chunk(2, -1)
    return (a, b) if gate_first else (b, a)


def _within(got, want, tol):
    assert got.shape == want.shape
    off = (got.double() - want).abs() - tol
    assert bool((off <= 0).all()), float(off.max())


def _tol(dtype):
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    return torch.finfo(dtype).eps / 2, (2e-6 if dtype == torch.float32 else 1e-5), tiny


FORMS = [(True, True), (True, False), (False, True)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,hidden", SHAPES)
@pytest.mark.parametrize("gated,gate_first", FORMS)
def test_gate_and_its_backward(dtype, rows, hidden, gated, gate_first):
    up = _data(rows, hidden * (2 if gated else 1), dtype, rows * 3 + hidden, 4.0)
    dh = _data(rows, hidden, dtype, rows * 5 + hidden, 1.0)
    half, soft, tiny = _tol(dtype)
    g, v = _act(up.double(), gated, gate_first)
    want = g * torch.sigmoid(g) * v
    h, q, s = ops.silu_gate_checkpoint(up, gated=gated, gate_first=gate_first)
    _within(h, want, (half + soft) * want.abs() + tiny)
    assert torch.equal(h, ops.silu_gate(up, gated=gated, gate_first=gate_first))
    q1, s1 = ops.checkpoint_activation(up)
    assert torch.equal(q.view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s, s1)

    dup, again = ops.silu_gate_backward(q, s, dh, gated=gated, gate_first=gate_first)
    kept = q.double() * s.double().repeat_interleave(128, 1)
    g, v = _act(kept, gated, gate_first)
    sig = torch.sigmoid(g)
    want_h = g * sig * v
    dg, size = dh.double() * v * sig * (1 + g * (1 - sig)), (dh.double() * v).abs() * sig * (1 + g.abs() * (1 - sig))
    _within(again, want_h, (half + soft) * want_h.abs() + tiny)
    got_g, got_v = _act(dup, gated, gate_first)
    # g (1 - sig) keeps the absolute error of sig: |g| 2^-23 of sig
    _within(got_g, dg, half * dg.abs() + (soft + 2.0 ** -23 * g.abs()) * size.clamp_min(0) + 2.0 ** -23 * (dh.double() * v * sig * g).abs() + tiny)
    if gated:
        dv = dh.double() * g * sig
        _within(got_v, dv, (half + soft) * dv.abs() + tiny)
    only, none = ops.silu_gate_backward(q, s, dh, gated=gated, gate_first=gate_first, activation=False)
    assert none is None and torch.equal(only, dup)


def test_gradient_against_differences():
    """Inputs that 8 bits hold exactly (multiples of 1/8 up to 1 + 7/8, blocks that reach it): the kept values are the inputs."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    up = torch.randint(-15, 16, (8, 512), generator=gen, device="cuda").float() / 8
    up[:, ::128] = 1.75
    dh = torch.randn(8, 256, generator=gen, device="cuda")
    x = up.clone().requires_grad_()
    grad, = torch.autograd.grad((ops.silu_gate(x).double() * dh).sum(), x)
    step = 2.0 ** -7
    for at in [(0, 0), (3, 17), (7, 300), (5, 511)]:
        ends = []
        for sign in (1, -1):
            moved = up.clone()
            moved[at] += sign * step
            ends.append(float((ops.silu_gate(moved).double() * dh).sum()))
        slope = (ends[0] - ends[1]) / (2 * step)
        # third order: h^2 / 6 times a third derivative below 2 |dh v|, and the fp32 values' own roundings over 2 h
        assert abs(slope - float(grad[at])) <= 1e-3 * (1 + abs(slope))


def test_large_and_special_inputs():
    up = torch.tensor([[-200.0, 200.0, -90.0, 0.0] * 32], device="cuda", dtype=torch.bfloat16)
    h, q, s = ops.silu_gate_checkpoint(up, gated=False)
    assert bool(h.isfinite().all()) and float(h[0, 1]) == 200.0 and float(h[0, 0]) == 0.0
    dup, again = ops.silu_gate_backward(q, s, torch.ones_like(up), gated=False)
    assert bool(dup.isfinite().all()) and float(dup[0, 1]) == 1.0 and float(dup[0, 0]) == 0.0 and float(dup[0, 3]) == 0.5
    up[0, 5] = float("nan")
    _h, q, s = ops.silu_gate_checkpoint(up, gated=False)
    dup, _again = ops.silu_gate_backward(q, s, torch.ones_like(up), gated=False)
    assert bool(dup[0, 5].isnan()) and int(dup.isnan().sum()) == 1


def test_views_graph_and_empty():
    up = _data(40, 512, torch.bfloat16, 8)
    want = ops.silu_gate_checkpoint(up)
    pad = torch.zeros(40, 520, device="cuda", dtype=torch.bfloat16)
    pad[:, 3:515] = up
    got = ops.silu_gate_checkpoint(pad[:, 3:515].view(4, 10, 512) if pad[:, 3:515].is_contiguous() else pad[:, 3:515])
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, q, s = ops.silu_gate_checkpoint(up)
        dup, again = ops.silu_gate_backward(q, s, h)
    up.copy_(_data(40, 512, torch.bfloat16, 9))
    graph.replay()
    h2, q2, s2 = ops.silu_gate_checkpoint(up)
    assert torch.equal(h, h2) and torch.equal(dup, ops.silu_gate_backward(q2, s2, h2)[0])
    empty = torch.zeros(0, 256, device="cuda", dtype=torch.bfloat16)
    h, q, s = ops.silu_gate_checkpoint(empty)
    assert h.shape == (0, 128) and ops.silu_gate_backward(q, s, h)[0].shape == (0, 256)
    assert ops.restore_activation(*ops.checkpoint_activation(empty)).shape == (0, 256)


def test_refusals():
    up = _data(4, 512, torch.bfloat16, 1)
    _h, q, s = ops.silu_gate_checkpoint(up)
    with pytest.raises(RuntimeError, match="forward-only"):
        ops.silu_gate_checkpoint(up.clone().requires_grad_())
    with pytest.raises(ValueError, match="multiple of 256"):
        ops.silu_gate(up[:, :384].contiguous())
    with pytest.raises(ValueError, match="scales must be"):
        ops.silu_gate_backward(q, s[:, :2], up[:, :256])
    with pytest.raises(ValueError, match="grad must be"):
        ops.silu_gate_backward(q, s, up)
    with pytest.raises(ValueError, match="e4m3"):
        ops.restore_activation(up, s)
    with pytest.raises(RuntimeError, match="does not support dtype"):
        ops.silu_gate(up.double())
