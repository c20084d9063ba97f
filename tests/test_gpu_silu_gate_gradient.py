"""`silu_gate` under autograd: the gradient at the input itself, and with `checkpoint=True` at what 8 bits keep of it.

Tolerances as in test_gpu_kept_activations.py: one rounding of half a step of the result's type, and in front of it fp32 with a sigmoid of
1e-5 (16-bit types) or 2e-6 (fp32); g (1 - sig) keeps the absolute error of sig."""
from __future__ import annotations

import pytest
import torch

from conftest import gpu_ready
from taac_2026_b200 import ops

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
FORMS = [(True, True), (True, False), (False, True)]


@pytest.fixture(autouse=True)
def _need_gpu():
    if not gpu_ready():
        pytest.fail("gpu tests need an sm_100 device and a built libtb200.so")


def _data(*shape, dtype, seed, scale):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _halves(u, gated, gate_first):
    if not gated:
        return u, torch.ones_like(u)
    a, b = u.chunk(2, -1)
    return (a, b) if gate_first else (b, a)


def _within(got, want, tol):
    assert got.shape == want.shape
    off = (got.double() - want).abs() - tol
    assert bool((off <= 0).all()), float(off.max())


def _check(dup, h, up, dh, gated, gate_first):
    dtype = dup.dtype
    half, soft = torch.finfo(dtype).eps / 2, 2e-6 if dtype == torch.float32 else 1e-5
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    g, v = _halves(up.double(), gated, gate_first)
    sig, d = torch.sigmoid(g), dh.double()
    want_h = g * sig * v
    if h is not None:
        _within(h, want_h, (half + soft) * want_h.abs() + tiny)
    dg, size = d * v * sig * (1 + g * (1 - sig)), (d * v).abs() * sig * (1 + g.abs() * (1 - sig))
    got_g, got_v = _halves(dup, gated, gate_first)
    _within(got_g, dg, half * dg.abs() + (soft + 2.0 ** -23 * g.abs()) * size + 2.0 ** -23 * (d * v * sig * g).abs() + tiny)
    if gated:
        dv = d * g * sig
        _within(got_v, dv, (half + soft) * dv.abs() + tiny)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 128), (77, 640), (4, 10, 256), (500, 2048), (20000, 128)])
@pytest.mark.parametrize("gated,gate_first", FORMS)
def test_gradient_at_the_input_itself(dtype, shape, gated, gate_first):
    up = _data(*shape[:-1], shape[-1] * (2 if gated else 1), dtype=dtype, seed=sum(shape), scale=4.0)
    dh = _data(*shape, dtype=dtype, seed=1, scale=1.0)
    leaf = up.clone().requires_grad_()
    h = ops.silu_gate(leaf, gated=gated, gate_first=gate_first)
    assert torch.equal(h.detach(), ops.silu_gate(up, gated=gated, gate_first=gate_first))
    h.backward(dh)
    _check(leaf.grad, h.detach(), up, dh, gated, gate_first)
    dup, again = ops.silu_gate_backward(up, None, dh, gated=gated, gate_first=gate_first)
    assert torch.equal(dup, leaf.grad) and torch.equal(again, h.detach())
    assert ops.silu_gate_backward(up, None, dh, gated=gated, gate_first=gate_first, activation=False)[1] is None
    kept = up.clone().requires_grad_()
    ops.silu_gate(kept, gated=gated, gate_first=gate_first, checkpoint=True).backward(dh)
    _h, q, s = ops.silu_gate_checkpoint(up, gated=gated, gate_first=gate_first)
    assert torch.equal(kept.grad, ops.silu_gate_backward(q, s, dh, gated=gated, gate_first=gate_first, activation=False)[0])


def test_gradient_against_differences():
    """fp32, inputs that 8 bits do not hold.  Third order: h^2 / 6 times a third derivative below 2 |dh v|, and the values' own
    roundings over 2 h."""
    up, dh = _data(8, 512, dtype=torch.float32, seed=2, scale=1.0), _data(8, 256, dtype=torch.float32, seed=3, scale=1.0)
    leaf = up.clone().requires_grad_()
    grad, = torch.autograd.grad((ops.silu_gate(leaf).double() * dh).sum(), leaf)
    step = 2.0 ** -7
    for at in [(0, 0), (3, 17), (7, 300), (5, 511)]:
        ends = []
        for sign in (1, -1):
            moved = up.clone()
            moved[at] += sign * step
            ends.append((float((ops.silu_gate(moved).double() * dh).sum()), float(moved[at].double())))
        slope = (ends[0][0] - ends[1][0]) / (ends[0][1] - ends[1][1])
        assert abs(slope - float(grad[at])) <= 1e-3 * (1 + abs(slope))


def test_views_graph_and_other_paths(monkeypatch):
    up, dh = _data(40, 512, dtype=torch.bfloat16, seed=4, scale=2.0), _data(40, 256, dtype=torch.bfloat16, seed=5, scale=1.0)
    want = ops.silu_gate_backward(up, None, dh)
    pad = torch.zeros(40, 520, device="cuda", dtype=torch.bfloat16)
    pad[:, 3:515] = up
    got = ops.silu_gate_backward(pad[:, 3:515], None, dh.t().contiguous().t())
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    sink = []
    ops.set_kernel_timing(sink)
    try:
        got = ops.silu_gate_backward(up, None, dh)
    finally:
        ops.set_kernel_timing(None)
    assert sink and all(torch.equal(a, b) for a, b in zip(want, got))
    with monkeypatch.context() as m:
        m.setattr(ops, "_host", ops._NoHost())
        got = ops.silu_gate_backward(up, None, dh)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = ops.silu_gate_backward(up, None, dh)
    up.mul_(0.5)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(captured, ops.silu_gate_backward(up, None, dh)))
    empty = up[:0]
    dup, h = ops.silu_gate_backward(empty, None, dh[:0])
    assert dup.shape == (0, 512) and h.shape == (0, 256)


def test_refusals():
    up, dh = _data(4, 512, dtype=torch.bfloat16, seed=6, scale=1.0), _data(4, 256, dtype=torch.bfloat16, seed=7, scale=1.0)
    with pytest.raises(ValueError, match="one dtype"):
        ops.silu_gate_backward(up, None, dh.float())
    with pytest.raises(ValueError, match="grad must be"):
        ops.silu_gate_backward(up, None, up)
    with pytest.raises(ValueError, match="multiple of 256"):
        ops.silu_gate_backward(up[:, :384].contiguous(), None, dh)
    with pytest.raises(RuntimeError, match="does not support dtype"):
        ops.silu_gate_backward(up.double(), None, dh.double())


@pytest.mark.parametrize("checkpoint", [False, True])
def test_between_layers_of_experts(checkpoint):
    """Up projections, activation, down projections: autograd's gradients are those of the calls one by one."""
    off = torch.tensor([0, 40, 40, 90], dtype=torch.int32, device="cuda")
    x, dy = (_data(90, 256, dtype=torch.bfloat16, seed=s, scale=1.0) for s in (8, 9))
    w_up, w_down = _data(3, 768, 256, dtype=torch.bfloat16, seed=10, scale=1 / 16), _data(3, 256, 384, dtype=torch.bfloat16, seed=11, scale=1 / 16)
    leaves = [t.clone().requires_grad_() for t in (x, w_up, w_down)]
    u = ops.ragged_linear(leaves[0], leaves[1], off, checkpoint=checkpoint)
    ops.ragged_linear(ops.silu_gate(u, checkpoint=checkpoint), leaves[2], off, checkpoint=checkpoint).backward(dy)
    u = ops.ragged_linear(x, w_up, off)
    h, q, s = ops.silu_gate_checkpoint(u)
    keep = (lambda t: ops.restore_activation(*ops.checkpoint_activation(t))) if checkpoint else (lambda t: t)
    dh, dw_down, _b = ops.ragged_linear_backward(keep(h), w_down, off, dy)
    du = ops.silu_gate_backward(*((q, s) if checkpoint else (u, None)), dh)[0]
    dx, dw_up, _b = ops.ragged_linear_backward(keep(x), w_up, off, du)
    assert all(torch.equal(leaf.grad, want) for leaf, want in zip(leaves, (dx, dw_up, dw_down)))
