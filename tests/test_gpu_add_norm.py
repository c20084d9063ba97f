"""Residual addition + RMSNorm (`add_rms_norm`, `add_rms_norm_quant`, `add_rms_norm_backward`) against the formulas in 64 bits.

Tolerances.  u = eps / 2 of the result's type is the one rounding of each stored value.  What comes before it is fp32: the sum
of squares adds at most 32 values in a lane and then 5 shuffles and 16 warps (53 roundings of 2^-24, halved by the root), rsqrtf is
within 2 ulp (2^-22), and the products add five more: below 40 * 2^-24 in all, relative."""
from __future__ import annotations

import pytest
import torch

from conftest import gpu_ready
from taac_2026_b200 import ops

pytestmark = pytest.mark.gpu

F32 = 40 * 2.0 ** -24
SHAPES = [(1, 128), (3, 128), (77, 256), (1, 512), (300, 512), (65, 640), (129, 1024), (7, 1152), (33, 2048), (20, 2560), (5, 4096), (3, 8192),
          (2, 16384), (5000, 128), (3001, 512)]
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(autouse=True)
def _need_gpu():
    if not gpu_ready():
        pytest.fail("gpu tests need an sm_100 device and a built libtb200.so")


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2      # half a subnormal step


def _inputs(rows, cols, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, r = make(rows, cols), 2 * make(rows, cols)
    x[rows // 2] *= 50
    return x.to(dtype), r.to(dtype), (1 + 0.1 * make(cols)).to(dtype), make(rows, cols).to(dtype), make(rows, cols).to(dtype)


def _formula(x, r, w, eps=1e-6):
    t = x.double() + (0 if r is None else r.double())
    s = torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + eps)
    return t, s, t * s * w.double()


def _within(got, want, tol):
    assert got.shape == want.shape
    off = (got.double() - want).abs() - tol
    assert bool((off <= 0).all()), float(off.max())


def _check_quant(n, q, scale):
    """q * scale against n: half an e4m3 step (2^-4 relative, 2^-10 scales among the subnormals); the largest value uses the range."""
    value = q.double() * scale.repeat_interleave(128, -1).double()
    wide = scale.repeat_interleave(128, -1).double()
    _within(value, n, torch.maximum(2.0 ** -4 * n.abs(), 2.0 ** -10 * wide) * (1 + 1e-5))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES + [(9, 8), (40, 24), (6, 1032), (4, 3000)])
def test_add_rms_norm(dtype, rows, cols):
    x, r, w, _a, _b = _inputs(rows, cols, dtype, rows + cols)
    total, normed = ops.add_rms_norm(x, r, w)
    t, _s, n = _formula(x, r, w)
    assert total.dtype == normed.dtype == dtype
    _within(total, t, (_half(dtype) + 2.0 ** -23) * t.abs() + _tiny(dtype))
    _within(normed, n, (_half(dtype) + F32) * n.abs() + _tiny(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("with_residual", [True, False])
def test_quantised_with_block_scales(dtype, rows, cols, with_residual):
    x, r, w, _a, _b = _inputs(rows, cols, dtype, rows * 3 + cols)
    r = r if with_residual else None
    total, q, scales = ops.add_rms_norm_quant(x, r, w)
    t, _s, n = _formula(x, r, w)
    assert q.dtype == torch.float8_e4m3fn and scales.shape == (rows, cols // 128) and scales.dtype == torch.float32
    if with_residual:
        _within(total, t, (_half(dtype) + 2.0 ** -23) * t.abs() + _tiny(dtype))
    else:
        assert total is x
    amax = n.view(rows, -1, 128).abs().amax(-1)
    _within(scales, amax / 448, (F32 + 2.0 ** -23) * amax / 448)
    _check_quant(n, q, scales)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 128), (200, 512), (128, 640), (130, 2560)])
def test_quantised_with_scale_atoms(dtype, rows, cols):
    x, r, w, _a, _b = _inputs(rows, cols, dtype, rows * 5 + cols)
    _total, q, atoms = ops.add_rms_norm_quant(x, r, w, scales="mx")
    n = _formula(x, r, w)[2]
    scale = ops.mx_atoms_to_scales(atoms, rows)
    _check_quant(n, q, scale)
    used = n.view(rows, -1, 128).abs().amax(-1) / scale.double()      # the smallest power of two that fits
    assert bool((used <= 448 * (1 + 1e-5)).all()) and bool((used > 224 * (1 - 1e-5)).all())
    assert torch.equal(ops.mx_scale_atoms((torch.log2(scale)).round().to(torch.int32)), atoms)      # slices repeated, no stray bytes


def test_rows_of_zeros_and_of_nan():
    x = torch.zeros(3, 512, device="cuda", dtype=torch.bfloat16)
    x[1, 7] = float("nan")
    w = torch.ones(512, device="cuda", dtype=torch.bfloat16)
    total, q, scales = ops.add_rms_norm_quant(x, torch.zeros_like(x), w)
    assert torch.equal(total[0], x[0]) and bool((q[0].float() == 0).all()) and bool((scales[0] == 1).all())
    assert bool(q[1].float().isnan().all()) and bool((q[2].float() == 0).all())      # one row's NaN stays in it
    _t, normed = ops.add_rms_norm(x, torch.zeros_like(x), w)
    assert bool(normed[1].isnan().all()) and bool((normed[[0, 2]] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES + [(9, 8), (40, 24), (6, 1032), (40000, 256)])
@pytest.mark.parametrize("both", [True, False])
def test_backward(dtype, rows, cols, both):
    t, _r, w, dn, dt = _inputs(rows, cols, dtype, rows * 7 + cols)
    grad, dw = ops.add_rms_norm_backward(t, w, dn, dt if both else None)
    td, s, _n = _formula(t, None, w)
    xh, g = td * s, dn.double() * w.double()
    m = (g * xh).mean(-1, keepdim=True)
    up = dt.double() if both else torch.zeros_like(td)
    want = s * (g - xh * m) + up
    size = s * (g.abs() + xh.abs() * (g * xh).abs().mean(-1, keepdim=True)) + up.abs()
    _within(grad, want, _half(dtype) * want.abs() + 2 * F32 * size + _tiny(dtype))
    # the rows of a column are added in fp32: one lane's share in order (rows / 296 CTAs at the fewest), then 8 warps, 19 + 32 partial sums
    depth = rows / 296 + 64
    terms = dn.double() * xh
    _within(dw, terms.sum(0), _half(dtype) * terms.sum(0).abs() + (depth * 2.0 ** -24 + F32) * terms.abs().sum(0) + _tiny(dtype))


def test_gradients_against_differences_and_repeatability():
    """fp32, the direction of steepest ascent: the loss's change over a step of h against the gradient, off by the third order."""
    x, r, w, dn, dt = _inputs(40, 256, torch.float32, 4)
    x, r, w = (v.requires_grad_() for v in (x, r, w))

    def loss(x, r, w):
        total, normed = ops.add_rms_norm(x, r, w)
        return (total.double() * dt).sum() + (normed.double() * dn).sum()

    gx, gr, gw = torch.autograd.grad(loss(x, r, w), (x, r, w))
    assert torch.equal(gx, gr)
    again = torch.autograd.grad(loss(x, r, w), (x, r, w))
    assert all(torch.equal(a, b) for a, b in zip((gx, gr, gw), again))
    for i, g in enumerate((gx, gr, gw)):
        g64, h = g.double(), 1e-2 / g.double().norm()
        args = [v.detach() for v in (x, r, w)]
        ends = []
        for sign in (1, -1):
            moved = list(args)
            moved[i] = (args[i].double() + sign * h * g64).float()
            ends.append((loss(*moved), (moved[i].double() - args[i].double())))
        slope = (ends[0][0] - ends[1][0])
        want = (g64 * (ends[0][1] - ends[1][1])).sum()
        assert abs(float(slope - want)) <= 2e-3 * abs(float(want))


def test_one_upstream_gradient_alone():
    x, r, w, dn, _dt = _inputs(10, 512, torch.bfloat16, 9)
    x.requires_grad_()
    total, normed = ops.add_rms_norm(x, r, w)
    total.backward(dn)
    assert torch.equal(x.grad, dn)                       # the residual stream passes it on
    x.grad = None
    total, normed = ops.add_rms_norm(x, r, w)
    normed.backward(dn)
    assert torch.equal(x.grad, ops.add_rms_norm_backward(total.detach(), w, dn)[0])


def test_views_streams_and_graphs():
    x, r, w, dn, dt = _inputs(64, 512, torch.bfloat16, 3)
    want = ops.add_rms_norm_quant(x, r, w)
    wide = torch.zeros(64, 1024, device="cuda", dtype=torch.bfloat16)
    wide[:, 4:516] = x                                   # rows off the 16-byte boundary, a stride of twice the width
    got = ops.add_rms_norm_quant(wide[:, 4:516], r.t().contiguous().t(), w)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(want, got))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.add_rms_norm_quant(x.view(4, 16, 512), r.view(4, 16, 512), w)
    torch.cuda.current_stream().wait_stream(side)
    assert got[1].shape == (4, 16, 512) and got[2].shape == (4, 16, 4)
    assert torch.equal(got[1].view(64, 512).view(torch.uint8), want[1].view(torch.uint8))
    # two captured calls, replayed after the inputs changed, in the other order
    grads = []
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            grads.append(ops.add_rms_norm_backward(x, w, dn, dt))
        graphs.append(graph)
    dn.copy_(dt)
    graphs[1].replay()
    graphs[0].replay()
    plain = ops.add_rms_norm_backward(x, w, dn, dt)
    for g in grads:
        assert torch.equal(g[0], plain[0]) and torch.equal(g[1], plain[1])


def test_empty_and_refused():
    w = torch.ones(512, device="cuda", dtype=torch.bfloat16)
    x = torch.zeros(0, 512, device="cuda", dtype=torch.bfloat16)
    total, q, s = ops.add_rms_norm_quant(x, x, w)
    assert total.shape == q.shape == (0, 512) and s.shape == (0, 4)
    grad, dw = ops.add_rms_norm_backward(x, w, x, x)
    assert grad.shape == (0, 512) and bool((dw == 0).all())
    y = torch.zeros(4, 512, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="forward-only"):
        ops.add_rms_norm_quant(y.clone().requires_grad_(), y, w)
    with pytest.raises(ValueError, match="dtype"):
        ops.add_rms_norm(y, y.float(), w)
    with pytest.raises(RuntimeError, match="does not support dtype"):
        ops.add_rms_norm(y.double(), y.double(), w)
