"""`add_rms_norm_quant` and `add_rms_norm_backward` at the ends of their range: blocks whose largest value lies anywhere in fp32, and
eps = 0 where lanes of a warp have no row.

Tolerances as in test_gpu_add_norm.py: F32 for the fp32 steps in front of a stored value, half an e4m3 step for q.  Next to fp32's
subnormal numbers the value and its block's scale are each off by up to half a step of 2^-149, the scale's counted up to 448 times."""
from __future__ import annotations

import pytest
import torch

from conftest import gpu_ready
from taac_2026_b200 import ops

pytestmark = pytest.mark.gpu

F32 = 40 * 2.0 ** -24
STEP = 2.0 ** -150      # half a step of fp32's subnormal numbers


@pytest.fixture(autouse=True)
def _need_gpu():
    if not gpu_ready():
        pytest.fail("gpu tests need an sm_100 device and a built libtb200.so")


def _within(got, want, tol):
    assert got.shape == want.shape
    off = (got.double() - want).abs() - tol
    assert bool((off <= 0).all()), float(off.max())


# around the borders of what the kernel tells apart, the ends of fp32, and ordinary values between
POWERS = [-149, -144, -140, -133, -130, -127, -126, -125, -122, -118, -117, -101, -100, -99, -50, 0, 50, 99, 100, 101, 118, 120, 124, 125, 126, 127]


@pytest.mark.parametrize("scales", ["1x128", "mx"])
@pytest.mark.parametrize("cols", [128, 512, 2560])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_blocks_of_every_magnitude(dtype, cols, scales):
    """Uniform in [-1, 1] the normalised values stay below 1.74 + a few per cent, so that 2^127 times them is still finite."""
    g = torch.Generator(device="cuda").manual_seed(cols)
    x = (torch.rand(9, cols, generator=g, device="cuda") * 2 - 1).to(dtype)
    xd = x.double()
    xh = xd * torch.rsqrt(xd.pow(2).mean(-1, keepdim=True) + 1e-6)
    assert float(xh.abs().max()) < 1.99
    for power in POWERS:
        weight = torch.full((cols,), 2.0 ** power, device="cuda", dtype=torch.float64).to(dtype)      # bf16 below 2^-133: zeros
        n = xh * weight.double()
        _total, q, sc = ops.add_rms_norm_quant(x, None, weight, scales=scales)
        if scales == "mx":
            sc = ops.mx_atoms_to_scales(sc, 9)
        amax = n.view(9, -1, 128).abs().amax(-1)
        if scales == "1x128":      # a scale that rounds to zero is one, its block zeros; n's own rounding may take it over that border
            want = torch.where(amax / 448 > STEP, amax / 448, torch.ones_like(amax))
            border = (amax / 448 - STEP).abs() <= 1e-2 * STEP
            _within(torch.where(border, want, sc.double()), want, (F32 + 2.0 ** -23) * want + 1.01 * STEP)
        assert bool(sc.isfinite().all()) and bool((sc > 0).all())
        wide = sc.double().repeat_interleave(128, -1)
        _within(q.double() * wide, n, torch.maximum(2.0 ** -4 * n.abs(), 2.0 ** -10 * wide) * (1 + 1e-5) + 450 * STEP)


def test_blocks_of_different_magnitude_in_a_row():
    """One row's blocks from 2^-140 to 2^120: each has a factor of its own."""
    powers = [-140, -127, -100, -99, 0, 100, 101, 120]
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.rand(5, 1024, generator=g, device="cuda") * 2 - 1
    weight = torch.cat([torch.full((128,), 2.0 ** p, device="cuda", dtype=torch.float64) for p in powers]).float()
    _total, q, sc = ops.add_rms_norm_quant(x, None, weight)
    xd = x.double()
    n = xd * torch.rsqrt(xd.pow(2).mean(-1, keepdim=True) + 1e-6) * weight.double()
    wide = sc.double().repeat_interleave(128, -1)
    _within(q.double() * wide, n, torch.maximum(2.0 ** -4 * n.abs(), 2.0 ** -10 * wide) * (1 + 1e-5) + 450 * STEP)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("cols", [8, 64, 128, 256, 1024])
@pytest.mark.parametrize("rows", [1, 2, 15, 17, 301])
def test_gradient_of_the_weight_without_eps(dtype, cols, rows):
    """A row of 16 lanes shares its warp with another, which has none where the number of rows is odd."""
    g = torch.Generator(device="cuda").manual_seed(rows * 1000 + cols)
    t, dn = (torch.randn(rows, cols, generator=g, device="cuda").to(dtype) for _ in range(2))
    w = torch.ones(cols, device="cuda", dtype=dtype)
    grad, dw = ops.add_rms_norm_backward(t, w, dn, None, eps=0.0)
    td, gd = t.double(), dn.double()
    s = torch.rsqrt(td.pow(2).mean(-1, keepdim=True))
    xh = td * s
    half, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    m = (gd * xh).mean(-1, keepdim=True)
    want = s * (gd - xh * m)
    _within(grad, want, half * want.abs() + 2 * F32 * s * (gd.abs() + xh.abs() * (gd * xh).abs().mean(-1, keepdim=True)) + tiny)
    terms = gd * xh
    _within(dw, terms.sum(0), half * terms.sum(0).abs() + ((rows / 296 + 64) * 2.0 ** -24 + F32) * terms.abs().sum(0) + tiny)
