"""Values kept in 8 bits at the upper end of their type's range: what is finite comes back finite, within half an e4m3 step."""
from __future__ import annotations

import pytest
import torch

from conftest import gpu_ready
from taac_2026_b200 import ops

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(autouse=True)
def _need_gpu():
    if not gpu_ready():
        pytest.fail("gpu tests need an sm_100 device and a built libtb200.so")


def _ends(dtype):
    """One block a row whose largest value is at the end of the range; 2^-4 of it is the last binade's half step: 31 / 32 of
    the power of two behind the range (63488 in fp16) is the first value that rounds to that power of two."""
    top = torch.finfo(dtype).max
    behind = 2.0 ** 16 if dtype == torch.float16 else 2.0 ** 128
    values = [top, -top, behind * 31 / 32, behind * 30.75 / 32, behind * 15 / 16, behind / 2, -behind * 31 / 32]
    x = torch.zeros(len(values) + 1, 128, device="cuda", dtype=torch.float64)
    for i, v in enumerate(values):
        x[i, i], x[i, 127] = v, 1.0
    x[-1] = top
    return x.to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_finite_values_come_back_finite(dtype):
    x = _ends(dtype)
    back = ops.restore_activation(*ops.checkpoint_activation(x), dtype)
    assert bool(back.isfinite().all())
    off = (back.double() - x.double()).abs()
    assert bool((off[x != 1] <= 2.0 ** -4 * x[x != 1].double().abs()).all())
    x[0, 3], x[1, 5] = float("nan"), float("inf")
    q, s = ops.checkpoint_activation(x)
    assert int(ops.restore_activation(q, s, dtype).isnan().sum()) == 2
    for other in TYPES:      # a type that the values do not fit: its largest number, with the sign
        got = ops.restore_activation(q, s, other)
        assert int(got.isnan().sum()) == 2 and bool(got[~got.isnan()].isfinite().all())
        assert torch.equal(torch.sign(got[2:].double()), torch.sign(ops.restore_activation(q, s, torch.float32)[2:].double()))


@pytest.mark.parametrize("dtype", TYPES)
def test_activation_of_finite_values_is_finite(dtype):
    """h again from the kept values where the forward pass's h is finite, and a gradient without NaN (silu's slope is 1 up there)."""
    x = _ends(dtype)
    h, q, s = ops.silu_gate_checkpoint(x, gated=False)
    assert bool(h.isfinite().all())
    dh = torch.ones_like(h)
    dup, again = ops.silu_gate_backward(q, s, dh, gated=False)
    assert bool(again.isfinite().all()) and bool(dup.isfinite().all())
    off = (again.double() - h.double()).abs()
    assert bool((off[h > 2] <= 2.0 ** -4 * h[h > 2].double()).all())
    assert bool((dup[x > 100] == 1).all()) and bool((dup[x < -200] == 0).all())
    # gate and value whose product is in range, and behind it after their rounding to 8 bits (31 -> 32 each)
    half = 8 if dtype == torch.float16 else 64
    up = torch.zeros(2, 256, device="cuda", dtype=torch.float64)
    up[0, :128], up[0, 128:] = 2.0 ** half * 31 / 32, 2.0 ** half * 31 / 32
    up[1, :128], up[1, 128:] = 2.0 ** half * 31 / 32, -(2.0 ** half) * 31 / 32
    up = up.to(dtype)
    h, q, s = ops.silu_gate_checkpoint(up)
    assert bool(h.isfinite().all())
    _dup, again = ops.silu_gate_backward(q, s, torch.ones_like(h))
    assert bool((again[0] == torch.finfo(dtype).max).all()) and bool((again[1] == -torch.finfo(dtype).max).all())
    up[0, 0] = float("nan")
    _h, q, s = ops.silu_gate_checkpoint(up)
    _dup, again = ops.silu_gate_backward(q, s, torch.ones_like(h))
    assert bool(again[0, 0].isnan()) and int(again.isnan().sum()) == 1


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_weight_gradient_of_a_kept_input_at_the_end_of_the_range(dtype):
    """Beside a zero of the gradient an infinite input would be NaN."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(40, 256, generator=g, device="cuda").to(dtype)
    x[3, 7], x[11, 200] = torch.finfo(dtype).max, -torch.finfo(dtype).max
    w = (torch.randn(2, 64, 256, generator=g, device="cuda") / 16).to(dtype)
    off = torch.tensor([0, 10, 40], dtype=torch.int32, device="cuda")
    dy = torch.randn(40, 64, generator=g, device="cuda").to(dtype)
    dy[3], dy[11] = 0, 0
    weight = w.clone().requires_grad_()
    out = ops.ragged_linear(x, weight, off, checkpoint=True)
    out.backward(dy)
    assert bool(weight.grad.isfinite().all())
    kept = x.clone()
    kept[3], kept[11] = 0, 0                              # rows that the gradient does not look at: any value is right
    values = ops.restore_activation(*ops.checkpoint_activation(kept), dtype)
    assert torch.equal(weight.grad, ops.ragged_linear_backward(values, w, off, dy)[1])


@pytest.mark.parametrize("dtype", TYPES)
def test_more_than_two_dimensions(dtype):
    """[4, 10, 512] and a strided view of it: the bits of the matrix of its rows, in its shape."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(4, 10, 512, generator=g, device="cuda").to(dtype)
    pad = torch.zeros(4, 11, 520, device="cuda", dtype=dtype)
    pad[:, :10, 3:515] = x
    bits = lambda ts: [t.contiguous().view(torch.uint8).flatten() for t in ts]  # noqa: E731
    for y in (x, pad[:, :10, 3:515]):
        q, s = ops.checkpoint_activation(y)
        assert q.shape == (4, 10, 512) and s.shape == (4, 10, 4)
        assert all(torch.equal(a, b) for a, b in zip(bits((q, s)), bits(ops.checkpoint_activation(x.view(40, 512)))))
        assert torch.equal(ops.restore_activation(q, s, dtype).view(40, 512), ops.restore_activation(q.view(40, 512), s.view(40, 4), dtype))
        h, q, s = ops.silu_gate_checkpoint(y)
        assert h.shape == (4, 10, 256) and q.shape == (4, 10, 512) and s.shape == (4, 10, 4)
        assert all(torch.equal(a, b) for a, b in zip(bits((h, q, s)), bits(ops.silu_gate_checkpoint(x.view(40, 512)))))
        dup, again = ops.silu_gate_backward(q, s, h)
        assert dup.shape == (4, 10, 512) and again.shape == (4, 10, 256)
        assert all(torch.equal(a, b) for a, b in zip(bits((dup, again)), bits(ops.silu_gate_backward(q.view(40, 512), s.view(40, 4), h.view(40, 256)))))
