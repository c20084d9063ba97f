"""The feed-forward operators without the host module and under kernel timing: the same bits as the plain call."""
from __future__ import annotations

import pytest
import torch

from conftest import gpu_ready
from taac_2026_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _need_gpu():
    if not gpu_ready():
        pytest.fail("gpu tests need an sm_100 device and a built libtb200.so")


def _calls():
    g = torch.Generator(device="cuda").manual_seed(2)
    make = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()  # noqa: E731
    x, r, w, up = make(90, 512), make(90, 512), make(512), make(90, 512)
    rows, weight, dy = make(90, 136), make(3, 264, 136), make(90, 264)
    bias = make(3, 264).float()
    off = torch.tensor([0, 30, 30, 90], dtype=torch.int32, device="cuda")
    kept = ops.silu_gate_checkpoint(up)
    return {
        "add_rms_norm": lambda: ops.add_rms_norm(x, r, w),
        "add_rms_norm_quant": lambda: ops.add_rms_norm_quant(x, r, w),
        "add_rms_norm_quant mx": lambda: ops.add_rms_norm_quant(x, None, w, scales="mx"),
        "add_rms_norm_bwd": lambda: ops.add_rms_norm_backward(x, w, r, up),
        "silu_gate": lambda: ops.silu_gate_checkpoint(up),
        "silu_gate plain": lambda: (ops.silu_gate(up, gate_first=False),),
        "silu_gate_bwd": lambda: ops.silu_gate_backward(kept[1], kept[2], kept[0]),
        "ragged_linear": lambda: (ops.ragged_linear(rows, weight, off, bias, silu=True),),
        "ragged_linear residual": lambda: (ops.ragged_linear(rows, weight, off, bias, residual=dy),),
        "ragged_linear_backward": lambda: ops.ragged_linear_backward(rows, weight, off, dy, bias=True),
    }


def _bits(values):
    return [v.contiguous().view(torch.uint8) for v in values]


@pytest.mark.parametrize("name", ["add_rms_norm", "add_rms_norm_quant", "add_rms_norm_quant mx", "add_rms_norm_bwd", "silu_gate", "silu_gate plain",
                                  "silu_gate_bwd", "ragged_linear", "ragged_linear residual", "ragged_linear_backward"])
def test_general_path_and_timing(name, monkeypatch):
    call = _calls()[name]
    plain = _bits(call())
    sink = []
    ops.set_kernel_timing(sink)
    try:
        timed = _bits(call())
    finally:
        ops.set_kernel_timing(None)
    torch.cuda.synchronize()
    assert sink and all(start.elapsed_time(end) > 0 for _n, _m, start, end in sink)
    monkeypatch.setattr(ops, "_host", ops._NoHost())
    general = _bits(call())
    assert len(plain) == len(timed) == len(general)
    for a, b, c in zip(plain, timed, general):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_every_public_name_is_there():
    for name in ("add_rms_norm", "add_rms_norm_quant", "add_rms_norm_backward", "checkpoint_activation", "restore_activation", "silu_gate",
                 "silu_gate_checkpoint", "silu_gate_backward", "ragged_linear", "ragged_linear_backward"):
        assert name in ops.__all__ and (getattr(ops, name).__doc__ or "").strip()
