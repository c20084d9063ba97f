"""Refusals of the feed-forward operators that need no GPU: shapes before the backend, no CPU path, and the C ABI's own checks."""
from __future__ import annotations

import ctypes

import pytest
import torch

from taac_2026_b200 import _lib, ops

OK, ERR_NULL, ERR_DTYPE, ERR_SHAPE, ERR_ALIGN, ERR_UNSUPPORTED = 0, -1, -2, -3, -4, -5
BF16 = 2
P = ctypes.c_void_p


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        pytest.skip("libtb200.so is not built")
    return _lib.load()


def test_shapes_are_looked_at_first():
    x, w = torch.ones(4, 256), torch.ones(256)
    with pytest.raises(ValueError, match="at least 2 dimensions"):
        ops.add_rms_norm(torch.ones(256), torch.ones(256), w)
    with pytest.raises(ValueError, match="does not match weight size"):
        ops.add_rms_norm(x, x, torch.ones(128))
    with pytest.raises(ValueError, match="residual must have"):
        ops.add_rms_norm(x, x[:2], w)
    with pytest.raises(ValueError, match="needs a residual"):
        ops.add_rms_norm(x, None, w)
    with pytest.raises(ValueError, match="multiple of 128"):
        ops.add_rms_norm_quant(torch.ones(4, 200), None, torch.ones(200))
    with pytest.raises(ValueError, match="unknown add_rms_norm_quant scales"):
        ops.add_rms_norm_quant(x, x, w, scales="rowwise")
    with pytest.raises(ValueError, match="unsupported add_rms_norm backend"):
        ops.add_rms_norm(x, x, w, backend="triton")
    with pytest.raises(ValueError, match="multiple of 8 of at most 16384"):
        ops.add_rms_norm(torch.ones(2, 16392), torch.ones(2, 16392), torch.ones(16392))
    with pytest.raises(ValueError, match="total's shape"):
        ops.add_rms_norm_backward(x, w, x[:2])
    with pytest.raises(ValueError, match="multiple of 128"):
        ops.checkpoint_activation(torch.ones(4, 100))
    with pytest.raises(ValueError, match="multiple of 256"):
        ops.silu_gate(torch.ones(4, 128))
    with pytest.raises(ValueError, match="unsupported silu_gate backend"):
        ops.silu_gate(x, backend="torch")


def test_no_cpu_path(monkeypatch):
    monkeypatch.setattr(ops, "cuda_available", lambda: True)
    x, w = torch.ones(4, 256), torch.ones(256)
    q, s = torch.ones(4, 256).to(torch.float8_e4m3fn), torch.ones(4, 2)
    for call in (lambda: ops.add_rms_norm(x, x, w), lambda: ops.add_rms_norm_quant(x, x, w), lambda: ops.add_rms_norm_backward(x, w, x, x),
                 lambda: ops.checkpoint_activation(x), lambda: ops.restore_activation(q, s), lambda: ops.silu_gate(x),
                 lambda: ops.silu_gate_checkpoint(x), lambda: ops.silu_gate_backward(q, s, x[:, :128])):
        with pytest.raises(RuntimeError, match="requires CUDA tensors"):
            call()


def test_add_norm_entries(lib):
    buf = (ctypes.c_uint8 * 256)()
    p = (ctypes.addressof(buf) + 15) & ~15

    def fwd(x=P(p), r=P(p), g=P(p), total=P(p), normed=P(p), q=None, s=None, kind=0, rows=4, cols=128, dtype=BF16):
        return lib.tb200_add_rmsnorm_fwd(x, r, g, total, normed, q, s, kind, rows, cols, 1e-6, dtype, None)

    assert fwd(rows=0) == OK
    assert fwd(rows=-1) == ERR_SHAPE and fwd(cols=0) == ERR_SHAPE
    assert fwd(dtype=7) == ERR_DTYPE and fwd(kind=3) == ERR_UNSUPPORTED
    assert fwd(cols=100) == ERR_UNSUPPORTED and fwd(cols=16392) == ERR_UNSUPPORTED
    assert fwd(kind=1, q=P(p), s=P(p), cols=136) == ERR_UNSUPPORTED       # blocks of 128
    assert fwd(x=None) == ERR_NULL and fwd(total=None, normed=None) == ERR_NULL
    assert fwd(kind=1, q=P(p)) == ERR_NULL and fwd(kind=2, s=P(p)) == ERR_NULL
    assert fwd(q=P(p)) == ERR_UNSUPPORTED                                 # 8 bits without a kind of scales
    assert fwd(x=P(p + 2)) == ERR_ALIGN and fwd(r=P(p + 8)) == ERR_ALIGN
    bwd = lib.tb200_add_rmsnorm_bwd
    assert bwd(P(p), P(p), P(p), None, P(p), P(p), P(p), -1, 128, 1e-6, BF16, None) == ERR_SHAPE
    assert bwd(P(p), P(p), None, None, P(p), P(p), P(p), 4, 128, 1e-6, BF16, None) == ERR_NULL
    assert bwd(P(p), P(p), P(p), None, P(p), P(p), None, 4, 128, 1e-6, BF16, None) == ERR_NULL
    assert bwd(P(p), P(p), P(p), P(p + 4), P(p), P(p), P(p), 4, 128, 1e-6, BF16, None) == ERR_ALIGN
    assert bwd(P(p), P(p), P(p), None, P(p), P(p), P(p), 4, 100, 1e-6, BF16, None) == ERR_UNSUPPORTED
    assert lib.tb200_add_rmsnorm_bwd_workspace_bytes(0) == 0 and lib.tb200_add_rmsnorm_bwd_workspace_bytes(512) >= 4 * 512


def test_kept_activation_entries(lib):
    buf = (ctypes.c_uint8 * 256)()
    p = (ctypes.addressof(buf) + 15) & ~15
    for fn in (lib.tb200_keep_fwd, lib.tb200_keep_restore):
        assert fn(P(p), P(p), P(p), 0, 128, BF16, None) == OK
        assert fn(P(p), P(p), P(p), 4, 100, BF16, None) == ERR_SHAPE
        assert fn(P(p), P(p), P(p), 4, 128, 9, None) == ERR_DTYPE
        assert fn(P(p), None, P(p), 4, 128, BF16, None) == ERR_NULL
    assert lib.tb200_keep_fwd(P(p + 2), P(p), P(p), 4, 128, BF16, None) == ERR_ALIGN
    fwd, bwd = lib.tb200_silu_gate_fwd, lib.tb200_silu_gate_bwd
    assert fwd(P(p), P(p), None, None, 0, 128, 1, 1, BF16, None) == OK
    assert fwd(P(p), P(p), P(p), None, 4, 128, 1, 1, BF16, None) == ERR_NULL          # values without scales
    assert fwd(P(p), P(p), None, None, 4, 64, 1, 1, BF16, None) == ERR_SHAPE
    assert fwd(P(p), P(p + 8), None, None, 4, 128, 1, 1, BF16, None) == ERR_ALIGN
    assert bwd(P(p), P(p), None, P(p), None, 4, 128, 1, 1, BF16, None) == ERR_NULL
    assert bwd(P(p), P(p), P(p), P(p), P(p + 8), 4, 128, 1, 1, BF16, None) == ERR_ALIGN


def test_ragged_shapes_are_looked_at_first():
    x, w, off = torch.ones(6, 64), torch.ones(2, 16, 64), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="rows \\[T, width\\]"):
        ops.ragged_linear(x[None], w, off)
    with pytest.raises(ValueError, match="do not fit weight"):
        ops.ragged_linear(x[:, :32], w, off)
    with pytest.raises(ValueError, match="offsets must be \\[E \\+ 1\\]"):
        ops.ragged_linear(x, w, off[:2])
    with pytest.raises(ValueError, match="offsets must be int32"):
        ops.ragged_linear(x, w, off.long())
    with pytest.raises(ValueError, match="N % 8"):
        ops.ragged_linear(x, w[:, :12], off)
    with pytest.raises(ValueError, match="grad_out"):
        ops.ragged_linear_backward(x, w, off, torch.ones(5, 16))
    with pytest.raises(ValueError, match="do not fit weight"):
        ops.ragged_linear_backward(x, w, off, torch.ones(6, 24))


def test_ragged_has_no_cpu_path(monkeypatch):
    monkeypatch.setattr(ops, "cuda_available", lambda: True)
    x, w, off = torch.ones(6, 64).bfloat16(), torch.ones(2, 16, 64).bfloat16(), torch.zeros(3, dtype=torch.int32)
    for call in (lambda: ops.ragged_linear(x, w, off), lambda: ops.ragged_linear_backward(x, w, off, x[:, :16].contiguous())):
        with pytest.raises(RuntimeError, match="requires CUDA tensors"):
            call()


def test_ragged_entries(lib):
    buf = (ctypes.c_uint8 * 256)()
    p = (ctypes.addressof(buf) + 15) & ~15

    def rows(x=P(p), w=P(p), off=P(p), bias=None, res=None, out=P(p), experts=2, T=4, n=64, k=64, act=0, dtype=BF16):
        return lib.tb200_ragged_gemm(x, w, off, bias, res, out, experts, T, n, k, act, 1, dtype, None, None)

    assert rows(T=0) == OK
    assert rows(T=-1) == ERR_SHAPE and rows(n=12) == ERR_SHAPE and rows(k=0) == ERR_SHAPE and rows(experts=5000) == ERR_SHAPE
    assert rows(T=1 << 31) == ERR_SHAPE                                    # row numbers are held in 32 bits
    assert rows(dtype=0) == ERR_DTYPE and rows(act=2) == ERR_UNSUPPORTED
    assert rows(x=None) == ERR_NULL and rows(off=None) == ERR_NULL and rows(w=None) == ERR_NULL and rows(out=None) == ERR_NULL
    assert rows(x=P(p + 2)) == ERR_ALIGN and rows(res=P(p + 8)) == ERR_ALIGN and rows(bias=P(p + 4)) == ERR_ALIGN and rows(off=P(p + 2)) == ERR_ALIGN
    dgrad, wgrad = lib.tb200_ragged_gemm_dgrad, lib.tb200_ragged_gemm_wgrad
    assert dgrad(P(p), P(p), P(p), P(p), 2, 0, 64, 64, BF16, None, None) == OK
    assert dgrad(P(p), None, P(p), P(p), 2, 4, 64, 64, BF16, None, None) == ERR_NULL
    assert dgrad(P(p), P(p), P(p), P(p + 8), 2, 4, 64, 64, BF16, None, None) == ERR_ALIGN
    assert wgrad(P(p), P(p), P(p), P(p), None, P(p), 0, 4, 64, 64, BF16, None, None) == OK
    assert wgrad(P(p), P(p), P(p), None, None, P(p), 2, 4, 64, 64, BF16, None, None) == ERR_NULL
    assert wgrad(P(p), P(p), P(p), P(p), None, None, 2, 4, 64, 64, BF16, None, None) == ERR_NULL
    assert wgrad(None, P(p), P(p), P(p), None, P(p), 2, 4, 64, 64, BF16, None, None) == ERR_NULL
    assert wgrad(P(p), P(p), P(p), P(p), P(p + 4), P(p), 2, 4, 64, 64, BF16, None, None) == ERR_ALIGN
    size = lib.tb200_ragged_wgrad_workspace_bytes
    assert size(0, 4, 64, 64) == 0 and size(2, -1, 64, 64) == 0 and size(2, 4, 12, 64) == 0
    assert size(1, 100000, 512, 512) >= 0 and size(8, 4096, 512, 512) >= 0          # without a device too
