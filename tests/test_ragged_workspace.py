"""What the weight gradients of ragged layers ask for as workspace: each kind of call its own, and nothing that it does not read."""
from __future__ import annotations

import pytest
import torch

from conftest import gpu_ready
from taac_2026_b200 import _lib, ops

SIZES = [(1, 1, 64, 64), (8, 4096, 512, 512), (1, 200000, 512, 512), (2048, 131072, 8192, 512), (16, 32768, 2048, 512)]


@pytest.mark.parametrize("experts,rows,n,k", SIZES)
def test_sizes_without_a_device(experts, rows, n, k):
    if not _lib.LIB_PATH.exists():
        pytest.skip("libtb200.so is not built")
    if torch.cuda.is_available():
        pytest.skip("needs a machine without a GPU")
    lib = _lib.load()
    assert lib.tb200_ragged_wgrad_workspace_bytes(experts, rows, n, k) == 0
    assert lib.tb200_ragged_wgrad_workspace_of(experts, rows, n, k, 0) == lib.tb200_ragged_wgrad_workspace_of(experts, rows, n, k, 1) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("experts,rows,n,k", SIZES)
def test_sizes(experts, rows, n, k):
    assert gpu_ready()
    lib = _lib.load()
    weights, bias = (lib.tb200_ragged_wgrad_workspace_of(experts, rows, n, k, w) for w in (1, 0))
    assert lib.tb200_ragged_wgrad_workspace_bytes(experts, rows, n, k) == max(weights, bias)
    assert bias >= 4 * (experts + 1) * n                  # a partial sum for every expert and every chunk of rows
    pairs = torch.cuda.get_device_properties(0).multi_processor_count // 2
    assert weights in (0, 4 * pairs * (8 + 2 * 256 + 2 * 256 * 256))      # two partial tiles a pair with their sums and places, or nothing
    for bad in ((0, rows, n, k), (experts, -1, n, k), (experts, rows, 12, k)):
        assert lib.tb200_ragged_wgrad_workspace_of(*bad, 0) == lib.tb200_ragged_wgrad_workspace_of(*bad, 1) == 0


@pytest.mark.gpu
def test_a_call_takes_no_more_than_its_results():
    """2048 experts: the table of the kernel for bias gradients alone would be 10 MB beside the results."""
    experts, rows, n, k = 2048, 4096, 1024, 8
    x, dy = (torch.randn(rows, c, device="cuda").bfloat16() for c in (k, n))
    w = torch.randn(experts, n, k, device="cuda").bfloat16()
    off = torch.arange(0, rows + 1, rows // experts, dtype=torch.int32, device="cuda")
    call = lambda: ops.ragged_linear_backward(x, w, off, dy, bias=True)  # noqa: E731
    results = sum(t.numel() * t.element_size() for t in call())
    assert ops._lib.load().tb200_ragged_wgrad_workspace_of(experts, rows, n, k, 1) == 0
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    call()
    assert torch.cuda.max_memory_allocated() - before <= results + (1 << 20)
