"""What a caller of `ragged_linear` asks for about waits that give up reaches the backward pass too (no GPU: the kernels' calls are replaced)."""
from __future__ import annotations

import pytest
import torch

from taac_2026_b200 import ops


@pytest.mark.parametrize("check", [False, True])
@pytest.mark.parametrize("with_word", [False, True])
def test_check_and_status_reach_the_backward_pass(monkeypatch, check, with_word):
    word = torch.zeros(1, dtype=torch.int32) if with_word else None
    seen = {}

    def forward(x, weight, offsets, bias=None, *, residual=None, check=False, status=None):
        seen["forward"] = (check, status)
        return x.new_zeros(x.shape[0], weight.shape[1])

    def backward(x, weight, offsets, grad_out, *, scales=None, bias=False, need_x=True, need_weight=True, check=False, status=None):
        seen["backward"] = (check, status)
        return torch.zeros_like(x), torch.zeros_like(weight), None

    monkeypatch.setattr(ops, "ragged_linear", forward)
    monkeypatch.setattr(ops, "ragged_linear_backward", backward)
    x, w = torch.ones(6, 64).requires_grad_(), torch.ones(2, 16, 64).requires_grad_()
    off = torch.tensor([0, 2, 6], dtype=torch.int32)
    ops._RaggedLinearFunction.apply(x, w, off, None, None, False, check, word).sum().backward()
    for which in ("forward", "backward"):
        assert seen[which][0] is check and seen[which][1] is word


def test_a_wait_that_gave_up_in_the_backward_pass_is_an_error(monkeypatch):
    """With check=True the incomplete gradients do not look like gradients."""
    monkeypatch.setattr(ops, "ragged_linear", lambda x, weight, offsets, bias=None, **kw: x.new_zeros(x.shape[0], weight.shape[1]))

    def backward(x, weight, offsets, grad_out, *, check=False, status=None, **kw):
        ops._raise_incomplete("ragged_linear_backward", check, torch.ones(1, dtype=torch.int32))
        return torch.zeros_like(x), torch.zeros_like(weight), None

    monkeypatch.setattr(ops, "ragged_linear_backward", backward)
    x, w = torch.ones(6, 64).requires_grad_(), torch.ones(2, 16, 64).requires_grad_()
    out = ops._RaggedLinearFunction.apply(x, w, torch.tensor([0, 2, 6], dtype=torch.int32), None, None, False, True, None)
    with pytest.raises(RuntimeError, match="gave up"):
        out.sum().backward()
