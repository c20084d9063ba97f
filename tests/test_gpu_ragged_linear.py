"""Linear layers grouped by expert with ragged sizes (`ragged_linear`, `ragged_linear_backward`) against 64 bits, group by group.

Tolerance of a sum of n products: one rounding of half a step of the result's type, and the tensor cores' fp32 accumulation, which
adds sixteen products at a time and may cut instead of round: (n / 16 + 16) steps of 2^-23 of the sum of the absolute products (the
16: bias, residual, the activation, and the joining of up to eight partial sums)."""
from __future__ import annotations

import pytest
import torch

from conftest import gpu_ready
from taac_2026_b200 import ops

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def _need_gpu():
    if not gpu_ready():
        pytest.fail("gpu tests need an sm_100 device and a built libtb200.so")


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def _case(sizes, n, k, dtype, seed, lead=0, behind=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    total = sum(sizes) + lead + behind
    x = torch.randn(total, k, generator=g, device="cuda").to(dtype)
    w = (torch.randn(len(sizes), n, k, generator=g, device="cuda") * k ** -0.5).to(dtype)
    dy = torch.randn(total, n, generator=g, device="cuda").to(dtype)
    bias = torch.randn(len(sizes), n, generator=g, device="cuda")
    ends = [lead]
    for s in sizes:
        ends.append(ends[-1] + s)
    return x, w, torch.tensor(ends, dtype=torch.int32, device="cuda"), dy, bias, ends


def _within(got, want, tol):
    assert got.shape == want.shape
    off = (got.double() - want).abs() - tol
    assert bool((off <= 0).all()), float(off.max())      # a NaN fails as well


def _steps(n):
    return (n / 16 + 16) * 2.0 ** -23


def _check_rows(out, x, w, ends, bias=None, silu=False, residual=None):
    dtype, k = out.dtype, w.shape[2]
    for e in range(len(ends) - 1):
        r = slice(ends[e], ends[e + 1])
        z = x[r].double() @ w[e].double().T
        size = x[r].double().abs() @ w[e].double().abs().T
        if bias is not None:
            z, size = z + bias[e].double(), size + bias[e].double().abs()
        if silu:      # slope at most 1.1; the exponential and the reciprocal within 1e-5
            z, size = z * torch.sigmoid(z), 1.1 * size + 1e-5 / 2.0 ** -23 / (k / 16 + 16) * z.abs()
        if residual is not None:
            z, size = z + residual[r].double(), size + residual[r].double().abs()
        _within(out[r], z, _half(dtype) * z.abs() + _steps(k) * size + _tiny(dtype))


def _check_grads(dx, dw, db, x, w, dy, ends):
    dtype, n = dx.dtype, w.shape[1]
    for e in range(len(ends) - 1):
        r = slice(ends[e], ends[e + 1])
        xe, we, ge = x[r].double(), w[e].double(), dy[r].double()
        want = ge @ we
        _within(dx[r], want, _half(dtype) * want.abs() + _steps(n) * (ge.abs() @ we.abs()) + _tiny(dtype))
        want = ge.T @ xe
        _within(dw[e], want, _half(dtype) * want.abs() + _steps(len(xe)) * (ge.abs().T @ xe.abs()) + _tiny(dtype))
        if db is not None:      # fp32: every eighth row in order in a lane (in a thread of 1 to 8 without dw), then 3 + 74 or 8 + 74 partial sums
            _within(db[e], ge.sum(0), (100 + len(xe) / 8) * 2.0 ** -24 * ge.abs().sum(0))


SIZES = [
    ([1], 64, 64), ([0], 64, 64), ([5, 0, 3], 8, 8), ([1, 1, 1, 1], 256, 512), ([17, 64, 0, 1, 100], 200, 72), ([63, 64, 65, 128, 129], 264, 520),
    ([256, 257, 255, 0, 0, 1], 512, 256), ([300, 1, 700, 12], 1000, 328), ([40] * 40, 128, 96), ([2000, 0, 3000, 50], 520, 512),
    ([0, 0, 4097], 256, 256), ([9000, 10, 1030], 776, 264),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes,n,k", SIZES)
def test_forward(dtype, sizes, n, k):
    x, w, off, dy, bias, ends = _case(sizes, n, k, dtype, n + k)
    _check_rows(ops.ragged_linear(x, w, off, check=True), x, w, ends)
    _check_rows(ops.ragged_linear(x, w, off, bias, silu=True, check=True), x, w, ends, bias, True)
    res = dy.clone()
    got = ops.ragged_linear(x, w, off, bias, residual=res, check=True)
    assert torch.equal(res, dy)
    _check_rows(got, x, w, ends, bias, False, dy)
    into = ops.ragged_linear(x, w, off, bias, residual=res, out=res, check=True)
    assert into.data_ptr() == res.data_ptr() and torch.equal(into, got)      # in place


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes,n,k", SIZES)
def test_backward(dtype, sizes, n, k):
    x, w, off, dy, bias, ends = _case(sizes, n, k, dtype, 3 * n + k)
    dx, dw, db = ops.ragged_linear_backward(x, w, off, dy, bias=True, check=True)
    assert dx.dtype == dw.dtype == dtype and db.dtype == torch.float32
    _check_grads(dx, dw, db, x, w, dy, ends)
    again = ops.ragged_linear_backward(x, w, off, dy, bias=True)
    assert all(torch.equal(a, b) for a, b in zip((dx, dw, db), again))       # sums in a fixed order
    only = ops.ragged_linear_backward(x, w, off, dy, need_x=False)
    assert only[0] is None and only[2] is None and torch.equal(only[1], dw)
    only = ops.ragged_linear_backward(x, w, off, dy, need_weight=False, bias=True)
    assert only[1] is None and torch.equal(only[0], dx)
    _check_grads(only[0], dw, only[2], x, w, dy, ends)                       # a kernel of its own adds the rows then


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [[3, 0, 70, 1], [130, 300, 2], [1, 2]])
def test_rows_of_no_expert(dtype, sizes):
    """Rows in front of the first expert and behind the last, with NaN in them: zero in a fresh result, untouched in `out`, and
    nothing of them in any gradient, where a block of 64 rows or a tile reaches over them."""
    n, k, lead, behind = 136, 200, 37, 90
    x, w, off, dy, bias, ends = _case(sizes, n, k, dtype, 5, lead, behind)
    for t in (x, dy):
        t[:lead], t[ends[-1]:] = float("nan"), float("nan")
    out = ops.ragged_linear(x, w, off, bias, check=True)
    _check_rows(out, x, w, ends, bias)
    assert bool((out[:lead] == 0).all()) and bool((out[ends[-1]:] == 0).all())
    into = torch.full_like(out, 7.0)
    ops.ragged_linear(x, w, off, bias, out=into, check=True)
    assert torch.equal(into[lead:ends[-1]], out[lead:ends[-1]])
    assert bool((into[:lead] == 7).all()) and bool((into[ends[-1]:] == 7).all())
    dx, dw, db = ops.ragged_linear_backward(x, w, off, dy, bias=True, check=True)
    _check_grads(dx, dw, db, x, w, dy, ends)
    assert bool((dx[:lead] == 0).all()) and bool((dx[ends[-1]:] == 0).all())


def test_one_experts_nan_stays_with_it():
    sizes = [100, 30, 200, 64]
    x, w, off, dy, bias, ends = _case(sizes, 256, 128, torch.bfloat16, 8)
    clean = ops.ragged_linear(x, w, off, bias), *ops.ragged_linear_backward(x, w, off, dy, bias=True)
    x[ends[1]:ends[2]], dy[ends[1]:ends[2]] = float("inf"), float("nan")
    w[3] = float("nan")
    out, dx, dw, db = ops.ragged_linear(x, w, off, bias), *ops.ragged_linear_backward(x, w, off, dy, bias=True)
    for e in (0, 2):
        r = slice(ends[e], ends[e + 1])
        assert torch.equal(out[r], clean[0][r]) and torch.equal(dx[r], clean[1][r])
    for e in (0, 2, 3):
        assert torch.equal(dw[e], clean[2][e]) and torch.equal(db[e], clean[3][e])


@pytest.mark.parametrize("offsets,means", [([0, 50, 20, 120], [0, 50, 50, 120]), ([-5, 30, 1000, 40], [0, 30, 120, 120]), ([500] * 4, [120] * 4),
                                           ([-1] * 4, [0] * 4)])
def test_offsets_that_make_no_sense_stay_inside_the_tensors(offsets, means):
    x, w, _off, dy, bias, _ends = _case([40, 40, 40], 128, 64, torch.bfloat16, 9)
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    out = ops.ragged_linear(x, w, off, bias, check=True)
    _check_rows(out, x, w, means, bias)
    dx, dw, db = ops.ragged_linear_backward(x, w, off, dy, bias=True, check=True)
    _check_grads(dx, dw, db, x, w, dy, means)
    mine = torch.zeros(120, dtype=torch.bool, device="cuda")
    mine[means[0]:means[-1]] = True
    assert bool((out[~mine] == 0).all()) and bool((dx[~mine] == 0).all())


def test_autograd_and_kept_inputs():
    sizes, n, k = [30, 0, 77, 20], 256, 384
    x, w, off, dy, bias, ends = _case(sizes, n, k, torch.bfloat16, 10)
    res = torch.randn_like(dy)
    leaves = [t.clone().requires_grad_() for t in (x, w, bias, res)]
    out = ops.ragged_linear(leaves[0], leaves[1], off, leaves[2], residual=leaves[3])
    assert torch.equal(out.detach(), ops.ragged_linear(x, w, off, bias, residual=res))
    out.backward(dy)
    dx, dw, db = ops.ragged_linear_backward(x, w, off, dy, bias=True)
    assert torch.equal(leaves[0].grad, dx) and torch.equal(leaves[1].grad, dw) and torch.equal(leaves[2].grad, db) and torch.equal(leaves[3].grad, dy)
    # the weight gradient from the kept 8 bits: that of the values they stand for
    kept = x.clone().requires_grad_()
    weight = w.clone().requires_grad_()
    ops.ragged_linear(kept, weight, off, checkpoint=True).backward(dy)
    values = ops.restore_activation(*ops.checkpoint_activation(x))
    assert torch.equal(kept.grad, dx) and torch.equal(weight.grad, ops.ragged_linear_backward(values, w, off, dy)[1])
    frozen = x.clone().requires_grad_()
    ops.ragged_linear(frozen, w, off).backward(dy)
    assert torch.equal(frozen.grad, dx)
    with pytest.raises(RuntimeError, match="forward-only"):
        ops.ragged_linear(frozen, w, off, silu=True)


def test_gradients_against_differences():
    """fp16 inputs, the loss summed in 64 bits: linear in x and in w, so a step in a direction changes it by step * slope."""
    sizes, n, k = [20, 45], 64, 128
    x, w, off, dy, _bias, ends = _case(sizes, n, k, torch.float16, 12)
    dx, dw, _db = ops.ragged_linear_backward(x, w, off, dy)
    for moved, grad in ((x, dx), (w, dw)):
        before = ops.ragged_linear(x, w, off).double()
        d = (grad.double() * 0.02).half()
        saved = moved.clone()
        moved += d
        step = moved.double() - saved.double()
        change = ((ops.ragged_linear(x, w, off).double() - before) * dy.double()).sum()
        moved.copy_(saved)
        want = (grad.double() * step).sum()
        # every output is off by half a step of fp16 on both sides
        noise = 2 * 2.0 ** -11 * (before.abs() * dy.double().abs()).pow(2).sum().sqrt() * 4
        assert abs(float(change - want)) <= float(noise) + 2e-3 * abs(float(want))


def test_views_stream_graph_and_other_forms():
    sizes = [50, 0, 14]
    x, w, off, dy, bias, ends = _case(sizes, 128, 64, torch.bfloat16, 13)
    want = ops.ragged_linear(x, w, off, bias)
    pad = torch.zeros(64, 80, device="cuda", dtype=torch.bfloat16)
    pad[:, 3:67] = x
    strided = torch.zeros(3, 128, 2, 64, device="cuda", dtype=torch.bfloat16)
    strided[:, :, 1] = w
    off2 = torch.stack([off, off], 1)[:, 0]
    assert torch.equal(ops.ragged_linear(pad[:, 3:67], strided[:, :, 1], off2, bias.double()), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.ragged_linear(x, w, off, bias)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    # captured twice, replayed with other sizes in the same buffers
    graphs, results = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append((ops.ragged_linear(x, w, off, bias), *ops.ragged_linear_backward(x, w, off, dy, bias=True)))
        graphs.append(graph)
    off.copy_(torch.tensor([0, 1, 40, 64], dtype=torch.int32))
    for graph in reversed(graphs):
        graph.replay()
    plain = (ops.ragged_linear(x, w, off, bias), *ops.ragged_linear_backward(x, w, off, dy, bias=True))
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(r, plain))
    _check_rows(plain[0], x, w, [0, 1, 40, 64], bias)


def test_empty_and_refused():
    x, w, off, dy, bias, _ends = _case([0, 0], 64, 64, torch.bfloat16, 1)
    assert ops.ragged_linear(x, w, off, bias).shape == (0, 64)
    dx, dw, db = ops.ragged_linear_backward(x, w, off, dy, bias=True)
    assert dx.shape == (0, 64) and bool((dw == 0).all()) and bool((db == 0).all())
    x, w, off, dy, bias, _ends = _case([5, 3], 64, 64, torch.bfloat16, 1)
    none = ops.ragged_linear(x, w[:0], off[:1])
    assert bool((none == 0).all())
    with pytest.raises(ValueError, match="one dtype"):
        ops.ragged_linear(x, w.half(), off)
    with pytest.raises(RuntimeError, match="does not support dtype"):
        ops.ragged_linear(x.float(), w.float(), off)
    with pytest.raises(ValueError, match="same device|bias must be"):
        ops.ragged_linear(x, w, off, bias[:1])
    with pytest.raises(ValueError, match="residual must be"):
        ops.ragged_linear(x, w, off, residual=dy.float())
    with pytest.raises(RuntimeError, match="same device"):
        ops.ragged_linear(x, w, off.cpu())


@pytest.mark.parametrize("experts", [200, 1500])
def test_many_experts(experts):
    g = torch.Generator().manual_seed(experts)
    sizes = torch.randint(0, 4, (experts,), generator=g).tolist()
    x, w, off, dy, bias, ends = _case(sizes, 16, 24, torch.bfloat16, experts)
    index = torch.repeat_interleave(torch.arange(experts, device="cuda"), torch.tensor(sizes, device="cuda"))
    out = ops.ragged_linear(x, w, off, bias, check=True)
    z = torch.einsum("tk,tnk->tn", x.double(), w.double()[index]) + bias.double()[index]
    _within(out, z, _half(torch.bfloat16) * z.abs() + 1e-5)
    dx, dw, db = ops.ragged_linear_backward(x, w, off, dy, bias=True, check=True)
    want = torch.einsum("tn,tnk->tk", dy.double(), w.double()[index])
    _within(dx, want, _half(torch.bfloat16) * want.abs() + 1e-5)
    want = torch.zeros(experts, 16, 24, device="cuda", dtype=torch.float64).index_add_(0, index, dy.double()[:, :, None] * x.double()[:, None])
    _within(dw, want, _half(torch.bfloat16) * want.abs() + 1e-5)


def test_first_call_of_a_thread():
    """A thread that has not touched the GPU yet has no context of its own for the tensor maps."""
    import threading

    x, w, off, dy, bias, ends = _case([50, 14], 128, 64, torch.bfloat16, 13)
    want = ops.ragged_linear(x, w, off, bias)
    torch.cuda.synchronize()
    got = []
    thread = threading.Thread(target=lambda: got.append(ops.ragged_linear(x, w, off, bias)))
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert got and torch.equal(got[0], want)
