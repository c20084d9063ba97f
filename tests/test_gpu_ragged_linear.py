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
        we, ge = w[e].double(), dy[r].double()
        want = ge @ we
        _within(dx[r], want, _half(dtype) * want.abs() + _steps(n) * (ge.abs() @ we.abs()) + _tiny(dtype))
    _check_weights(dw, db, x, dy, ends)


def _check_weights(dw, db, x, dy, ends):
    dtype = dw.dtype
    for e in range(len(ends) - 1):
        r = slice(ends[e], ends[e + 1])
        xe, ge = x[r].double(), dy[r].double()
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


@pytest.mark.parametrize("sizes,n,k", [([3, 0, 70, 1], 136, 200), ([1500, 1500], 1024, 1024)])
def test_residual_of_rows_of_no_expert(sizes, n, k):
    """In a fresh result those rows are the residual's: what its gradient, the upstream one of every row, says too."""
    lead, behind = 37, 90
    x, w, off, dy, bias, ends = _case(sizes, n, k, torch.bfloat16, 15, lead, behind)
    res = torch.randn_like(dy).requires_grad_()
    out = ops.ragged_linear(x, w, off, bias, residual=res)
    _check_rows(out.detach(), x, w, ends, bias, False, res.detach())
    assert torch.equal(out[:lead], res[:lead]) and torch.equal(out[ends[-1]:], res[ends[-1]:])
    out.backward(dy)
    assert torch.equal(res.grad, dy)
    into = res.detach().clone()
    assert torch.equal(ops.ragged_linear(x, w, off, bias, residual=into, out=into), out)
    none = ops.ragged_linear(x, w[:0], off[:1], residual=res.detach())
    assert torch.equal(none, res)
    assert bool((ops.ragged_linear(x, w[:0], off[:1]) == 0).all())


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
    for taken in (x, w[0, :8]):                          # N = K = 64: they would fit
        with pytest.raises(ValueError, match="shares no memory"):
            ops.ragged_linear(x, w, off, out=taken)
    long = torch.zeros(16, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="shares no memory"):
        ops.ragged_linear(x, w, off, residual=long[:8], out=long[4:12])
    with pytest.raises(ValueError, match="out must be contiguous"):
        ops.ragged_linear(x, w, off, out=torch.zeros(8, 128, device="cuda", dtype=torch.bfloat16)[:, :64])


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


def test_offsets_past_32_bits():
    """2.2 * 10^9 outputs: the last expert's rows stand behind 2^32 bytes and 2^31 elements."""
    rows, n, k = 540_000, 4096, 64
    x = torch.zeros(rows, k, device="cuda", dtype=torch.bfloat16)
    g = torch.Generator(device="cuda").manual_seed(3)
    x[-300:] = torch.randn(300, k, generator=g, device="cuda").bfloat16()
    w = torch.randn(2, n, k, generator=g, device="cuda").bfloat16()
    ends = [0, rows - 200, rows]
    off = torch.tensor(ends, dtype=torch.int32, device="cuda")
    out = ops.ragged_linear(x, w, off, check=True)
    for e, r in ((0, slice(rows - 300, rows - 200)), (1, slice(rows - 200, rows))):
        want = x[r].double() @ w[e].double().T
        _within(out[r], want, _half(torch.bfloat16) * want.abs() + _steps(k) * (x[r].double().abs() @ w[e].double().abs().T) + 1e-9)
    assert bool((out[:1000] == 0).all())
    dx, dw, db = ops.ragged_linear_backward(x, w, off, out, bias=True, check=True)
    r = slice(rows - 200, rows)
    want = out[r].double() @ w[1].double()
    _within(dx[r], want, _half(torch.bfloat16) * want.abs() + _steps(n) * (out[r].double().abs() @ w[1].double().abs()) + 1e-9)
    want = out[r].double().T @ x[r].double()
    _within(dw[1], want, _half(torch.bfloat16) * want.abs() + _steps(200) * (out[r].double().abs().T @ x[r].double().abs()) + 1e-9)


@pytest.mark.parametrize("sizes", [[9000], [60, 60, 9000, 60], [1, 6000, 1, 1]])
def test_tiles_shared_by_pairs(sizes):
    """Few long tiles: their rows are cut between pairs and the partial sums joined, the bias gradient's among them."""
    x, w, off, dy, bias, ends = _case(sizes, 520, 264, torch.bfloat16, 21)
    dx, dw, db = ops.ragged_linear_backward(x, w, off, dy, bias=True, check=True)
    _check_grads(dx, dw, db, x, w, dy, ends)
    again = ops.ragged_linear_backward(x, w, off, dy, bias=True)
    assert all(torch.equal(a, b) for a, b in zip((dx, dw, db), again))


@pytest.mark.parametrize("sizes,n,k", [([1000, 900], 512, 512), ([2200, 0, 5, 4000], 136, 72), ([3000], 128, 256), ([0, 9000, 1], 264, 200), ([130, 3500, 64], 512, 128)])
@pytest.mark.parametrize("dtype", TYPES)
def test_weight_gradients_in_parts(sizes, n, k, dtype):
    """Few tiles with long contractions, a part of them for each CTA of a cluster of two, four or eight; some ranks have no rows."""
    x, w, off, dy, bias, ends = _case(sizes, n, k, dtype, 51, 3, 70)
    x[:3], x[-70:], dy[:3], dy[-70:] = float("nan"), float("inf"), float("nan"), float("nan")
    for biased in (True, False):
        _dx, dw, db = ops.ragged_linear_backward(x, w, off, dy, bias=biased, need_x=False, check=True)
        _check_weights(dw, db, x, dy, ends)
        again = ops.ragged_linear_backward(x, w, off, dy, bias=biased, need_x=False)
        assert torch.equal(dw, again[1]) and (not biased or torch.equal(db, again[2]))


def test_workspace_for_partial_tiles_only_where_pairs_share_them():
    from taac_2026_b200 import _lib

    size = _lib.load().tb200_ragged_wgrad_workspace_bytes
    assert size(8, 4096, 512, 512) < 1 << 23 <= size(1, 200000, 512, 512)


def test_parts_on_two_streams_and_in_a_graph():
    """Clusters, pairs and single CTAs, each with tensor memory of its own, beside one another on two streams and captured."""
    cases = [_case(sizes, n, k, torch.bfloat16, 60 + i) for i, (sizes, n, k) in enumerate([([3000], 128, 256), ([700] * 20, 512, 512), ([20000, 9000], 256, 256), ([9] * 30, 264, 520)])]
    run = lambda: [ops.ragged_linear_backward(x, w, off, dy, bias=True) for x, w, off, dy, _bias, _ends in cases]
    want = run()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    results = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for s, out in zip(streams, results):
            with torch.cuda.stream(s):
                out.append(run())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = run()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for got in results[0] + results[1] + [captured]:
        assert all(torch.equal(a, b) for case, right in zip(got, want) for a, b in zip(case, right))


EDGES = [1, 0, 31, 32, 33, 127, 128, 129, 255, 256, 257, 1500, 900]


@pytest.mark.parametrize("sizes,n,k", [(EDGES, 1000, 520), (EDGES, 1000, 512), ([5000, 0, 1, 3000, 4097, 70], 1000, 520), ([5000, 0, 1, 3000, 4097, 70], 1024, 512),
                                       ([17000, 60, 1], 520, 264), ([0, 1, 20000, 0], 264, 512), ([150, 151, 163] * 500, 512, 64), ([800, 790, 830] * 100, 136, 72)])
@pytest.mark.parametrize("dtype", TYPES)
def test_tiles_of_pairs(sizes, n, k, dtype):
    """Sizes at the edges of a tile, a quarter and a warp, experts without rows and many experts, in sums large enough for CTA pairs
    (the first two and the 1500 experts: rows and their gradients; the others: weight gradients)."""
    x, w, off, dy, bias, ends = _case(sizes, n, k, dtype, 41, 5, 3)
    _check_rows(ops.ragged_linear(x, w, off, bias, residual=dy, check=True), x, w, ends, bias, False, dy)
    _check_rows(ops.ragged_linear(x, w, off, bias, silu=True, check=True), x, w, ends, bias, True)
    dx, dw, db = ops.ragged_linear_backward(x, w, off, dy, bias=True, check=True)
    _check_grads(dx, dw, db, x, w, dy, ends)
    assert bool((dx[:5] == 0).all()) and bool((dx[-3:] == 0).all())


@pytest.mark.parametrize("sizes,n,k", [([3, 1, 0, 2], 512, 1024), ([30, 20], 256, 2048), ([60, 64, 65], 128, 4096), ([1], 2048, 1024), ([17] * 70, 136, 520)])
@pytest.mark.parametrize("dtype", TYPES)
def test_few_rows(sizes, n, k, dtype):
    """The kernel of few rows, with its contraction split over two and four CTAs and not at all, in both directions."""
    x, w, off, dy, bias, ends = _case(sizes, n, k, dtype, 31)
    _check_rows(ops.ragged_linear(x, w, off, bias, residual=dy, check=True), x, w, ends, bias, False, dy)
    _check_rows(ops.ragged_linear(x, w, off, bias, silu=True, check=True), x, w, ends, bias, True)
    dx, dw, db = ops.ragged_linear_backward(x, w, off, dy, bias=True, check=True)
    _check_grads(dx, dw, db, x, w, dy, ends)


def test_status_word_and_two_streams_at_once():
    """Two calls at once on two streams, with a persistent status word each."""
    cases = [_case([700, 300, 900], 520, 264, torch.bfloat16, s) for s in (41, 42)]
    wants = [(ops.ragged_linear(x, w, off, bias), *ops.ragged_linear_backward(x, w, off, dy, bias=True)) for x, w, off, dy, bias, _e in cases]
    words = [torch.zeros(1, dtype=torch.int32, device="cuda") for _ in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(3):
        for i, (x, w, off, dy, bias, _e) in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i] = (ops.ragged_linear(x, w, off, bias, status=words[i]), *ops.ragged_linear_backward(x, w, off, dy, bias=True, status=words[i]))
    torch.cuda.synchronize()
    assert all(int(v) == 0 for v in words)
    for g, want in zip(got, wants):
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_feed_forward_layer_as_a_training_step_uses_it():
    """Residual norm, up projections by expert, gated activation kept in 8 bits, down projections, against the same chain in 64 bits
    with the kept values in the backward pass's places: the loss's gradients of every weight."""
    sizes, d, hidden = [40, 0, 100, 20], 256, 384
    total_rows = sum(sizes)
    g = torch.Generator(device="cuda").manual_seed(50)
    make = lambda *s, k=1.0: torch.randn(*s, generator=g, device="cuda") * k  # noqa: E731
    x, r = make(total_rows, d).bfloat16(), make(total_rows, d).bfloat16()
    gamma = (1 + 0.1 * make(d)).bfloat16()
    w_up, w_down = make(4, 2 * hidden, d, k=d ** -0.5).bfloat16(), make(4, d, hidden, k=hidden ** -0.5).bfloat16()
    b_up, b_down = make(4, 2 * hidden, k=0.1), make(4, d, k=0.1)
    dy = make(total_rows, d).bfloat16()
    off = torch.tensor([0, 40, 40, 140, 160], dtype=torch.int32, device="cuda")
    leaves = [t.clone().requires_grad_() for t in (x, r, gamma, w_up, b_up, w_down, b_down)]
    t, n = ops.add_rms_norm(leaves[0], leaves[1], leaves[2])
    u = ops.ragged_linear(n, leaves[3], off, leaves[4], checkpoint=True)
    h = ops.silu_gate(u)
    y = ops.ragged_linear(h, leaves[5], off, leaves[6], residual=t)
    y.backward(dy)
    assert torch.equal(leaves[0].grad, leaves[1].grad)

    ref = [v.double().requires_grad_() for v in (x, r, gamma, w_up, b_up, w_down, b_down)]
    td = ref[0] + ref[1]
    nd = td * torch.rsqrt(td.pow(2).mean(-1, keepdim=True) + 1e-6) * ref[2]
    index = torch.repeat_interleave(torch.arange(4, device="cuda"), torch.tensor(sizes, device="cuda"))
    ud = torch.einsum("tk,tnk->tn", nd, ref[3][index]) + ref[4][index]
    hd = torch.nn.functional.silu(ud[:, :hidden]) * ud[:, hidden:]
    yd = torch.einsum("tk,tnk->tn", hd, ref[5][index]) + ref[6][index] + td
    yd.backward(dy.double())
    # roundings of bf16 (2^-8 each, four in a row forward, five back) and of e4m3 in the kept values (2^-4), as independent
    # errors: in the 2-norm below 2^-4 / sqrt(3) * 1.5 for what passes the kept values, 10 * 2^-9 for the result
    rel = lambda a, b: float((a.double() - b).norm() / b.norm())  # noqa: E731
    assert rel(y.detach(), yd.detach()) <= 10 * 2.0 ** -9
    for got, want in zip(leaves, ref):
        assert got.grad is not None and rel(got.grad, want.grad) <= 1.5 * 2.0 ** -4 / 3 ** 0.5
    # an expert without rows has zero gradients
    for i in (3, 4, 5, 6):
        assert bool((leaves[i].grad[1] == 0).all())


def test_served_in_8_bits():
    """The same layer as it is served: quantised residual norm -> e4m3 gated feed-forward layer with the sum as residual."""
    g = torch.Generator(device="cuda").manual_seed(51)
    x, r = (torch.randn(200, 512, generator=g, device="cuda").bfloat16() for _ in range(2))
    gamma = torch.ones(512, device="cuda", dtype=torch.bfloat16)
    w_up, w_down = (torch.randn(n, 512, generator=g, device="cuda") * 512 ** -0.5 for n in (1024, 512))
    weights = ops.Fp8FfnWeights(w_up, w_down, gated=True)
    total, q, scales = ops.add_rms_norm_quant(x, r, gamma)
    h, sh = ops.fp8_gemm(q, scales, weights.w_up, weights.s_up, mode="swiglu", check=True)
    got = ops.fp8_gemm(h, sh, weights.w_down, weights.s_down, mode="linear", residual=total, check=True)
    n = _norm64(x.double() + r.double())
    gate, value = (n @ w_up.double().T).chunk(2, -1)
    want = (torch.nn.functional.silu(gate) * value) @ w_down.double().T
    # Four e4m3 roundings, each at most 2^-4 of a value and as good as independent: 2^-4 / sqrt(3) = 0.036 in the 2-norm.  Rows and
    # weights give gate and value 0.051 each, their product 0.072; with the hidden values' and the second weights' own it is 0.088.
    # (Two such chains whose inputs differ by 2^-9 differ by a good part of that: a value that crosses a border of the
    # first rounding moves hidden values over borders of the next, so they are not compared with each other.)
    rel = float((got.double() - total.double() - want).norm() / want.norm())
    assert rel <= 0.088


def _norm64(t):
    return t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + 1e-6)


def test_status_word_under_autograd():
    """The caller's word and check=True serve the backward pass as well, with the same gradients."""
    x, w, off, dy, bias, _ends = _case([700, 0, 300], 264, 136, torch.bfloat16, 61)
    want = ops.ragged_linear_backward(x, w, off, dy, bias=True)
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    for kw in ({"status": word}, {"check": True}, {"status": word, "check": True}):
        leaves = [t.clone().requires_grad_() for t in (x, w, bias)]
        ops.ragged_linear(leaves[0], leaves[1], off, leaves[2], **kw).backward(dy)
        assert all(torch.equal(leaf.grad, v) for leaf, v in zip(leaves, want)) and int(word) == 0
