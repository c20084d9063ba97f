"""Every way in which the weight gradients of ragged layers are shared out, each at sizes that the rule sends there: single CTAs or clusters
on 128 x 128 tiles, or CTA pairs on 256 x 256 tiles, with whole tiles round robin, some rounds of them and the rest cut, all tiles cut, or
no workspace for cut tiles at all; with tensor maps in chunks (N and K multiples of 64) and without, with and without a bias gradient.

The rule is restated below, so that a change of it that moves a size elsewhere is noticed."""
from __future__ import annotations

import pytest
import torch

from conftest import gpu_ready
from taac_2026_b200 import _lib, ops
from test_gpu_ragged_linear import _case, _check_weights

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _need_gpu():
    if not gpu_ready():
        pytest.fail("gpu tests need an sm_100 device and a built libtb200.so")


def _up(a, b):
    return -(-a // b)


def _pairs():
    return torch.cuda.get_device_properties(0).multi_processor_count // 2


def _few(experts, rows, n, k):
    """0: pairs of CTAs; else how many CTAs share a 128 x 128 tile.  Expected times, in hundredths of a microsecond."""
    pairs, here = _pairs(), 4 * _pairs()
    if rows > 1 << 26:
        return 0
    blocks = _up(rows // experts, 64)
    small, large = (experts * _up(n, t) * _up(k, t) for t in (128, 256))
    split = next((s for s in (8, 4, 2) if s * small <= here and blocks >= 4 * s and blocks >= 12), 1)
    few = (900 if split > 1 else 600) + 65 * _up(small * split, here) * max(_up(blocks, split), 5)
    length = max(blocks, 7)
    whole = 1200 + 53 * _up(large, pairs) * length
    shared = 1500 + 45 * pairs // large + 53 * large * length // pairs
    return split if few < min(whole, shared) else 0


def _plan(sizes, rows, n, k):
    split = _few(len(sizes), rows, n, k)
    if split:
        return "clusters" if split > 1 else "single"
    if rows < 512:
        return "never shared"
    pairs, tiles = _pairs(), _up(n, 256) * _up(k, 256)
    lengths = [max(6, _up(s, 64)) for s in sizes]
    share = sum(lengths) * tiles // pairs
    width = share // 32 + 1
    line = sorted(lengths, key=lambda b: 32 if b > share else 31 - (b - 1) // width)      # the longest first, those beyond a share last
    shorter = sum(b <= share for b in lengths)
    span = sum(line[w * pairs // tiles] for w in range(_up(len(line) * tiles, pairs)))
    if shorter == len(line) and 2 * span <= 3 * share + 48:
        return "whole"
    waves = reached = 0
    while waves < shorter * tiles // pairs and reached + line[waves * pairs // tiles] + width <= share:
        reached += line[waves * pairs // tiles] + width
        waves += 1
    return "rounds and cut" if waves else "cut"


CASES = [
    ("single", [300, 0, 64, 65, 1, 700], 264, 520), ("single", [128] * 30 + [0, 5], 512, 512),
    ("clusters", [2000, 0, 1903], 264, 520), ("clusters", [4000], 256, 128),
    ("whole", [0] + [2300] * 7 + [1] + [2000] * 6 + [0], 1024, 512), ("whole", [0] + [2900] * 4 + [63] + [2901] * 3, 2040, 1032),
    ("rounds and cut", [900] * 30 + [0, 1] + [897] * 30 + [30001], 512, 512), ("rounds and cut", [2000] * 24 + [0, 14000, 14033], 1000, 520),
    ("cut", [5000, 0, 1, 3000, 4097, 70], 1024, 512), ("cut", [40009], 264, 520), ("cut", [0, 130, 30000, 0], 520, 520),
    ("never shared", [500], 8192, 4608), ("never shared", [497], 6152, 6152),
]


@pytest.mark.parametrize("biased", [True, False])
@pytest.mark.parametrize("plan,sizes,n,k", CASES)
def test_every_plan(plan, sizes, n, k, biased):
    """NaN in the rows of no expert on both sides: a last block or a tile that reaches over them takes nothing of them."""
    rows, lead, behind = sum(sizes), 3, 2
    assert _plan(sizes, rows + lead + behind, n, k) == plan
    dtype = torch.bfloat16 if len(sizes) % 2 else torch.float16
    x, w, off, dy, _bias, ends = _case(sizes, n, k, dtype, rows + n, lead, behind)
    for t in (x, dy):
        t[:lead], t[ends[-1]:] = float("nan"), float("inf")
    _dx, dw, db = ops.ragged_linear_backward(x, w, off, dy, bias=biased, need_x=False, check=True)
    assert (db is not None) == biased
    _check_weights(dw, db, x, dy, ends)
    for e, s in enumerate(sizes):
        if s == 0:
            assert bool((dw[e] == 0).all()) and (db is None or bool((db[e] == 0).all()))
    again = ops.ragged_linear_backward(x, w, off, dy, bias=biased, need_x=False)
    assert torch.equal(dw, again[1]) and (not biased or torch.equal(db, again[2]))


def test_the_rule_is_the_one_stated_here():
    """Calls that pairs serve ask for a workspace of partial tiles, the others do not."""
    lib = _lib.load()
    seen = set()
    for experts in (1, 2, 5, 16, 60, 300):
        for rows in (512, 700, 3000, 12168, 33000, 100000, 400000):
            for n, k in ((64, 64), (128, 256), (264, 520), (512, 512), (1000, 520), (2048, 512), (2048, 2048), (8192, 4608)):
                pairs = _few(experts, rows, n, k) == 0
                assert (lib.tb200_ragged_wgrad_workspace_of(experts, rows, n, k, 1) > 0) == pairs, (experts, rows, n, k)
                seen.add(pairs)
    assert seen == {True, False}


def test_the_longest_chain_is_shared():
    """300 experts, one of them with 270 million rows: one CTA's chain of 4.2 million blocks would outlast its bounded waits (2.2 s), so
    pairs share it.  The values are 1, 0 and -1, every 2^20th row: fp32 sums them without rounding."""
    experts, long, n, k = 300, 270_000_000, 8, 8
    rows = long + experts - 1
    assert _few(experts, rows, n, k) == 0
    x, dy = (torch.zeros(rows, c, device="cuda", dtype=torch.bfloat16) for c in (k, n))
    g = torch.Generator(device="cuda").manual_seed(1)
    for t in (x, dy):
        some = t[::1 << 20]
        some.copy_(torch.randint(-1, 2, some.shape, generator=g, device="cuda"))
        t[long:] = torch.randint(-1, 2, t[long:].shape, generator=g, device="cuda").bfloat16()
    off = torch.cat([torch.zeros(1, dtype=torch.int32), torch.arange(long, rows + 1, dtype=torch.int32)]).cuda()
    w = torch.zeros(experts, n, k, device="cuda", dtype=torch.bfloat16)
    _dx, dw, db = ops.ragged_linear_backward(x, w, off, dy, bias=True, need_x=False, check=True)
    xs, ds = x[:long:1 << 20].double(), dy[:long:1 << 20].double()
    assert torch.equal(dw[0].double(), ds.T @ xs) and torch.equal(db[0].double(), ds.sum(0))
    want = dy[long:].double()[:, :, None] * x[long:].double()[:, None]
    assert torch.equal(dw[1:].double(), want) and torch.equal(db[1:].double(), dy[long:].double())


def test_two_pair_plans_at_once():
    """Pairs with cut tiles and with whole ones, and single CTAs, beside one another on two streams and captured: a workspace each."""
    cases = [_case(sizes, n, k, torch.bfloat16, 70 + i) for i, (sizes, n, k) in enumerate(
        [([5000, 0, 1, 3000, 4097, 70], 1024, 512), ([0] + [2300] * 7 + [1] + [2000] * 6 + [0], 1024, 512), ([300, 0, 64, 65, 1, 700], 264, 520)])]
    assert [_plan([b - a for a, b in zip(c[5], c[5][1:])], len(c[0]), c[1].shape[1], c[1].shape[2]) for c in cases] == ["cut", "whole", "single"]
    run = lambda: [ops.ragged_linear_backward(x, w, off, dy, bias=True) for x, w, off, dy, _bias, _ends in cases]  # noqa: E731
    want = run()
    streams, results = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, out in zip(streams, results):
            with torch.cuda.stream(s):
                out.append(run())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for got in results[0] + results[1] + [captured]:
        assert all(torch.equal(a, b) for case, right in zip(got, want) for a, b in zip(case, right))
