"""The grouped products in every form that their rule chooses, by name: large tiles and small ones, with
and without rows, half row tiles, several segments of rows' offsets, split contractions."""

import ctypes

import numpy as np
import pytest
import torch

from hi2_amd import _lib
from hi2_amd.experts import grouped_linear
from test_gpu_grouped import check, oracle, rounded, routing, run_case, sums, values

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}

# (n, k, counts): 256-tiles for the product, the tokens' gradient and the weights'.  Some expert has more
# than 4096 slots, some none, some last row tiles 128 rows or fewer, some more.
ODD = (1100, 1300, [9000, 0, 5000, 3, 12000, 130, 7867, 6000])  # rows are copied
EVEN = (512, 512, [0, 9001, 4096, 4097, 100, 128, 129] + [24] * 40 + [313])
LARGE = [ODD, EVEN]


def form(what, e, n, k, slots, dtype=2):
    splits = ctypes.c_int64(-1)
    side = _lib.lib().hi2x_grouped_form(what, dtype, e, n, k, slots, ctypes.byref(splits))
    return side, splits.value


def test_forms_by_size():
    """On the host: what the shapes of the tests below take."""
    for n, k, counts in LARGE:
        for what in range(3):
            assert form(what, len(counts), n, k, sum(counts)) == (256, 1), (n, k, what)
    assert form(0, 8, 1024, 2048, 32)[0] == 16 and form(0, 8, 1024, 2048, 33)[0] == 128
    assert form(0, 8, 1024, 2047, 256)[0] == 16 and form(0, 8, 1024, 2047, 257)[0] == 128
    assert form(0, 8, 1024, 2048, 1, dtype=0) == (64, 1)
    assert form(1, 2, 4096, 130, 130)[1] > 1  # a split contraction
    assert _lib.lib().hi2x_grouped_form(3, 2, 1, 1, 1, 1, None) == -1
    assert _lib.lib().hi2x_grouped_form(0, 3, 1, 1, 1, 1, None) == -1
    assert _lib.lib().hi2x_grouped_form(0, 2, 0, 1, 1, 1, None) == -1
    assert _lib.lib().hi2x_grouped_form(0, 2, 1, 1, 1, 1, None) == 16


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("case", LARGE, ids=["odd", "even"])
def test_large_tiles(dev, dtype, gather, case):
    n, k, counts = case
    s = sum(counts)
    assert [form(w, len(counts), n, k, s)[0] for w in range(3)] == [256] * 3
    run_case(TYPES[dtype], len(counts), n, k, counts, s // 4 if gather else s, 4 if gather else 1,
             gather, seed=21)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("case", LARGE, ids=["odd", "even"])
def test_large_tiles_with_gaps_and_bad_rows(dev, dtype, case):
    """Slots of no expert before and behind the ranges hold what they like; a row outside x makes its
    slot's row NaN and its expert's gradient, and leaves every other bit."""
    t = TYPES[dtype]
    n, k, counts = case
    e, s, tokens = len(counts), sum(counts), sum(counts) // 4
    offs, rows, slots = routing(counts, tokens, 4, 7)
    x, w = values((tokens, k), t, 1), values((e, n, k), t, 2, 0.05)
    dy = values((s, n), t, 3, 0.1)
    # 70 slots in front, 300 behind
    nan = torch.full((300, n), float("nan"), dtype=t, device="cuda")
    dy_gaps = torch.cat([nan[:70], dy, nan])
    rows_gaps = torch.cat([torch.full((70,), -3, device="cuda"), rows,
                           torch.full((300,), tokens + 5, device="cuda")])
    assert [form(q, e, n, k, s + 370)[0] for q in range(3)] == [256] * 3

    def run(rows, offs, dy):
        wr = w.clone().requires_grad_(True)
        y = grouped_linear(x, wr, offs, rows)
        return y.detach(), torch.autograd.grad(y, wr, dy)[0]

    y, dw = run(rows, offs, dy)
    yg, dwg = run(rows_gaps, offs + 70, dy_gaps)
    assert torch.equal(yg[70:70 + s], y) and not yg[:70].any() and not yg[70 + s:].any()
    assert torch.equal(dwg, dw) and not dw[[c == 0 for c in counts]].any()
    hit = int(np.argmax(counts))
    bad = int(offs[hit]) + counts[hit] - 3
    rows2 = rows.clone()
    rows2[bad] = tokens
    y2, dw2 = run(rows2, offs, dy)
    keep = torch.arange(s, device="cuda") != bad
    assert torch.isnan(y2[bad]).all() and torch.equal(y2[keep], y[keep])
    others = [i for i in range(e) if i != hit]
    assert torch.isnan(dw2[hit]).all() and torch.equal(dw2[others], dw[others])
    # the tokens' gradient of slots behind the ranges is zero
    xs = values((s + 370, k), t, 5).requires_grad_(True)
    dx, = torch.autograd.grad(grouped_linear(xs, w, offs + 70), xs, dy_gaps)
    assert not dx[:70].any() and not dx[70 + s:].any() and torch.isfinite(dx).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_large_tiles_of_strided_rows(dev, dtype):
    """Rows apart at multiples of 16 bytes are read as they lie; what lies between them is not."""
    t = TYPES[dtype]
    n, k, counts = EVEN
    offs = torch.from_numpy(np.concatenate([[0], np.cumsum(counts)])).cuda()
    s = sum(counts)
    wide = torch.full((s, k + 16), float("nan"), dtype=t, device="cuda")
    dwide = torch.full((s, n + 24), float("inf"), dtype=t, device="cuda")
    x, dy = wide[:, 8:8 + k], dwide[:, 16:16 + n]
    x.copy_(values((s, k), t, 1)), dy.copy_(values((s, n), t, 2, 0.1))
    w = values((len(counts), n, k), t, 3, 0.05)
    out = []
    for a, d in ((x, dy), (x.contiguous(), dy.contiguous())):
        ar, wr = a.detach().requires_grad_(True), w.clone().requires_grad_(True)
        y = grouped_linear(ar, wr, offs)
        out.append((y.detach(), *torch.autograd.grad(y, (ar, wr), d)))
    assert all(torch.equal(a, b) for a, b in zip(*out))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_large_tiles_captured(dev, dtype):
    """Replays over other ranges, with eager work in between, give what eager calls give."""
    t = TYPES[dtype]
    n, k, counts = EVEN
    s, e = sum(counts), len(counts)
    offs, rows, slots = routing(counts, s // 4, 4, 1)
    x = values((s // 4, k), t, 1).requires_grad_(True)
    w = values((e, n, k), t, 2, 0.05).requires_grad_(True)
    dy = values((s, n), t, 3, 0.1)

    def step():
        y = grouped_linear(x, w, offs, rows, slots)
        return [y.detach(), *torch.autograd.grad(y, (x, w), dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(3):
        more = counts[i:] + counts[:i]
        with torch.no_grad():
            for to, v in zip((offs, rows, slots), routing(more, s // 4, 4, 30 + i)):
                to.copy_(v)
            x.copy_(values((s // 4, k), t, 40 + i))
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in outs]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("counts", [[2, 5], [60, 70], EVEN[2]], ids=["few", "small", "large"])
def test_subnormal_values(dev, dtype, counts):
    """Subnormal values of the types are multiplied as they are: by one and by zeros they stay."""
    t = TYPES[dtype]
    k, s, e = 512, sum(counts), len(counts)
    offs = torch.from_numpy(np.concatenate([[0], np.cumsum(counts)])).cuda()
    f = torch.finfo(t)
    g = torch.Generator().manual_seed(1)
    whole = torch.randint(-100, 101, (s, k), generator=g).double()
    x = (whole * (f.tiny * f.eps)).to(t).cuda().requires_grad_(True)
    w = torch.eye(k).expand(e, k, k).contiguous().to(t).cuda()
    y = grouped_linear(x, w, offs)
    assert torch.equal(y, x)
    dx, = torch.autograd.grad(y, x, x.detach().flip(0).contiguous())
    assert torch.equal(dx, x.detach().flip(0))
    assert bool(y.any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_one_expert_takes_most_slots(dev, dtype):
    """A routing far from even: the rule goes by the mean, the results by the ranges."""
    t = TYPES[dtype]
    counts = [30, 20000, 0, 7] + [5] * 12
    n, k = 256, 520
    offs, rows, slots = routing(counts, sum(counts), 1, 3)
    x, w = values((sum(counts), k), t, 1), values((len(counts), n, k), t, 2, 0.05)
    dy = values((sum(counts), n), t, 3, 0.1)
    xr, wr = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = grouped_linear(xr, wr, offs, rows, slots)
    dx, dw = torch.autograd.grad(y, (xr, wr), dy)
    y0, ym, d0, dm, dw0, dwm = oracle(x, w, offs, rows, slots, dy)
    check(y, y0, rounded(y0, sums(ym, k), t))
    check(dx, d0[slots[:, 0]], rounded(d0, sums(dm, n), t)[slots[:, 0]])
    check(dw, dw0, rounded(dw0, sums(dwm, max(counts)), t))
