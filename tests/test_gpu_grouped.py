"""The products grouped by expert and their gradients, the gated activation, and the MLP of experts
made of them, against the same in 64 bits."""

import numpy as np
import pytest
import torch

from hi2_amd.experts import experts_mlp, gated, grouped_linear
from hi2_amd.moe import route

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def half_step(dtype):
    """A rounding's largest relative error, and a subnormal's absolute one."""
    f = torch.finfo(dtype)
    return f.eps / 2, f.tiny * f.eps / 2


def rounded(value, bound, dtype, scale=1.0):
    """How far a float32 sum that is off by `bound` may be off once rounded to dtype."""
    rel, least = half_step(dtype)
    return bound * (1 + rel) + rel * value.abs() * scale + least


def sums(magnitude, length):
    """A float32 sum of `length` products: each of the additions rounds (by up to a whole step, as
    the matrix unit may cut instead of round) a partial sum no larger than `magnitude`."""
    return (length + 8) * 2.0 ** -23 * magnitude


def check(got, want, bound):
    off = (got.double() - want).abs()
    assert torch.isfinite(got.double()).all()
    assert bool((off <= bound).all()), float((off / bound.clamp_min(1e-300)).max())


def routing(counts, tokens, top_k, seed):
    """(offs, rows, slots) of slots that are dealt to experts by counts: slot j's token is any, each
    (token, choice) has one slot."""
    rng = np.random.default_rng(seed)
    offs = np.concatenate([[0], np.cumsum(counts)])
    order = rng.permutation(tokens * top_k)
    assert offs[-1] == tokens * top_k
    slots = np.empty(tokens * top_k, np.int64)
    slots[order] = np.arange(tokens * top_k)
    return [torch.from_numpy(np.ascontiguousarray(v)).cuda() for v in
            (offs, order // top_k, slots.reshape(tokens, top_k))]


def values(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(shape, generator=g)).to(dtype).cuda()


def oracle(x, w, offs, rows, slots, dy):
    """y, dx and dw and what bounds their sums, in 64 bits."""
    x, w, dy = x.double(), w.double(), dy.double()
    e, n, k = w.shape
    s = dy.shape[0]
    src = torch.arange(s, device=x.device) if rows is None else rows
    y, dw = x.new_zeros(s, n), x.new_zeros(e, n, k)
    ym, dwm = torch.zeros_like(y), torch.zeros_like(dw)
    d, dm = x.new_zeros(s, k), x.new_zeros(s, k)
    o = offs.tolist()
    for i in range(e):
        at = slice(o[i], o[i + 1])
        a = x[src[at]]
        y[at], ym[at] = a @ w[i].T, a.abs() @ w[i].abs().T
        d[at], dm[at] = dy[at] @ w[i], dy[at].abs() @ w[i].abs()
        dw[i], dwm[i] = dy[at].T @ a, dy[at].abs().T @ a.abs()
    return y, ym, d, dm, dw, dwm


def run_case(dtype, e, n, k, counts, tokens, top_k, gather, seed=0):
    if gather:
        offs, rows, slots = routing(counts, tokens, top_k, seed)
        x = values((tokens, k), dtype, seed + 1)
    else:
        offs = torch.from_numpy(np.concatenate([[0], np.cumsum(counts)])).cuda()
        rows = slots = None
        x = values((int(sum(counts)), k), dtype, seed + 1)
    w = values((e, n, k), dtype, seed + 2, 0.05)
    dy = values((int(sum(counts)), n), dtype, seed + 3, 0.1)
    xr, wr = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = grouped_linear(xr, wr, offs, rows, slots)
    dx, dw = torch.autograd.grad(y, (xr, wr), dy)
    assert y.dtype == dx.dtype == dw.dtype == dtype and dx.shape == x.shape
    with torch.no_grad():
        assert torch.equal(grouped_linear(x, w, offs, rows), y)
    y0, ym, d0, dm, dw0, dwm = oracle(x, w, offs, rows, slots, dy)
    check(y, y0, rounded(y0, sums(ym, k), dtype))
    length = max(counts) if len(counts) else 0
    check(dw, dw0, rounded(dw0, sums(dwm, length), dtype))
    bound = sums(dm, n)
    if slots is None:
        check(dx, d0, rounded(d0, bound, dtype))
    else:
        # each slot's row is rounded, then their sum in float32, then the result
        each = rounded(d0, bound, dtype)
        want, mag = d0[slots].sum(1), d0.abs()[slots].sum(1)
        check(dx, want, rounded(want, each[slots].sum(1) + sums(mag, slots.shape[1]), dtype))


SHAPES = [
    # (experts, n, k, counts, tokens, top_k, gather)
    (1, 1, 1, [1], 1, 1, True),
    (1, 64, 64, [3], 3, 1, False),
    (4, 64, 128, [0, 5, 0, 3], 4, 2, True),
    (4, 96, 40, [0, 0, 0, 0], 0, 1, True),
    (3, 33, 17, [7, 0, 2], 9, 1, True),
    (5, 130, 70, [1, 64, 65, 0, 30], 40, 4, True),
    (2, 256, 512, [300, 212], 256, 2, True),
    (2, 264, 520, [257, 15], 272, 1, False),
    (8, 128, 256, [16, 17, 1, 0, 2, 15, 33, 44], 16, 8, True),
    (3, 300, 1000, [128, 1, 129], 129, 2, True),
    (2, 513, 385, [500, 11], 511, 1, False),
    (70, 72, 88, [i % 5 for i in range(70)], 140, 1, True),
]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("case", SHAPES, ids=lambda c: f"{c[0]}x{c[1]}x{c[2]}_{c[4]}t{c[5]}")
def test_products_and_gradients(dev, dtype, case):
    run_case(TYPES[dtype], *case)


FEW = [
    # (experts, n, k, counts, tokens, top_k, gather): a few slots, odd sizes, more slots of odd ones
    (64, 128, 256, [1 if i % 8 == 3 else 0 for i in range(64)], 1, 8, True),
    (3, 40, 2048, [0, 17, 0], 17, 1, True),
    (2, 17, 1000, [16, 15], 31, 1, False),
    (130, 24, 72, [1 if i > 120 else 0 for i in range(130)], 9, 1, True),
    (4, 100, 1003, [33, 0, 100, 1], 67, 2, True),
    (2, 999, 77, [3, 29], 8, 4, True),
    (600, 24, 40, [1 if i % 100 == 7 else 0 for i in range(600)], 6, 1, True),
]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("case", FEW, ids=lambda c: f"{c[0]}x{c[1]}x{c[2]}_{c[4]}t{c[5]}")
def test_few_slots(dev, dtype, case):
    run_case(TYPES[dtype], *case, seed=3)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("n,k,counts", [
    (1024, 4096, [3, 60, 5, 0]), (2048, 512, [130, 600, 2]), (512, 256, [5000, 0, 9100, 17]),
    (257, 2050, [700, 40]), (4096, 96, [1, 300, 64, 1000]),
])
def test_every_tile_form(dev, dtype, n, k, counts):
    """Shapes that take 256-tiles, 128-tiles and, for the weights' gradient, several segments of
    rows' offsets."""
    run_case(TYPES[dtype], len(counts), n, k, counts, sum(counts), 1, True, seed=9)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_large_ragged(dev, dtype):
    counts = [1500, 0, 700, 3, 1, 890, 257, 745]
    run_case(TYPES[dtype], 8, 768, 1024, counts, sum(counts) // 4, 4, True, seed=5)


LONG = [
    # (experts, n, k, counts, tokens, top_k, gather): few tiles, a long contraction of the product,
    # of the input's gradient or of the weights'
    (1, 256, 8192, [100], 50, 2, True),
    (3, 136, 5000, [130, 0, 1], 131, 1, True),
    (4, 130, 4100, [64, 1, 0, 63], 128, 1, False),
    (2, 9000, 200, [33, 97], 65, 2, True),
    (4, 128, 264, [9000, 0, 33, 3167], 6100, 2, True),
    (2, 70, 130, [7001, 8], 7009, 1, False),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("case", LONG, ids=lambda c: f"{c[0]}x{c[1]}x{c[2]}_{c[4]}t{c[5]}")
def test_long_contractions_of_few_tiles(dev, dtype, case):
    run_case(TYPES[dtype], *case, seed=13)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_long_contractions_with_gaps_and_bad_rows(dev, dtype):
    """Slots of no expert, rows outside and experts without slots where contractions are split, and
    the same bits each time."""
    t = TYPES[dtype]
    n, k = 160, 4096
    offs = torch.tensor([7, 47, 47, 6047, 6048]).cuda()
    g = torch.Generator().manual_seed(2)
    rows = torch.randint(0, 500, (6100,), generator=g).cuda()
    x, w = values((500, k), t, 1, 0.1), values((4, n, k), t, 2, 0.1)
    dy = values((6100, n), t, 3, 0.1)
    dy[:7] = float("nan")
    dy[6048:] = float("inf")
    rows[:7] = -5
    few = torch.tensor([7, 27, 27, 126, 127]).cuda()
    for at, slots in ((offs, 6100), (few, 140)):
        for bad in (None, 20):
            r = rows[:slots].clone()
            if bad is not None:
                r[bad] = 500
            wr = w.clone().requires_grad_(True)
            y = grouped_linear(x, wr, at, r)
            dw, = torch.autograd.grad(y, wr, dy[:slots])
            o = at.tolist()
            assert not y[:o[0]].any() and not y[o[-1]:].any() and not dw[1].any()
            nan = torch.isnan(y).any(1)
            assert nan.nonzero().flatten().tolist() == ([] if bad is None else [bad])
            assert bool(torch.isnan(dw[0]).all()) == (bad is not None)
            assert torch.isfinite(dw[2:]).all()
            keep = ~nan
            # (the oracle without the slots that no expert has)
            inner, d = r.clamp(0, 499)[o[0]:o[-1]], dy[o[0]:o[-1]]
            y0, ym, _, _, dw0, dwm = oracle(x, w, at - o[0], inner, None, d)
            pick = keep[o[0]:o[-1]]
            check(y[o[0]:o[-1]][pick], y0[pick], rounded(y0, sums(ym, k), t)[pick])
            check(dw[2:], dw0[2:], rounded(dw0, sums(dwm, 6000), t)[2:])
            again = grouped_linear(x, wr, at, r)
            assert torch.equal(again[keep], y[keep])
            assert torch.equal(torch.autograd.grad(again, wr, dy[:slots])[0][2:], dw[2:])
    # the input's gradient over a long contraction, with gaps
    w2 = values((4, k, n), t, 4, 0.1)
    xr = values((140, n), t, 5).requires_grad_(True)
    d = values((140, k), t, 6, 0.1)
    d[:7] = float("nan")
    d[127:] = float("nan")
    dx, = torch.autograd.grad(grouped_linear(xr, w2, few), xr, d)
    assert not dx[:7].any() and not dx[127:].any()
    _, _, d0, dm, _, _ = oracle(xr.detach()[7:127], w2, few - 7, None, None, d[7:127])
    check(dx[7:127], d0, rounded(d0, sums(dm, k), t))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_strides_and_alignment(dev, dtype):
    """Rows that begin anywhere give what contiguous ones do, bit for bit."""
    t = TYPES[dtype]
    offs = torch.tensor([0, 40, 40, 101]).cuda()
    wide, dwide = values((101, 300), t, 1), values((101, 200), t, 2)
    w = values((3, 72, 96), t, 3)
    base = values((3 * 72 * 96 + 8,), t, 4)
    for ox, ow, od in ((0, 0, 0), (1, 0, 1), (8, 1, 3), (5, 3, 8)):
        x, dy = wide[:, ox:ox + 96], dwide[:, od:od + 72]
        base[ow:ow + w.numel()] = w.reshape(-1)
        v = base[ow:ow + w.numel()].view(3, 72, 96)
        xr, vr = x.detach().requires_grad_(True), v.detach().requires_grad_(True)
        y = grouped_linear(xr, vr, offs)
        dx, dw = torch.autograd.grad(y, (xr, vr), dy)
        xc, wc = x.detach().clone().requires_grad_(True), w.clone().requires_grad_(True)
        yc = grouped_linear(xc, wc, offs)
        dxc, dwc = torch.autograd.grad(yc, (xc, wc), dy.clone())
        for a, b in ((y, yc), (dx, dxc), (dw, dwc)):
            check(a, b.double(), rounded(b.double(), sums(torch.full_like(b, 40.0).double(), 8), t, 2))
    # transposed weights and expanded gradients
    vt = w.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(grouped_linear(wide[:, :96], vt, offs), grouped_linear(
        wide[:, :96], w, offs))
    xr = wide[:, :96].detach().requires_grad_(True)
    ones, = torch.autograd.grad(grouped_linear(xr, w, offs).sum(), xr)
    want, = torch.autograd.grad(grouped_linear(xr, w, offs), xr,
                                torch.ones(101, 72, dtype=t, device="cuda"))
    assert torch.equal(ones, want)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_slots_outside_the_ranges(dev, dtype):
    """A padded batch: zeros behind the last range (and before the first), gradients of zero."""
    t = TYPES[dtype]
    offs = torch.tensor([5, 20, 20, 90]).cuda()
    x, w = values((300, 64), t, 1), values((3, 48, 64), t, 2)
    x[95:] = float("nan")
    x[:5] = float("inf")
    dy = values((300, 48), t, 3)
    dy[90:] = float("nan")
    xr, wr = x.requires_grad_(True), w.requires_grad_(True)
    y = grouped_linear(xr, wr, offs)
    dx, dw = torch.autograd.grad(y, (xr, wr), dy)
    assert not y[:5].any() and not y[90:].any() and not dx[:5].any() and not dx[90:].any()
    assert torch.isfinite(dw).all() and not dw[1].any()
    inner = torch.tensor([0, 15, 15, 85]).cuda()
    xi = x.detach()[5:90].clone().requires_grad_(True)
    yi = grouped_linear(xi, wr, inner)
    dxi, dwi = torch.autograd.grad(yi, (xi, wr), dy[5:90].clone())
    assert torch.equal(y[5:90], yi) and torch.equal(dx[5:90], dxi) and torch.equal(dw, dwi)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_rows_outside_are_nan(dev, dtype):
    t = TYPES[dtype]
    offs = torch.tensor([0, 4, 8, 12]).cuda()
    rows = torch.tensor([0, 1, 2, 3, 4, -1, 5, 99, 6, 7, 8, 9]).cuda()
    x, w = values((10, 32), t, 1), values((3, 24, 32), t, 2).requires_grad_(True)
    y = grouped_linear(x, w, offs, rows)
    bad = torch.isnan(y).all(1).tolist()
    assert bad == [j in (5, 7) for j in range(12)] and torch.isfinite(y[[0, 4, 6, 8]]).all()
    dw, = torch.autograd.grad(y, w, values((12, 24), t, 3))
    assert torch.isfinite(dw[0]).all() and torch.isfinite(dw[2]).all()
    assert torch.isnan(dw[1]).all()
    # a slot outside in the sum over a token's slots
    slots = torch.tensor([[0], [1], [2], [3], [4], [6], [8], [9], [10], [500]]).cuda()
    xr = x.clone().requires_grad_(True)
    good = rows.clamp(0, 9)
    dx, = torch.autograd.grad(grouped_linear(xr, w, offs, good, slots), xr,
                              values((12, 24), t, 3))
    assert torch.isfinite(dx[:9]).all() and torch.isnan(dx[9]).all()


def test_infinities_stay_in_their_rows(dev):
    t = torch.bfloat16
    offs = torch.tensor([0, 70, 200]).cuda()
    x, w = values((200, 256), t, 1), values((2, 128, 256), t, 2)
    want = grouped_linear(x, w, offs)
    x[69, 3] = float("inf")
    x[130, 200] = float("nan")
    got = grouped_linear(x, w, offs)
    keep = torch.ones(200, dtype=torch.bool)
    keep[[69, 130]] = False
    assert torch.equal(got[keep.cuda()], want[keep.cuda()])
    assert not torch.isfinite(got[69]).any() and torch.isnan(got[130]).all()


def test_only_the_gradient_asked_for(dev):
    offs, rows, slots = routing([20, 12], 16, 2, 0)
    x, w = values((16, 64), torch.float16, 1), values((2, 32, 64), torch.float16, 2)
    dy = values((32, 32), torch.float16, 3)
    xr, wr = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    both = torch.autograd.grad(grouped_linear(xr, wr, offs, rows, slots), (xr, wr), dy)
    one, = torch.autograd.grad(grouped_linear(xr, w, offs, rows, slots), xr, dy)
    two, = torch.autograd.grad(grouped_linear(x, wr, offs, rows), wr, dy)
    assert torch.equal(both[0], one) and torch.equal(both[1], two)


def test_refusals(dev):
    x, w = torch.zeros(4, 8, device=dev), torch.zeros(2, 6, 8, device=dev)
    offs = torch.tensor([0, 2, 4]).cuda()
    rows, slots = torch.arange(4).cuda(), torch.arange(4).view(4, 1).cuda()
    for match, err, args in [
        ("expected", ValueError, (x[0], w, offs)),
        ("expected", ValueError, (x[:, :7], w, offs)),
        ("expected torch.float32", ValueError, (x, w.half(), offs)),
        ("float32, float16 or bfloat16", ValueError, (x.double(), w.double(), offs)),
        ("offs", ValueError, (x, w, offs[:2])),
        ("offs", ValueError, (x, w, offs.int())),
        ("rows", ValueError, (x, w, offs, rows.int())),
        ("without rows", ValueError, (x, w, offs, None, slots)),
        ("for 4 tokens", ValueError, (x, w, offs, rows, slots[:3])),
        ("int64", ValueError, (x, w, offs, rows, slots.int())),
        ("takes slots", ValueError, (x.clone().requires_grad_(True), w, offs, rows)),
        ("empty", ValueError, (x, w[:, :0], offs)),
        ("MI355X only", RuntimeError, (x.cpu(), w, offs)),
    ]:
        with pytest.raises(err, match=match):
            grouped_linear(*args)
    with pytest.raises(RuntimeError, match="forward-mode"):
        with torch.autograd.forward_ad.dual_level():
            grouped_linear(torch.autograd.forward_ad.make_dual(x, x), w, offs)
    with pytest.raises(ValueError, match="one shape"):
        gated(x, x[:3])
    with pytest.raises(ValueError, match="as the others"):
        gated(x, x.half())
    with pytest.raises(ValueError, match="activation"):
        gated(x, x, "tanh")
    with pytest.raises(RuntimeError, match="once_differentiable|not have been used"):
        xr = x.clone().requires_grad_(True)
        d, = torch.autograd.grad(grouped_linear(xr, w, offs).square().sum(), xr, create_graph=True)
        torch.autograd.grad(d.sum(), xr)


# ---- the gated activation ------------------------------------------------------------------
def act64(x, act):
    """(activation, derivative, how many steps of float32 their relative errors may be)."""
    one = torch.ones_like(x)
    if act == "none":
        return x, one, one
    if act == "relu":
        return x.clamp_min(0), (x > 0).double(), one
    if act == "silu":
        p, q = torch.sigmoid(x), torch.sigmoid(-x)
        return x * p, p + x * p * q, 16 + 4 * x.abs()
    if act == "gelu":
        p = torch.special.erfc(-x * 0.5 ** 0.5) / 2
        return (x * p, p + x * torch.exp(-x * x / 2) * (2 * np.pi) ** -0.5, 16 + 4 * x * x)
    u = (2 / np.pi) ** 0.5 * (x + 0.044715 * x ** 3)
    p, q = torch.sigmoid(2 * u), torch.sigmoid(-2 * u)
    return (x * p, p + x * p * q * 2 * (2 / np.pi) ** 0.5 * (1 + 3 * 0.044715 * x * x),
            16 + 8 * u.abs())


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_gated(dev, dtype, act):
    t = TYPES[dtype]
    for rows, n, halves in [(1, 1, False), (3, 8, False), (5, 17, False), (37, 264, True),
                            (4, 1000, True), (2, 51, True), (300, 128, False), (1, 5003, False),
                            (0, 8, False)]:
        if halves:
            gate, up = values((rows, 2 * n), t, 1, 3.0).split(n, 1)
        else:
            gate, up = values((rows, n), t, 1, 3.0), values((rows, n), t, 2, 3.0)
        gate, up = gate.detach().requires_grad_(True), up.detach().requires_grad_(True)
        dh = values((rows, n), t, 3, 0.5)
        out = gated(gate, up, act)
        dg, du = torch.autograd.grad(out, (gate, up), dh)
        with torch.no_grad():
            assert torch.equal(gated(gate, up, act), out)
        g, u, d = gate.detach().double(), up.detach().double(), dh.double()
        h, slope, steps = act64(g, act)
        # the derivative is a sum of p and x p (1 - p) (or x times the density), each so far off
        terms = slope.abs() + 2 * (slope - torch.where(g == 0, slope, h / g)).abs()
        err = steps * 2.0 ** -24
        check(out, h * u, rounded(h * u, err * (h * u).abs() + 2.0 ** -140, t))
        check(dg, d * u * slope, rounded(d * u * slope, err * (d * u).abs() * terms + 2.0 ** -140, t))
        check(du, d * h, rounded(d * h, err * (d * h).abs() + 2.0 ** -140, t))


def test_gated_shapes_and_extremes(dev):
    x = torch.tensor([[-1e4, -200.0, -100.0, -40.0, -0.0, 0.0, 40.0, 100.0, 1e4, 3e38]]).cuda()
    one = torch.ones_like(x)
    for act in ("relu", "silu", "gelu", "gelu_tanh"):
        g, u = x.clone().requires_grad_(True), one.clone().requires_grad_(True)
        y = gated(g, u, act)
        dg, du = torch.autograd.grad(y, (g, u), one)
        assert torch.equal(y, du) and torch.isfinite(dg).all()
        assert (y[0, :3].abs() < 1e-30).all() and torch.equal(y[0, 7:], x[0, 7:])
        assert (dg[0, :3].abs() < 1e-30).all() and torch.equal(dg[0, 7:], one[0, 7:])
    nan = torch.full((2, 9), float("nan")).cuda()
    assert torch.isnan(gated(nan, torch.ones_like(nan), "relu")).all()
    a = values((2, 3, 20), torch.bfloat16, 1).requires_grad_(True)
    y = gated(a, a, "silu")  # the same tensor twice
    assert y.shape == a.shape
    d, = torch.autograd.grad(y.float().sum(), a)
    b = a.detach().double().requires_grad_(True)
    want, = torch.autograd.grad((torch.nn.functional.silu(b) * b).sum(), b)
    assert float((d.double() - want).abs().max()) < 3 * 2.0 ** -8 * float(want.abs().max())
    assert gated(values((7,), torch.float32, 1), values((7,), torch.float32, 2)).shape == (7,)
    assert gated(torch.zeros(0, 4, 5, device=dev), torch.zeros(0, 4, 5, device=dev)).shape == (
        0, 4, 5)


# ---- streams and graphs ---------------------------------------------------------------------
def test_captured_forward_and_backward(dev):
    """Replays, with eager work between them, give what eager calls give on the same values."""
    t = torch.bfloat16
    offs, rows, slots = routing([33, 0, 70, 25], 64, 2, 0)
    x = values((64, 128), t, 1).requires_grad_(True)
    gate, up = (values((4, 96, 128), t, i, 0.1).requires_grad_(True) for i in (2, 3))
    dy = values((128, 96), t, 4)

    def step():
        h = gated(grouped_linear(x, gate, offs, rows, slots),
                  grouped_linear(x, up, offs, rows, slots))
        return [h.detach(), *torch.autograd.grad(h, (x, gate, up), dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        with torch.no_grad():
            x.copy_(values((64, 128), t, 20 + i))
            gate.mul_(1.0 + 0.1 * i)
            o, r, s = routing([10 * i, 50, 78 - 10 * i, 0], 64, 2, i)
            offs.copy_(o), rows.copy_(r), slots.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in outs]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_other_streams(dev):
    offs, rows, slots = routing([100, 156], 128, 2, 0)
    x, w = values((128, 256), torch.float16, 1), values((2, 256, 256), torch.float16, 2)
    want = grouped_linear(x, w, offs, rows)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for st in streams:
        with torch.cuda.stream(st):
            outs.append(grouped_linear(x, w, offs, rows))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


# ---- together --------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", list(TYPES))
def test_experts_mlp(dev, dtype):
    """The MLP and every gradient against autograd in 64 bits on the same routing."""
    t = TYPES[dtype]
    e, k, hidden, inter, tokens = 6, 3, 72, 40, 50
    x = values((5, 10, hidden), t, 1).requires_grad_(True)
    logits = values((tokens, e), torch.float32, 2).requires_grad_(True)
    gate, up = (values((e, inter, hidden), t, i, 0.1).requires_grad_(True) for i in (3, 4))
    down = values((e, hidden, inter), t, 5, 0.1).requires_grad_(True)
    res = values((5, 10, hidden), t, 6).requires_grad_(True)
    r = route(logits, k)
    y = experts_mlp(x, r, gate, up, down, residual=res)
    assert y.shape == x.shape and y.dtype == t
    dy = values(y.shape, t, 7)
    leaves = (x, gate, up, down, res, logits)
    got = torch.autograd.grad(y, leaves, dy)
    a = [v.detach().double().requires_grad_(True) for v in leaves]
    p = torch.softmax(a[5], -1).gather(1, r.index)
    p = p / p.sum(-1, keepdim=True)
    flat = a[0].reshape(tokens, hidden)
    h = torch.nn.functional.silu(torch.matmul(a[1], flat.T)) * torch.matmul(a[2], flat.T)
    every = torch.matmul(a[3], h).permute(2, 0, 1)  # [T, E, hidden]
    out = (every.gather(1, r.index[..., None].expand(-1, -1, hidden)) * p[..., None]).sum(1)
    want_y = out.view(y.shape) + a[4]
    want = torch.autograd.grad(want_y, a, dy.double())
    # up to seven roundings to the type lie on the way to a gradient, each of a relative size of
    # half a step on its values, and add up (in norm) at most linearly
    rel = 8 * torch.finfo(t).eps / 2 + 1e-6
    for g, w in zip((y, *got), (want_y, *want)):
        assert float((g.double() - w).norm()) <= rel * float(w.norm())
