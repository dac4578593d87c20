"""Products by packed tensors (hi2_amd.packed) on the MI355X against float64: every row
class and block, activations of one row to several tiles, odd sizes, every input type, the
epilogue, strides, extreme and non-finite inputs; the experts' products over routed slots
with empty experts and transforms of their own; the weighted sum; capture and streams.
Bounds follow from the roundings named in packed_data.bound."""

import numpy as np
import pytest
import torch

from packed_data import act64, bound, order64, packed_tensor, stored

pytestmark = pytest.mark.gpu

ALL = [(2, 16), (2, 32), (2, 64), (4, 16), (4, 32), (4, 64), (8, 32), (8, 64)]
MIX = [(2, 32), (4, 64)]
F = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def tokens(t, k, dtype, seed, dev):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(t, k, generator=g)
    x[:, torch.randperm(k, generator=g)[: -(-k // 100)]] *= 20.0
    return x.to(dtype).to(dev)


def N(t):
    return t.detach().double().cpu().numpy()


def check(got, want, lim, what=""):
    got = N(got).reshape(want.shape)
    off = np.abs(got - want) - lim
    assert np.isfinite(got).all() and (off <= 0).all(), \
        f"{what}: off by {np.abs(got - want).max():.3g}, {(off > 0).sum()} of {off.size} beyond"


SHAPES = [  # n, k, t
    (1, 16, 1), (3, 48, 2), (17, 64, 5), (64, 128, 1), (65, 192, 16), (130, 320, 17),
    (257, 448, 33), (300, 256, 64), (96, 1024, 100), (512, 640, 129), (40, 2304, 257),
    (1030, 384, 7),
]


@pytest.mark.parametrize("n,k,t", SHAPES)
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_product_of_mixed_rows(n, k, t, dt, dev):
    from hi2_amd.packed import PackedLinear, packed_linear

    print("product", n, k, t, dt, flush=True)
    classes = [(nb, b) for nb, b in ALL if k % b == 0]
    p, w = packed_tensor(n, k, classes, 3 * n + t, had=0.8)
    x = tokens(t, k, F[dt], t, dev)
    got = packed_linear(x, PackedLinear(p, dev))
    xs = stored(N(x), p)
    want = xs @ w.T
    assert got.dtype == F[dt] and got.shape == (t, n)
    check(got, want, bound(want, F[dt], F[dt], xs, w, 1.0))


@pytest.mark.parametrize("nb,b", ALL)
@pytest.mark.parametrize("t", [1, 24, 200])
def test_product_of_one_class(nb, b, t, dev):
    from hi2_amd.packed import PackedLinear, packed_linear

    n, k = 144, 704
    print("class", nb, b, t, flush=True)
    p, w = packed_tensor(n, k, [(nb, b)], nb + b, smooth=True)
    x = tokens(t, k, torch.bfloat16, 5, dev)
    xs = stored(N(x), p)
    want = xs @ w.T
    check(packed_linear(x, PackedLinear(p, dev), out_dtype=torch.float32), want,
          bound(want, torch.float32, torch.bfloat16, xs, w, 1.0))


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("t", [1, 9, 150])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_epilogue(act, t, dt, dev):
    from hi2_amd.packed import PackedLinear, packed_linear

    n, k = 200, 256
    print("epilogue", act, t, dt, flush=True)
    p, w = packed_tensor(n, k, MIX, 9)
    x = tokens(t, k, F[dt], 1, dev)
    g = torch.Generator().manual_seed(2)
    bias = torch.randn(n, generator=g).to(F[dt]).to(dev)
    # rows of wider matrices: strides other than n
    mul = torch.randn(t, n + 7, generator=g).to(F[dt]).to(dev)[:, 3:n + 3]
    res = torch.randn(t, 2 * n, generator=g).to(dev)[:, :n]
    got = packed_linear(x, PackedLinear(p, dev), bias=bias, activation=act, mul=mul, residual=res)
    xs = stored(N(x), p)
    pre = xs @ w.T + N(bias)
    want = act64(pre, act) * N(mul) + N(res)
    # the steepest slope of the activations is below 1.13; the f32 steps of the epilogue are
    # each within 4 units of their values
    lim = bound(want, F[dt], F[dt], xs, w, 1.13 * np.abs(N(mul))) + \
        2.0 ** -20 * (np.abs(pre * N(mul)) + np.abs(N(res)))
    check(got, want, lim)


def test_magnitudes_and_zeros(dev):
    from hi2_amd.packed import PackedLinear, packed_linear

    n, k = 70, 384
    p, w = packed_tensor(n, k, MIX, 4)
    x = tokens(40, k, torch.float32, 1, dev)
    scale = torch.ones(40, device=dev)
    scale[::4], scale[1::4], scale[2::4] = 1e30, 1e-30, 0.0
    x = x * scale[:, None]
    for dtype in (torch.float32, torch.bfloat16):
        xd = x.to(dtype)
        xs = stored(N(xd), p)
        want = xs @ w.T
        check(packed_linear(xd, PackedLinear(p, dev)), want,
              bound(want, dtype, dtype, xs, w, 1.0))


def test_non_finite_rows_stay_theirs(dev):
    from hi2_amd.packed import PackedLinear, packed_linear

    n, k = 48, 256
    p, w = packed_tensor(n, k, MIX, 6, had=0.5)
    for t in (4, 140):
        x = tokens(t, k, torch.bfloat16, 3, dev)
        clean = packed_linear(x, PackedLinear(p, dev))
        x[1, 17] = float("nan")
        x[2, 40] = float("inf")
        got = packed_linear(x, PackedLinear(p, dev))
        keep = [i for i in range(t) if i not in (1, 2)]
        assert torch.equal(got[keep], clean[keep])
        assert torch.isnan(got[1]).all() and not torch.isfinite(got[2]).any()


def test_subnormal_weights_count(dev):
    """Steps and values below fp16's normal range are decoded and multiplied as they are."""
    from hi2_amd.packed import PackedLinear, packed_linear

    p, _ = packed_tensor(32, 256, [(4, 64)], 5, had=0.0, step=6e-8 * 40)
    p.row_consts[:, :2] = 0
    c = p.row_consts.double().numpy()
    u = p.blk_params.numpy().reshape(32, 4, 2)[..., 1].astype(np.float64)
    st = (u * c[:, 2:3]).astype(np.float32).astype(np.float16).astype(np.float64)
    words = p.codes.numpy().view(np.uint32).reshape(32, 32)
    codes = ((words[..., None] >> (4 * np.arange(8, dtype=np.uint32))) & 15).reshape(32, 4, 64)
    w = (codes * st[..., None]).astype(np.float16).astype(np.float64).reshape(32, 256)
    assert 0 < np.abs(w[w != 0]).min() < 2.0 ** -14
    x = torch.eye(256, device=dev)
    got = packed_linear(x, PackedLinear(p, dev))
    assert np.array_equal(N(got), w.T)


def test_every_code_decodes_to_the_formats_value(dev):
    """Against unit vectors the product is the decoded weight itself, bit for bit."""
    from hi2_amd.packed import PackedLinear, packed_linear

    for k, classes in ((704, [(2, 64), (4, 32), (8, 64)]), (272, [(2, 16), (4, 16)])):
        p, w = packed_tensor(90, k, classes, 8, had=0.0)
        got = packed_linear(torch.eye(k, device=dev), PackedLinear(p, dev))
        assert np.array_equal(N(got), w.T)
        few = torch.zeros(3, k, device=dev)
        few[0, 0] = few[1, k - 1] = few[2, k // 2] = 1.0
        got = packed_linear(few, PackedLinear(p, dev))
        assert np.array_equal(N(got), w.T[[0, k - 1, k // 2]])


def test_shapes_strides_and_nothing_to_do(dev):
    from hi2_amd.packed import PackedLinear, activations, packed_linear

    n, k = 66, 320
    p, w = packed_tensor(n, k, MIX, 2)
    plan = PackedLinear(p, dev)
    x = tokens(24, k, torch.bfloat16, 1, dev)
    whole = packed_linear(x, plan)
    assert torch.equal(packed_linear(x.view(2, 3, 4, k), plan), whole.view(2, 3, 4, n))
    wide = torch.zeros(24, k + 9, dtype=x.dtype, device=dev)
    wide[:, 5:5 + k] = x
    assert torch.equal(packed_linear(wide[:, 5:5 + k], plan), whole)
    assert torch.equal(packed_linear(x.t().contiguous().t(), plan), whole)
    assert torch.equal(packed_linear(x.flip(0)[::2], plan), whole.flip(0)[::2])
    assert torch.equal(packed_linear(x[0], plan), packed_linear(x[:1], plan)[0])
    assert torch.equal(packed_linear(activations(x, plan), plan), whole)
    assert packed_linear(x[:0], plan).shape == (0, n)
    one = packed_linear(x[:1].expand(24, k), plan)
    assert torch.equal(one, one[:1].expand(24, n))
    # device buffers lay out to the same
    for f in ("codes", "blk_params", "row_consts"):
        setattr(p, f, getattr(p, f).to(dev))
    assert torch.equal(packed_linear(x, PackedLinear(p, dev)), whole)


def test_repeats_and_streams_agree(dev):
    from hi2_amd.packed import PackedLinear, packed_linear

    p, _ = packed_tensor(400, 1024, MIX, 2)
    plan = PackedLinear(p, dev)
    torch.cuda.synchronize()
    for t in (1, 6, 40, 300):
        x = tokens(t, 1024, torch.bfloat16, t, dev)
        want = packed_linear(x, plan)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            got = [packed_linear(x, plan) for _ in range(3)]
        side.synchronize()
        assert all(torch.equal(g, want) for g in got)


def test_more_than_four_gib_of_activations(dev):
    from hi2_amd.packed import PackedLinear, packed_linear

    n, k, t = 16, 4096, 560_000
    p, w = packed_tensor(n, k, [(4, 64)], 2)
    x = torch.zeros(t, k, dtype=torch.bfloat16, device=dev)
    at = torch.tensor([0, 262_143, 262_144, 524_287, 524_288, t - 1], device=dev)
    x[at] = tokens(len(at), k, torch.bfloat16, 3, dev)
    got = packed_linear(x, PackedLinear(p, dev))
    xs = stored(N(x[at]), p)
    want = xs @ w.T
    check(got[at], want, bound(want, torch.bfloat16, torch.bfloat16, xs, w, 1.0))
    got[at] = 0
    assert not got.any()


def test_capture_replays(dev):
    from hi2_amd.moe import route
    from hi2_amd.packed import PackedExperts, PackedLinear, moe_mlp, packed_linear

    p, _ = packed_tensor(200, 256, MIX, 2)
    plan = PackedLinear(p, dev)
    ex = [PackedExperts([packed_tensor(n, k, MIX, 10 * i + j)[0] for j in range(8)], dev)
          for i, (n, k) in enumerate(((128, 256), (128, 256), (256, 128)))]
    x = tokens(5, 256, torch.bfloat16, 1, dev)
    logits = torch.randn(5, 8, device=dev)

    def step():
        return packed_linear(x, plan, activation="silu"), moe_mlp(x, route(logits, 2), *ex)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        x.copy_(tokens(5, 256, torch.bfloat16, seed + 7, dev))
        logits.copy_(torch.randn(5, 8, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- experts --------------------------------------------------------------------------------
def _experts(e, n, k, seed, own=False, classes=MIX):
    made = [packed_tensor(n, k, classes, seed + i, had=0.5 if own else 1.0,
                          smooth=own and i % 2 == 0) for i in range(e)]
    return [m[0] for m in made], [m[1] for m in made]


@pytest.mark.parametrize("sizes", [[1], [0, 3, 0, 1], [5, 0, 200, 17, 129], [0, 0, 2], [0, 0],
                                   [1] * 70 + [0] * 10 + [130]])
@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_experts_products(sizes, own, dt, dev):
    from hi2_amd.packed import PackedExperts, experts_linear

    e, n, k = len(sizes), 80, 192
    print("experts", sizes[:6], own, dt, flush=True)
    ts, ws = _experts(e, n, k, 40, own)
    plan = PackedExperts(ts, dev)
    assert (plan.transform is None) == (own and e > 1)
    s = sum(sizes)
    x = tokens(max(50, s // 2), k, F[dt], 2, dev)
    g = torch.Generator().manual_seed(1)
    rows = torch.randint(0, len(x), (s,), generator=g).to(dev)
    offs = torch.tensor(np.concatenate([[0], np.cumsum(sizes)]), dtype=torch.int64, device=dev)
    mul = torch.randn(s, n, generator=g).to(dev)
    got = experts_linear(x, plan, offs, rows, activation="silu", mul=mul)
    assert got.shape == (s, n) and got.dtype == F[dt]
    pre_ordered = experts_linear(x[rows], plan, offs, activation="silu", mul=mul)
    assert torch.equal(got, pre_ordered)
    o, r, m = N(offs).astype(int), N(rows).astype(int), N(mul)
    for i in range(e):
        a, b = o[i], o[i + 1]
        if a == b:
            continue
        xs = stored(N(x)[r[a:b]], ts[i])
        pre = xs @ ws[i].T
        want = act64(pre, "silu") * m[a:b]
        lim = bound(want, F[dt], F[dt], xs, ws[i], 1.13 * np.abs(m[a:b])) + \
            2.0 ** -20 * np.abs(pre * m[a:b])
        check(got[a:b], want, lim, f"expert {i}")


def test_rows_outside_the_batch_are_nan(dev):
    from hi2_amd.packed import PackedExperts, experts_linear

    ts, _ = _experts(2, 64, 128, 3)
    for own in (False, True):
        plan = PackedExperts(_experts(2, 64, 128, 3, own)[0], dev)
        x = tokens(6, 128, torch.bfloat16, 2, dev)
        rows = torch.tensor([0, 5, -1, 6, 2, 1 << 40], device=dev)
        offs = torch.tensor([0, 3, 6], device=dev)
        got = experts_linear(x, plan, offs, rows)
        ok = torch.tensor([0, 1, 4])
        assert torch.isnan(got[[2, 3, 5]]).all() and torch.isfinite(got[ok]).all()
        rows[[2, 3, 5]] = 0
        assert torch.equal(experts_linear(x, plan, offs, rows)[ok], got[ok])


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("t,n,k", [(1, 64, 8), (9, 333, 3), (300, 2048, 2), (4, 1, 1)])
def test_combine(t, n, k, dt, dev):
    from hi2_amd.packed import combine

    g = torch.Generator().manual_seed(t)
    y = torch.randn(t * k, n, generator=g).to(F[dt]).to(dev)
    slots = torch.randperm(t * k, generator=g).reshape(t, k).to(dev)
    w = torch.rand(t, k, generator=g).to(dev)
    for res in (None, torch.randn(t, n, generator=g).to(F[dt]).to(dev)):
        got = combine(y, slots, w, residual=res)
        terms = N(w)[..., None] * N(y)[N(slots).astype(int)]
        want = terms.sum(1) + (0 if res is None else N(res))
        mass = np.abs(terms).sum(1) + (0 if res is None else np.abs(N(res)))
        unit = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 0}[dt]
        check(got, want, unit * np.abs(want) + (k + 1) * 2.0 ** -23 * mass + 2.0 ** -24)
    slots[0, 0] = t * k
    assert torch.isnan(combine(y, slots, w)[0]).all()


@pytest.mark.parametrize("t,e,k,h,i,own", [(1, 8, 2, 256, 128, False), (3, 64, 8, 128, 64, False),
                                           (130, 8, 2, 256, 192, True), (700, 6, 3, 128, 64, False)])
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_moe_mlp(t, e, k, h, i, own, dt, dev):
    """Router, experts and sum together, as a norm against float64 (the hidden values pass a
    second product): the roundings of the input, the hidden values and the output."""
    from hi2_amd.moe import route
    from hi2_amd.packed import PackedExperts, moe_mlp

    print("mlp", t, e, k, h, i, own, dt, flush=True)
    gs, us, ds = _experts(e, i, h, 100, own), _experts(e, i, h, 200, own), _experts(e, h, i, 300, own)
    plans = [PackedExperts(s[0], dev) for s in (gs, us, ds)]
    x = tokens(t, h, F[dt], 4, dev)
    g = torch.Generator().manual_seed(3)
    r = route(torch.randn(t, e, generator=g).to(dev), k)
    res = torch.randn(t, h, generator=g).to(F[dt]).to(dev)
    got = moe_mlp(x, r, *plans, residual=res)
    index, w = N(r.index).astype(int), N(r.weights)
    want = N(res)
    for j in range(e):
        tok, c = np.nonzero(index == j)
        if not len(tok):
            continue
        a = act64(stored(N(x)[tok], gs[0][j]) @ gs[1][j].T, "silu")
        a = a * (stored(N(x)[tok], us[0][j]) @ us[1][j].T)
        np.add.at(want, tok, w[tok, c][:, None] * (stored(a, ds[0][j]) @ ds[1][j].T))
    rel = np.linalg.norm(N(got) - want) / np.linalg.norm(want)
    assert rel < {"bf16": 2.0 ** -8, "f16": 2.0 ** -10, "f32": 2.0 ** -19}[dt], rel
    order = order64(index, e)
    assert np.array_equal(N(r.rows), order[0]) and np.array_equal(N(r.offs), order[1])
    assert np.array_equal(N(r.slots), order[2])


def test_refusals(dev):
    from hi2_amd.packed import (PackedExperts, PackedLinear, activations, combine,
                                experts_linear, moe_mlp, packed_linear)

    p, _ = packed_tensor(32, 128, MIX, 1)
    other, _ = packed_tensor(32, 128, MIX, 1, smooth=True)
    plan, two = PackedLinear(p, dev), PackedExperts([p, other], dev)
    x = torch.randn(4, 128, device=dev)
    offs = torch.tensor([0, 2, 4], device=dev)
    with pytest.raises(RuntimeError, match="MI355X only"):
        packed_linear(x.cpu(), plan)
    with pytest.raises(ValueError, match="128 columns"):
        packed_linear(x[:, :64], plan)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        packed_linear(x.double(), plan)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        packed_linear(x, plan, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="bias"):
        packed_linear(x, plan, bias=x[0])
    with pytest.raises(ValueError, match="residual"):
        packed_linear(x, plan, residual=x)
    with pytest.raises(ValueError, match="activation"):
        packed_linear(x, plan, activation="tanh")
    with pytest.raises(RuntimeError, match="no gradient"):
        packed_linear(x.clone().requires_grad_(True), plan)
    with pytest.raises(TypeError):
        packed_linear(x, two)
    with pytest.raises(ValueError, match="transform"):
        packed_linear(activations(x, plan), PackedLinear(other, dev))
    with pytest.raises(ValueError, match="of their own"):
        activations(x, two)
    with pytest.raises(ValueError, match="offs"):
        experts_linear(x, two, offs[:2])
    with pytest.raises(ValueError, match="rows"):
        experts_linear(x, two, offs, offs.int())
    with pytest.raises(ValueError, match="one shape"):
        combine(x, offs[None], torch.ones(1, 2, device=dev))
    with pytest.raises(ValueError, match="same experts"):
        moe_mlp(x, None, two, two, PackedExperts([p, p, p], dev))
    with torch.no_grad():
        packed_linear(x.clone().requires_grad_(True), plan)
