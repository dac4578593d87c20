"""Every form of the packed products on the MI355X against float64: fragments a wave, waves
a workgroup, rows transformed inside and before, tiles of each size, columns in shares, long
rows, experts' tiles; with operands in every type and what infinities become.  Bounds as in
test_gpu_packed."""

import numpy as np
import pytest
import torch

from packed_data import act64, bound, packed_tensor, stored
from test_gpu_packed import F, MIX, N, _experts, check, tokens

pytestmark = pytest.mark.gpu

EVERY = [(nb, b) for nb in (2, 4, 8) for b in (16, 32, 64)]


def some(t, most=300):
    """Row numbers to check: the first and last of tiles, and some between."""
    if t <= most:
        return np.arange(t)
    edge = np.concatenate([np.arange(0, t, 128), np.arange(127, t, 128), [t - 1]])
    return np.unique(np.concatenate([np.random.default_rng(t).integers(0, t, most), edge]))


def product(n, k, t, dt, dev, classes=EVERY, had=0.8, smooth=False):
    from hi2_amd.packed import PackedLinear, packed_linear

    print("product", n, k, t, dt, flush=True)
    p, w = packed_tensor(n, k, [c for c in classes if k % c[1] == 0], n + t, had=had,
                         smooth=smooth)
    x = tokens(t, k, F[dt], t, dev)
    got = packed_linear(x, PackedLinear(p, dev))
    at = some(t)
    xs = stored(N(x[at]), p)
    want = xs @ w.T
    check(got[at], want, bound(want, F[dt], F[dt], xs, w, 1.0))
    return p, x, got


# one row: one to eight waves, by columns and fragments; two to eight rows, with four and
# eight waves; up to 16 rows, one, two and four fragments a wave
FEW = [(40, 512, 1), (40, 1024, 1), (40, 2048, 1), (40, 4096, 1), (40, 5120, 1), (8300, 384, 1),
       (8300, 1152, 1), (40, 1536, 2), (40, 1152, 3), (40, 1152, 8), (8300, 256, 2),
       (8300, 256, 4), (8300, 128, 7), (200, 640, 12), (3300, 256, 16), (8500, 128, 9)]


@pytest.mark.parametrize("n,k,t", FEW)
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_few_rows(n, k, t, dt, dev):
    product(n, k, t, dt, dev)


# 64 x 64, 128 x 64 and 256 x 128 tiles; columns in 2 to 16 shares
TILES = [(150, 256, 70), (2100, 256, 1030), (4200, 256, 2100), (1000, 192, 16100),
         (300, 4096, 100), (600, 2048, 200), (80, 512, 40), (20, 8320, 17)]


@pytest.mark.parametrize("n,k,t", TILES)
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_tiles(n, k, t, dt, dev):
    product(n, k, t, dt, dev, EVERY if n < 1000 else MIX)


@pytest.mark.parametrize("k", [192, 1040, 2064, 4160, 8256, 16384, 17024])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_rows_of_every_length(k, dt, dev):
    """The transform in front: a row by 64 to 1024 threads, kept in registers or read twice;
    and the same activations handed on."""
    from hi2_amd.packed import PackedLinear, activations, packed_linear

    p, x, got = product(24, k, 37, dt, dev, smooth=True)
    plan = PackedLinear(p, dev)
    assert torch.equal(packed_linear(activations(x, plan), plan), got)
    product(24, k, 5, dt, dev, smooth=True)


@pytest.mark.parametrize("t", [1, 6, 12, 90])
@pytest.mark.parametrize("op", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
def test_operands_of_every_type(t, op, out, dev):
    """Bias, factor and residual of one type, the result of another; rows of strided views."""
    from hi2_amd.packed import PackedLinear, packed_linear

    n, k = 75, 192
    p, w = packed_tensor(n, k, MIX, 5)
    x = tokens(t, k, torch.bfloat16, t, dev)
    g = torch.Generator().manual_seed(t)
    bias = torch.randn(n, generator=g).to(F[op]).to(dev)
    mul, res = torch.randn(2, t, n + 9, generator=g).to(F[op]).to(dev)[..., :n]
    got = packed_linear(x, PackedLinear(p, dev), bias=bias, mul=mul, residual=res,
                        activation="relu", out_dtype=F[out])
    assert got.dtype == F[out]
    xs = stored(N(x), p)
    pre = xs @ w.T + N(bias)
    want = act64(pre, "relu") * N(mul) + N(res)
    lim = bound(want, F[out], torch.bfloat16, xs, w, np.abs(N(mul))) + \
        2.0 ** -21 * (np.abs(pre) + np.abs(N(bias))) * np.abs(N(mul)) + 2.0 ** -22 * np.abs(N(res))
    check(got, want, lim)


@pytest.mark.parametrize("t", [1, 5, 14, 60])
@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
def test_an_infinity_gives_infinities(t, dt, dev):
    """An infinite activation in a column that is not rotated gives the sign of its weight,
    in one plane and in two."""
    from hi2_amd.packed import PackedLinear, packed_linear

    p, w = packed_tensor(33, 128, MIX, 8, had=0.5)
    p.had[2], p.had[3] = 0, 1
    x = tokens(t, 128, F[dt], 1, dev)
    x[0, 37] = float("inf")
    got = N(packed_linear(x, PackedLinear(p, dev)))
    assert (w[:, 37] != 0).all()
    assert np.array_equal(got[0], np.where(w[:, 37] > 0, np.inf, -np.inf))
    assert np.isfinite(got[1:]).all()


@pytest.mark.parametrize("n,k,t,e", [(100, 128, 700, 4), (520, 256, 8100, 4),
                                     (1000, 192, 16100, 3), (2100, 128, 8, 8)])
@pytest.mark.parametrize("own", [False, True])
def test_tiles_of_experts(n, k, t, e, own, dev):
    """Experts' products in 64 x 64, 128 x 64 and 256 x 128 tiles and one row at a time, one
    expert with none."""
    from hi2_amd.packed import PackedExperts, experts_linear

    print("experts", n, k, t, e, own, flush=True)
    ts, ws = _experts(e, n, k, 70, own)
    g = np.random.default_rng(t)
    cuts = np.sort(g.integers(0, t + 1, e - 2))
    o = np.concatenate([[0], cuts, [t, t]])  # the last expert gets none
    x = tokens(t // 2 + 1, k, torch.bfloat16, 2, dev)
    r = g.integers(0, len(x), t)
    got = experts_linear(x, PackedExperts(ts, dev), torch.from_numpy(o).to(dev),
                         torch.from_numpy(r).to(dev))
    for i in range(e):
        at = o[i] + some(o[i + 1] - o[i])
        if not len(at):
            continue
        xs = stored(N(x[r[at]]), ts[i])
        want = xs @ ws[i].T
        check(got[at], want, bound(want, torch.bfloat16, torch.bfloat16, xs, ws[i], 1.0),
              f"expert {i}")


@pytest.mark.parametrize("t,e,k,h,i", [(2, 8, 4, 1088, 256), (1, 2, 1, 128, 2304),
                                       (2, 3, 2, 192, 1152), (40, 4, 2, 256, 512),
                                       (20, 2, 1, 2304, 1152), (20, 2, 1, 8256, 64),
                                       (30, 70, 2, 128, 64), (9, 3, 3, 64, 5120)])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_gated_mlp_of_unlike_tensors(t, e, k, h, i, dt, dev):
    """gate, up and down cut into rows of different classes, gate and up of different
    transforms; as a norm against float64."""
    from hi2_amd.moe import route
    from hi2_amd.packed import PackedExperts, moe_mlp

    print("mlp", t, e, k, h, i, dt, flush=True)
    gs, us = _experts(e, i, h, 100), _experts(e, i, h, 200, classes=[(8, 64), (2, 16), (4, 32)])
    for u in us[0]:
        u.had[1:] = 0
    ds = _experts(e, h, i, 300, classes=[(4, 64)])
    plans = [PackedExperts(s[0], dev) for s in (gs, us, ds)]
    x = tokens(t, h, F[dt], 4, dev)
    r = route(torch.randn(t, e, generator=torch.Generator().manual_seed(3)).to(dev), k)
    got = moe_mlp(x, r, *plans)
    index, w = N(r.index).astype(int), N(r.weights)
    want = np.zeros((t, h))
    for j in range(e):
        tok, c = np.nonzero(index == j)
        if not len(tok):
            continue
        a = act64(stored(N(x)[tok], gs[0][j]) @ gs[1][j].T, "silu")
        a = a * (stored(N(x)[tok], us[0][j]) @ us[1][j].T)
        np.add.at(want, tok, w[tok, c][:, None] * (stored(a, ds[0][j]) @ ds[1][j].T))
    rel = np.linalg.norm(N(got) - want) / np.linalg.norm(want)
    assert rel < {"bf16": 2.0 ** -8, "f32": 2.0 ** -19}[dt], rel


@pytest.mark.parametrize("size", [1e-30, 1.0, 1e18])
def test_gated_mlp_at_any_scale(size, dev):
    """What the experts hand on is scaled, so that neither tiny nor huge tokens overflow or
    vanish on the way; a token with an infinity and one with a NaN keep to themselves."""
    from hi2_amd.moe import route
    from hi2_amd.packed import PackedExperts, moe_mlp

    t, e, k, h, i = 60, 4, 2, 128, 192
    gs, us, ds = _experts(e, i, h, 100), _experts(e, i, h, 200), _experts(e, h, i, 300)
    plans = [PackedExperts(s[0], dev) for s in (gs, us, ds)]
    x = (tokens(t, h, torch.float32, 4, dev) * size).bfloat16()
    x[3, 5], x[7, 9] = float("inf"), float("nan")
    r = route(torch.randn(t, e, generator=torch.Generator().manual_seed(3)).to(dev), k)
    got = moe_mlp(x, r, *plans, activation="relu")
    ok = np.setdiff1d(np.arange(t), [3, 7])
    assert not torch.isfinite(got[3]).any() and torch.isnan(got[7]).all()
    index, w = N(r.index).astype(int), N(r.weights)
    want = np.zeros((t, h))
    for j in range(e):
        tok, c = np.nonzero(index == j)
        c, tok = c[np.isin(tok, ok)], tok[np.isin(tok, ok)]
        a = act64(stored(N(x)[tok], gs[0][j]) @ gs[1][j].T, "relu")
        a = a * (stored(N(x)[tok], us[0][j]) @ us[1][j].T)
        np.add.at(want, tok, w[tok, c][:, None] * (stored(a, ds[0][j]) @ ds[1][j].T))
    if size < 1e-20:  # (products below the smallest float32)
        assert np.abs(N(got)[ok]).max() <= 1e-37
    else:
        rel = np.linalg.norm(N(got)[ok] - want[ok]) / np.linalg.norm(want[ok])
        assert rel < 2.0 ** -8, rel


def test_gated_mlp_refuses_what_is_no_routing_of_its_tokens(dev):
    from dataclasses import replace

    from hi2_amd.moe import route
    from hi2_amd.packed import PackedExperts, moe_mlp

    gate, down = (PackedExperts(_experts(3, n, k, 5)[0], dev) for n, k in ((64, 128), (128, 64)))
    x = tokens(6, 128, torch.bfloat16, 1, dev)
    r = route(torch.randn(6, 3, generator=torch.Generator().manual_seed(2)).to(dev), 2)
    good = moe_mlp(x, r, gate, gate, down)
    for wrong, match in ((dict(rows=r.rows[:3]), "belong together"),
                         (dict(weights=r.weights[:, :1]), "belong together"),
                         (dict(slots=r.slots[:4]), "of 4 tokens for 6"),
                         (dict(offs=r.offs[:3]), "over 2 experts for 3"),
                         (dict(rows=r.rows.int()), "int64"),
                         (dict(slots=r.slots.int()), "int64"),
                         (dict(weights=r.weights.double()), "float32")):
        with pytest.raises(ValueError, match=match):
            moe_mlp(x, replace(r, **wrong), gate, gate, down)
    with pytest.raises(RuntimeError):
        moe_mlp(x, replace(r, offs=r.offs.cpu()), gate, gate, down)
    same = replace(r, slots=r.slots.t().contiguous().t(), weights=r.weights.t().contiguous().t())
    assert not same.slots.is_contiguous()
    assert torch.equal(moe_mlp(x, same, gate, gate, down), good)


def test_half_precision_mlp_with_one_plain_projection(dev):
    """fp16 tokens that gate takes as they are and up rotates: the rotated ones need both
    planes."""
    from hi2_amd.moe import route
    from hi2_amd.packed import PackedExperts, moe_mlp

    t, e, k, h, i = 40, 3, 2, 128, 64
    gs, us, ds = _experts(e, i, h, 100), _experts(e, i, h, 200), _experts(e, h, i, 300)
    for g in gs[0]:
        g.had[:] = 0
    plans = [PackedExperts(s[0], dev) for s in (gs, us, ds)]
    assert plans[0].plain and not plans[1].plain
    x = tokens(t, h, torch.float16, 4, dev)
    r = route(torch.randn(t, e, generator=torch.Generator().manual_seed(3)).to(dev), k)
    got = moe_mlp(x, r, *plans)
    index, w = N(r.index).astype(int), N(r.weights)
    want = np.zeros((t, h))
    for j in range(e):
        tok, c = np.nonzero(index == j)
        a = act64(stored(N(x)[tok], gs[0][j]) @ gs[1][j].T, "silu")
        a = a * (stored(N(x)[tok], us[0][j]) @ us[1][j].T)
        np.add.at(want, tok, w[tok, c][:, None] * (stored(a, ds[0][j]) @ ds[1][j].T))
    # only the result's rounding: half an ulp of each, at most 2^-11 (one plane would add as much)
    off = np.abs(N(got) - want) - 2.0 ** -11 * np.abs(want)
    assert off.max() < 2.0 ** -13 * np.abs(want).max()
