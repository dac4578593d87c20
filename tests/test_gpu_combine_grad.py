"""Gradients of the experts' weighted sum (hi2_amd.packed.combine) on the MI355X against the
formula in float64 and against differences, and a router trained through frozen experts
(moe.route, packed.moe_mlp)."""

import numpy as np
import pytest
import torch

from packed_data import act64, order64, stored
from test_gpu_packed import F, N, _experts, tokens

pytestmark = pytest.mark.gpu

UNIT = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def made(t, n, k, dt, dev, seed=1, rows=None):
    g = torch.Generator().manual_seed(seed)
    rows = t * k if rows is None else rows
    y = torch.randn(rows, n, generator=g).to(F[dt]).to(dev)
    slots = torch.randperm(rows, generator=g)[:t * k].reshape(t, k).to(dev)
    w = torch.rand(t, k, generator=g).to(dev)
    res = torch.randn(t, n, generator=g).to(F[dt]).to(dev)
    c = torch.randn(t, n, generator=g).to(dev)
    return y, slots, w, res, c


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("out", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("t,n,k", [(1, 64, 8), (9, 333, 3), (300, 1024, 2), (4, 1, 1), (130, 260, 5)])
def test_gradients_against_the_formula(t, n, k, dt, out, dev):
    from hi2_amd.packed import combine

    y, slots, w, res, c = made(t, n, k, dt, dev, rows=t * k + 3)
    for v in (y, w, res):
        v.requires_grad_(True)
    o = combine(y, slots, w, residual=res, out_dtype=F[out])
    g = c.to(F[out])
    o.backward(g)
    g, s = N(g), N(slots).astype(int)
    terms = g[:, None] * N(y)[s]
    assert w.grad.dtype == torch.float32
    assert (np.abs(N(w.grad) - terms.sum(-1)) <= (n + 8) * 2.0 ** -24 * np.abs(terms).sum(-1)).all()
    want = np.zeros((t * k + 3, n))
    want[s.reshape(-1)] = (N(w)[..., None] * g[:, None]).reshape(-1, n)
    assert y.grad.dtype == F[dt]  # a product in float32, rounded to y's type
    assert (np.abs(N(y.grad) - want) <= (UNIT[dt] + 2.0 ** -23) * np.abs(want) + 2.0 ** -24).all()
    assert torch.equal(res.grad, torch.from_numpy(g).to(F[dt]).to(dev))


def test_gradients_against_differences(dev):
    """The sum is linear in each input: a difference over a whole step is the derivative, up to
    the sums' float32 rounding."""
    from hi2_amd.packed import combine

    y, slots, w, res, c = made(20, 68, 4, "f32", dev)
    inputs = [y, w, res]
    for v in inputs:
        v.requires_grad_(True)
    (combine(y, slots, w, residual=res) * c).sum().backward()
    g = torch.Generator().manual_seed(9)

    def loss(vs):
        with torch.no_grad():
            return (N(combine(vs[0], slots, vs[1], residual=vs[2])) * N(c))

    for i, v in enumerate(inputs):
        d = torch.randn(v.shape, generator=g).to(dev)
        vs = [[u.detach() + h * d if j == i else u.detach() for j, u in enumerate(inputs)]
              for h in (1.0, -1.0)]
        a, b = loss(vs[0]), loss(vs[1])
        # each element is at most 6 float32 roundings from its value, inputs' own included
        lim = 16 * 2.0 ** -24 * (np.abs(a).sum() + np.abs(b).sum() + 8 * np.abs(N(c)).sum())
        assert abs((a.sum() - b.sum()) / 2 - (N(v.grad) * N(d)).sum()) <= lim


def test_part_gradients_and_slots_outside(dev):
    from hi2_amd.packed import combine

    y, slots, w, res, c = made(6, 48, 2, "bf16", dev)
    w.requires_grad_(True)
    combine(y, slots, w).float().sum().backward()
    only = w.grad.clone()
    slots[2, 1], w.grad = 99, None
    y.requires_grad_(True)
    combine(y, slots, w).float().sum().backward()
    bad = torch.zeros(6, 2, dtype=torch.bool, device=dev)
    bad[2, 1] = True
    assert torch.isnan(w.grad[bad]).all() and torch.equal(w.grad[~bad], only[~bad])
    assert torch.isfinite(y.grad).all()
    empty = torch.zeros(0, 2, device=dev, requires_grad=True)
    out = combine(y, slots[:0], empty)
    out.sum().backward()
    assert out.shape == (0, 48) and empty.grad.shape == (0, 2)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_router_trained_through_frozen_experts(dt, dev):
    """The logits' gradient through weights, experts and sum, against float64; and the call
    without gradients gives the same values up to its own roundings."""
    from hi2_amd.moe import route
    from hi2_amd.packed import PackedExperts, moe_mlp

    t, e, k, h, i = 40, 6, 3, 128, 192
    gs, us, ds = _experts(e, i, h, 100), _experts(e, i, h, 200), _experts(e, h, i, 300)
    plans = [PackedExperts(s[0], dev) for s in (gs, us, ds)]
    x = tokens(t, h, F[dt], 4, dev)
    logits = torch.randn(t, e, generator=torch.Generator().manual_seed(3)).to(dev)
    logits.requires_grad_(True)
    res = torch.randn(t, h, generator=torch.Generator().manual_seed(5)).to(F[dt]).to(dev)
    r = route(logits, k)
    out = moe_mlp(x, r, *plans, residual=res)
    c = torch.randn(t, h, generator=torch.Generator().manual_seed(6)).to(F[dt]).to(dev)
    out.backward(c)
    index = N(r.index).astype(int)
    ys = np.zeros((t, k, h))
    for j in range(e):
        tok, at = np.nonzero(index == j)
        if len(tok):
            a = act64(stored(N(x)[tok], gs[0][j]) @ gs[1][j].T, "silu")
            a = a * (stored(N(x)[tok], us[0][j]) @ us[1][j].T)
            ys[tok, at] = stored(a, ds[0][j]) @ ds[1][j].T
    p = np.exp(N(logits) - N(logits).max(1, keepdims=True))
    p = p / p.sum(1, keepdims=True)
    chosen = np.take_along_axis(p, index, 1)
    w = chosen / chosen.sum(1, keepdims=True)
    dw = (N(c)[:, None] * ys).sum(-1)
    want = np.zeros((t, e))  # renormalised softmax: w_j (dw_j - sum w dw)
    np.put_along_axis(want, index, w * (dw - (w * dw).sum(1, keepdims=True)), 1)
    value = N(res) + (w[..., None] * ys).sum(1)
    # the hidden values are float32 here and round nothing; inputs of 16 bits in one plane do
    rel = np.linalg.norm(N(logits.grad) - want) / np.linalg.norm(want)
    assert rel < {"bf16": 2.0 ** -8, "f32": 2.0 ** -17}[dt], rel
    assert np.linalg.norm(N(out) - value) < 2.0 ** -8 * np.linalg.norm(value)
    with torch.no_grad():
        plain = moe_mlp(x, r, *plans, residual=res)
    assert np.linalg.norm(N(plain) - N(out)) < 2.0 ** -7 * np.linalg.norm(value)
    with pytest.raises(RuntimeError, match="no gradient"):
        moe_mlp(x.clone().requires_grad_(True), r, *plans)
    assert np.array_equal(N(r.slots), order64(index, e)[2])
