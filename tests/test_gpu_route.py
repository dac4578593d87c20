"""The router (hi2_amd.moe.route) on the MI355X against its definition in float64: choices,
weights, slot order and gradient, over one token to several workgroups, ties, masked and NaN
logits, groups and biases; the order feeds ExpertHessians unchanged."""

import numpy as np
import pytest
import torch

from packed_data import order64, route64

pytestmark = pytest.mark.gpu

F = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def N(t):
    return t.detach().double().cpu().numpy()


def logits_of(t, e, dtype, seed, dev, masked=0.0):
    g = torch.Generator().manual_seed(seed)
    x = 1.5 * torch.randn(t, e, generator=g)
    x[torch.rand(t, e, generator=g) < masked] = float("-inf")
    return x.to(dtype).to(dev)


def check(r, index, weights, e):
    assert np.array_equal(N(r.index), index)
    # scores are within a few units of float32 (the exponential, two quotients), sums of k
    assert np.allclose(N(r.weights), weights, rtol=64 * 2.0 ** -24, atol=1e-37)
    rows, offs, slots = order64(index, e)
    assert np.array_equal(N(r.rows), rows) and np.array_equal(N(r.offs), offs)
    assert np.array_equal(N(r.slots), slots)
    assert r.index.dtype == r.rows.dtype == r.offs.dtype == r.slots.dtype == torch.int64
    assert r.weights.dtype == torch.float32


@pytest.mark.parametrize("t", [1, 2, 33, 64, 65, 200, 1000])
@pytest.mark.parametrize("e,k", [(1, 1), (5, 5), (16, 2), (64, 8), (60, 4), (129, 1), (257, 8),
                                 (512, 32)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_softmax_choices_weights_and_order(t, e, k, dt, dev):
    from hi2_amd.moe import route

    print("route", t, e, k, dt, flush=True)
    x = logits_of(t, e, F[dt], t + e, dev)  # bf16: many ties
    for renorm in (True, False):
        r = route(x, k, renormalise=renorm, scale=2.5)
        index, w, _ = route64(N(x), k, renorm=renorm, scale=2.5)
        check(r, index, w, e)


def separated(x, bias, k, groups, top_groups):
    """Rows whose ranking by score + bias is decided by more than float32's rounding."""
    p = 1 / (1 + np.exp(-x))
    key = np.sort(p + bias, 1)
    ok = (np.diff(key, axis=1) > 1e-6).all(1)
    if top_groups < groups:
        by = np.sort((p + bias).reshape(len(x), groups, -1), 2)
        good = np.sort(by[..., -1] + (by[..., -2] if by.shape[2] > 1 else 0), 1)
        ok &= (np.diff(good, axis=1) > 1e-6).all(1)
    return ok


@pytest.mark.parametrize("t", [1, 64, 300])
@pytest.mark.parametrize("e,k,groups,top", [(64, 6, 1, 1), (64, 6, 8, 3), (256, 8, 8, 4),
                                            (60, 3, 4, 2), (128, 2, 64, 5), (32, 4, 32, 4),
                                            (384, 8, 12, 6)])
def test_sigmoid_bias_and_groups(t, e, k, groups, top, dev):
    from hi2_amd.moe import route

    print("groups", t, e, k, groups, top, flush=True)
    x = logits_of(t, e, torch.float32, e + k, dev)
    bias = torch.linspace(-0.3, 0.3, e)[torch.randperm(e, generator=torch.Generator()
                                                       .manual_seed(1))].to(dev)
    ok = separated(N(x), N(bias), k, groups, top)
    x = x[torch.from_numpy(np.flatnonzero(ok)).to(dev)].contiguous()
    assert len(x) >= t // 2
    r = route(x, k, scoring="sigmoid", bias=bias, groups=groups, top_groups=top)
    index, w, _ = route64(N(x), k, "sigmoid", N(bias), groups, top)
    check(r, index, w, e)
    # without a bias the logits rank
    r = route(x, k, groups=groups, top_groups=top)
    index, w, _ = route64(N(x), k, groups=groups, top_groups=top)
    check(r, index, w, e)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_masked_rows_and_nan(scoring, dev):
    from hi2_amd.moe import route

    x = logits_of(100, 24, torch.float32, 3, dev, masked=0.7)
    x[5] = float("-inf")
    x[6] = float("nan")
    x[7] = float("-inf")
    x[7, 20] = 0.5
    x[8] = torch.finfo(torch.float32).min
    x[9, 3] = float("nan")
    x[10] = 0.0
    x[10, ::2] = -0.0  # equal to 0: ties by index
    bias = torch.linspace(-1, 1, 24, device=dev)
    for b, groups, top in ((None, 1, 1), (None, 6, 2), (bias, 1, 1)):
        if b is not None and scoring == "softmax":
            continue
        r = route(x, 4, scoring=scoring, bias=b, groups=groups, top_groups=top)
        index, w, _ = route64(N(x), 4, scoring, None if b is None else N(b), groups, top)
        check(r, index, w, 24)
        assert torch.equal(r.index[5], r.index[6])
        assert not r.weights[5:7].any()


def test_no_tokens_strides_and_streams(dev):
    from hi2_amd.moe import route

    r = route(torch.empty(0, 16, device=dev), 4)
    assert r.index.shape == r.weights.shape == r.slots.shape == (0, 4)
    assert r.rows.numel() == 0 and not r.offs.any() and r.offs.numel() == 17
    x = logits_of(90, 40, torch.float32, 1, dev)
    want = route(x[:, 4:36].contiguous(), 3)
    for y in (x[:, 4:36], x.t().contiguous().t()[:, 4:36]):
        got = route(y, 3)
        assert torch.equal(got.index, want.index) and torch.equal(got.weights, want.weights)
    one = route(x[:1, 4:36], 3)
    assert torch.equal(one.index, want.index[:1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = route(x[:, 4:36], 3)
    side.synchronize()
    assert torch.equal(got.slots, want.slots) and torch.equal(got.rows, want.rows)


def test_many_workgroups(dev):
    from hi2_amd.moe import route, route_order

    for t, e in ((16384, 64), (40_000, 96), (36_000, 300)):  # scanned counts above 512 workgroups
        x = logits_of(t, e, torch.float32, t, dev)
        r = route(x, 8)
        assert torch.equal(r.index, x.sort(dim=-1, descending=True, stable=True).indices[:, :8])
        rows, offs = route_order(r.index, e)
        assert torch.equal(r.rows, rows) and torch.equal(r.offs, offs)
        assert torch.equal(r.rows[r.slots], torch.arange(t, device=dev)[:, None].expand(t, 8))
        again = route(x, 8)
        assert torch.equal(again.slots, r.slots) and torch.equal(again.weights, r.weights)


def test_order_feeds_the_experts_hessians(dev):
    from hi2_amd.moe import ExpertHessians, route, route_order
    from hi2_amd.workloads import activations

    x = activations(500, 256, 3, dev)
    r = route(logits_of(500, 8, torch.float32, 3, dev), 2)
    a, b = ExpertHessians(8, 256, dev), ExpertHessians(8, 256, dev)
    a.update_routed(x, r.offs, r.rows)
    rows, offs = route_order(r.index, 8)
    b.update_routed(x, offs, rows)
    assert torch.equal(a.S, b.S) and torch.equal(a.n, b.n)


GRADS = [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)]


@pytest.mark.parametrize("scoring,renorm", GRADS)
@pytest.mark.parametrize("t,e,k", [(1, 4, 2), (50, 64, 8), (300, 200, 5), (20, 400, 16)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_gradient_against_the_formula(scoring, renorm, t, e, k, dt, dev):
    from hi2_amd.moe import route

    x = logits_of(t, e, F[dt], e, dev).requires_grad_(True)
    g = torch.randn(t, k, generator=torch.Generator().manual_seed(5)).to(dev)
    r = route(x, k, scoring=scoring, renormalise=renorm, scale=1.5)
    got, = torch.autograd.grad(r.weights, x, g)
    assert got.dtype == F[dt] and not r.index.requires_grad
    index, _, p = route64(N(x), k, scoring, renorm=renorm, scale=1.5)
    want = np.zeros((t, e))
    mass = np.zeros((t, e))
    for i in range(t):
        at, gi = index[i], 1.5 * N(g)[i]
        s = p[i][at].sum()
        jac = np.zeros((k, e))  # d score_j / d logit
        for j, x_j in enumerate(at):
            if scoring == "sigmoid":
                jac[j, x_j] = p[i][x_j] * (1 - p[i][x_j])
            else:
                jac[j] = -p[i][x_j] * p[i]
                jac[j, x_j] += p[i][x_j]
        if renorm:
            w = p[i][at] / s
            jac = (jac - w[:, None] * jac.sum(0)) / s
        want[i] = gi @ jac
        mass[i] = p[i] * (np.abs(gi).sum() / (s if renorm else 1))
    # float32 throughout: a few units of the terms that cancel, then the rounding of the type
    unit = {"f32": 0.0, "bf16": 2.0 ** -8}[dt]
    assert (np.abs(N(got) - want) <= 64 * 2.0 ** -24 * mass + unit * np.abs(want) + 1e-30).all()


@pytest.mark.parametrize("scoring,renorm", GRADS)
def test_gradient_against_differences(scoring, renorm, dev):
    from hi2_amd.moe import route

    t, e, k, h = 3, 12, 4, 1e-2
    x = (torch.arange(t * e).reshape(t, e) * 7 % 12).float().to(dev) * 0.3  # gaps above 2 h
    g = torch.randn(t, k, generator=torch.Generator().manual_seed(2)).to(dev)

    def value(y):
        r = route(y, k, scoring=scoring, renormalise=renorm)
        return (r.weights.double() * g.double()).sum(1)

    leaf = x.clone().requires_grad_(True)
    got, = torch.autograd.grad(route(leaf, k, scoring=scoring, renormalise=renorm).weights, leaf, g)
    for c in range(e):
        d = torch.zeros(e, device=dev)
        d[c] = h
        num = (value(x + d) - value(x - d)) / (2 * h)
        # the third derivative's term h^2 / 6 (below 2 |g|_1 in size), float32 noise 2^-22 / h
        lim = g.abs().sum(1) * (2 * h * h / 6 + 2.0 ** -22 / h)
        assert ((got[:, c].double() - num).abs() <= lim).all()


def test_gradient_of_masked_rows_is_zero(dev):
    from hi2_amd.moe import route

    x = torch.full((3, 8), float("-inf"), device=dev)
    x[1, 2] = 1.0
    x.requires_grad_(True)
    r = route(x, 4)
    got, = torch.autograd.grad(r.weights, x, torch.randn(3, 4, device=dev))
    assert not got.any()


def test_refusals(dev):
    from hi2_amd.moe import route

    x = torch.randn(4, 16, device=dev)
    for kw, match in ((dict(top_k=0), "choices"), (dict(top_k=17), "choices"),
                      (dict(top_k=2, groups=3), "groups"),
                      (dict(top_k=5, groups=4, top_groups=1), "choices"),
                      (dict(top_k=2, groups=4, top_groups=5), "groups")):
        with pytest.raises(RuntimeError, match=match):
            route(x, **kw)
    with pytest.raises(RuntimeError, match="experts"):
        route(torch.randn(4, 513, device=dev), 2)
    with pytest.raises(ValueError, match="scoring"):
        route(x, 2, scoring="tanh")
    with pytest.raises(ValueError, match="bias"):
        route(x, 2, bias=x[0, :8])
    with pytest.raises(ValueError, match="float"):
        route(x.double(), 2)
    with pytest.raises(RuntimeError, match="MI355X only"):
        route(x.cpu(), 2)
