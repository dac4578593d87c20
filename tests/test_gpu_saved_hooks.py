"""Saved tensors' hooks: what comes back has the values that were saved, in any strides."""

import pytest
import torch

from hi2_amd.experts import experts_mlp, gated, grouped_linear
from hi2_amd.moe import route
from hi2_amd.packed import combine

pytestmark = pytest.mark.gpu


def swapped(t):
    """The tensor with its last two dimensions' strides exchanged."""
    return t.transpose(-1, -2).contiguous().transpose(-1, -2) if t.dim() > 1 else \
        torch.stack([t, t], -1)[..., 0]


def thinned(t):
    """A constant tensor in one element."""
    return t.reshape(-1)[:1].reshape((1,) * t.dim()).expand(t.shape) \
        if t.numel() and bool((t == t.reshape(-1)[0]).all()) else t


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hook", [swapped, thinned])
@pytest.mark.parametrize("constant", [False, True])
def test_gradients_are_the_same(dev, dtype, hook, constant):
    g = torch.Generator().manual_seed(0)
    t, k, n, e = 70, 48, 40, 3

    def value(*shape):
        return torch.full(shape, 0.25, dtype=dtype, device=dev) if constant else \
            torch.randn(shape, generator=g).to(dtype).to(dev)

    x, w, up = value(t, k), value(e, n, k), value(2 * t, n)
    dy = torch.randn(2 * t, n, generator=g).to(dtype).to(dev)
    r = route(torch.randn(t, e, generator=g).to(dev), 2)
    out = []
    for pack in (lambda v: v, hook):
        xr, wr, ur = (v.clone().requires_grad_(True) for v in (x, w, up))
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda v: v):
            y = gated(grouped_linear(xr, wr, r.offs, r.rows, r.slots), ur)
        out.append(torch.autograd.grad(y, (xr, wr, ur), dy))
    assert all(torch.equal(a, b) for a, b in zip(*out))


def test_saved_on_the_host(dev):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(30, 24, generator=g).to(dev).requires_grad_(True)
    gate, up = (torch.randn(4, 16, 24, generator=g).to(dev).requires_grad_(True) for _ in range(2))
    down = torch.randn(4, 24, 16, generator=g).to(dev).requires_grad_(True)
    r = route(torch.randn(30, 4, generator=g).to(dev), 2)
    leaves = x, gate, up, down
    want = torch.autograd.grad(experts_mlp(x, r, gate, up, down).sum(), leaves)
    with torch.autograd.graph.save_on_cpu():
        y = experts_mlp(x, r, gate, up, down)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y.sum(), leaves), want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hook", [swapped, thinned])
def test_router_and_weighted_sum(dev, dtype, hook):
    g = torch.Generator().manual_seed(2)
    logits = torch.zeros(40, 8) + torch.arange(8.0)  # (rows alike)
    y = torch.full((80, 24), 0.5, dtype=dtype, device=dev)
    dy = torch.randn(40, 24, generator=g).to(dtype).to(dev)
    for constant in (False, True):
        lo = (torch.zeros(40, 8) if constant else logits + torch.randn(40, 8, generator=g)).to(dev)
        out = []
        for pack in (lambda v: v, hook):
            lr, yr = lo.clone().requires_grad_(True), y.clone().requires_grad_(True)
            with torch.autograd.graph.saved_tensors_hooks(pack, lambda v: v):
                r = route(lr, 2)
                z = combine(yr, r.slots, r.weights, None, dtype)
            out.append(torch.autograd.grad(z, (lr, yr), dy))
        assert all(torch.equal(a, b) for a, b in zip(*out))
