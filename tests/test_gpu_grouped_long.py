"""Long contractions in float32: running sums of 256 products, added to one another."""

import pytest
import torch

from hi2_amd.experts import grouped_linear

pytestmark = pytest.mark.gpu


def bound(length, magnitude):
    """Each addition rounds by up to a step (2^-23) of the magnitudes' sum: 256 of a running sum, one
    for each of them."""
    return (256 + length / 256 + 8) * 2.0 ** -23 * magnitude


def all_three(x, w, offs, dy):
    xr, wr = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = grouped_linear(xr, wr, offs)
    return (y.detach(), *torch.autograd.grad(y, (xr, wr), dy))


@pytest.mark.parametrize("length", [300, 6408, 14336])
def test_a_large_first_product(dev, length):
    """2^24 and quarters: a running sum of all of them would lose every quarter."""
    ones = torch.ones(length, device=dev)
    line = torch.full((length,), 0.25, device=dev)
    line[0] = 2.0 ** 24
    total = line.double().sum()

    def check(got):
        assert bool(((got.double() - total).abs() <= bound(length, total)).all())

    # the product, over K
    w = ones.expand(1, 5, length).contiguous()
    check(all_three(line.expand(3, length).contiguous(), w, torch.tensor([0, 3], device=dev),
                    torch.zeros(3, 5, device=dev))[0])
    # the tokens' gradient, over N
    w = ones[:, None].expand(1, length, 5).contiguous()
    check(all_three(torch.zeros(3, 5, device=dev), w, torch.tensor([0, 3], device=dev),
                    line.expand(3, length).contiguous())[1])
    # the weights' gradient, over slots
    check(all_three(ones[:, None].expand(length, 3).contiguous(), torch.zeros(1, 5, 3, device=dev),
                    torch.tensor([0, length], device=dev),
                    line[:, None].expand(length, 5).contiguous())[2])


@pytest.mark.parametrize("n,k,counts", [(70, 6408, [3, 0, 9]), (9001, 33, [40, 1]),
                                        (40, 66, [7001, 0, 255, 257])])
def test_against_64_bits(dev, n, k, counts):
    g = torch.Generator().manual_seed(1)
    e, s = len(counts), sum(counts)
    x, w, dy = (torch.randn(v, generator=g).to(dev) for v in ((s, k), (e, n, k), (s, n)))
    offs = torch.tensor([sum(counts[:i]) for i in range(e + 1)], device=dev)
    y, dx, dw = all_three(x, w, offs, dy)
    o = offs.tolist()
    for i in range(e):
        a, b, d = x[o[i]:o[i + 1]].double(), w[i].double(), dy[o[i]:o[i + 1]].double()
        for got, p, q, length in ((y[o[i]:o[i + 1]], a, b.T, k), (dx[o[i]:o[i + 1]], d, b, n),
                                  (dw[i], d.T, a, counts[i])):
            assert bool(((got.double() - p @ q).abs() <= bound(length, p.abs() @ q.abs()) + 1e-30)
                        .all())
