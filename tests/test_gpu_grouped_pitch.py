"""Rows of the grouped products' operands far apart."""

import pytest
import torch

from hi2_amd.experts import grouped_linear

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("stride", [(1 << 21) - 8, 1 << 21, (1 << 21) + 1])
@pytest.mark.parametrize("indexed", [False, True])
def test_rows_a_sequence_apart(dev, dtype, stride, indexed):
    """The last token of each long sequence: x, and the gradient that comes back, give what they
    give as contiguous tensors."""
    t, k, n = 40, 72, 56
    g = torch.Generator().manual_seed(1)
    offs = torch.tensor([0, 11, 11, 40], device=dev)
    rows = torch.randperm(t, generator=g).to(dev) if indexed else None
    slots = None
    if indexed:
        slots = torch.empty_like(rows)
        slots[rows] = torch.arange(t, device=dev)
        slots = slots[:, None]
    w = torch.randn(3, n, k, generator=g).to(dtype).to(dev)
    near = torch.randn(t, k, generator=g).to(dtype).to(dev)
    dy = torch.randn(t, n, generator=g).to(dtype).to(dev)
    base = torch.empty(t * stride, dtype=dtype, device=dev)
    far, dfar = (torch.as_strided(base, (t, c), (stride, 1), o) for c, o in ((k, 0), (n, 1024)))
    far.copy_(near), dfar.copy_(dy)
    out = []
    for x, d in ((near, dy), (far, dfar)):
        xr, wr = x.detach().requires_grad_(True), w.clone().requires_grad_(True)
        y = grouped_linear(xr, wr, offs, rows, slots)
        out.append((y, *torch.autograd.grad(y, (xr, wr), d)))
        with torch.no_grad():
            assert torch.equal(grouped_linear(x, w, offs, rows), y)
    assert all(torch.equal(a, b) for a, b in zip(*out))
