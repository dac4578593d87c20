"""Rows of the grouped products' operands far apart."""

import pytest
import torch

from hi2_amd import _lib
from hi2_amd.experts import grouped_linear

_lib_types = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


@pytest.mark.gpu
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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,k", [(56, 72), (40, 70), (13, 9), (300, 264)])
@pytest.mark.parametrize("pitch", [0, 8, 1 << 31, 1 << 40])
def test_the_pitch_of_one_row_does_not_count(dev, dtype, n, k, pitch):
    """One token of one expert through the C entries, with and without the workspace they ask for."""
    dt = _lib_types[dtype]
    g = torch.Generator().manual_seed(2)
    x, w, dy = (torch.randn(s, generator=g).to(dtype).to(dev) for s in ((1, k), (2, n, k), (1, n)))
    offs = torch.tensor([0, 0, 1], device=dev)
    zero = torch.zeros(1, dtype=torch.int64, device=dev)
    wide = dtype == torch.float32
    size = _lib.lib().hi2x_grouped_workspace_bytes
    for rows, own in ((None, False), (zero, True), (None, True)):
        out, dx, dw = (torch.full(s, float("nan"), dtype=dtype, device=dev)
                       for s in ((1, n), (1, k), (2, n, k)))
        spaces = []
        for what in range(3):
            bytes_ = size(what, dt, 1, pitch, 2, n, k, 1, rows is not None and what != 1,
                          n % 8 == 0 if what else k % 8 == 0, k % 8 == 0)
            assert bytes_ >= 0
            spaces.append((torch.empty(max(bytes_, 256), dtype=torch.uint8, device=dev).data_ptr(),
                           bytes_) if own else (None, 0))
        _lib.call("hi2x_grouped_linear", dev, x.data_ptr(), dt, pitch, 1, w.data_ptr(), 2, n, k,
                  _lib.ptr(rows), offs.data_ptr(), 1, out.data_ptr(), *spaces[0])
        _lib.call("hi2x_grouped_grad_x", dev, dy.data_ptr(), dt, pitch, w.data_ptr(), 2, n, k,
                  offs.data_ptr(), 1, None, 1, 1, dx.data_ptr(), *spaces[1])
        _lib.call("hi2x_grouped_grad_w", dev, dy.data_ptr(), dt, pitch, x.data_ptr(), pitch, 1, 2,
                  n, k, _lib.ptr(rows), offs.data_ptr(), 1, dw.data_ptr(), *spaces[2])
        torch.cuda.synchronize()
        # one product a result of dw: exact in float32, rounded once
        assert not dw[0].any()
        assert torch.equal(dw[1], (dy[0].double()[:, None] * x[0].double()).to(dtype)) or wide
        half = torch.finfo(dtype).eps / 2
        for got, want, mag, length in (
                (out[0], w[1].double() @ x[0].double(), w[1].double().abs() @ x[0].double().abs(), k),
                (dx[0], dy[0].double() @ w[1].double(), dy[0].double().abs() @ w[1].double().abs(),
                 n),
                (dw[1], dy[0].double()[:, None] * x[0].double(), 0.0, 1)):
            sums = (length + 8) * 2.0 ** -23 * mag
            bound = sums * (1 + half) + half * want.abs() + torch.finfo(dtype).tiny
            assert bool(((got.double() - want).abs() <= bound).all())


def test_one_row_and_a_workspace_for_its_copy():
    """On the host: a row whose length is not a multiple of 16 bytes is copied, wherever it begins."""
    size = _lib.lib().hi2x_grouped_workspace_bytes
    assert size(2, 2, 1, 72, 2, 40, 70, 1, 0, 1, 1) == size(2, 2, 1, 70, 2, 40, 70, 1, 0, 1, 0)
    assert size(2, 2, 1, 72, 2, 40, 72, 1, 0, 1, 1) == size(2, 2, 1, 1 << 40, 2, 40, 72, 1, 1, 1, 1)
