"""Products grouped by expert where no slot is: empty results, gradients of zero."""

import pytest
import torch

from hi2_amd.experts import grouped_linear

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,k", [(16, 32), (5, 7), (300, 260)])
@pytest.mark.parametrize("tokens", [0, 1, 5])
def test_no_slots_but_tokens(dev, dtype, n, k, tokens):
    """A batch none of whose tokens has a slot: the weights' gradient is zero, whatever x has."""
    none = torch.zeros(0, dtype=torch.int64, device=dev)
    offs = torch.zeros(4, dtype=torch.int64, device=dev)
    for x in (torch.full((tokens, k), float("nan"), dtype=dtype, device=dev),
              torch.ones(tokens, k + 3, dtype=dtype, device=dev)[:, 3:]):
        w = torch.ones(3, n, k, dtype=dtype, device=dev, requires_grad=True)
        y = grouped_linear(x, w, offs, none)
        assert y.shape == (0, n) and y.dtype == dtype
        dw, = torch.autograd.grad(y, w, torch.zeros_like(y))
        assert dw.shape == w.shape and torch.equal(dw, torch.zeros_like(w))
        with torch.no_grad():
            assert grouped_linear(x, w, offs, none).shape == (0, n)


def test_no_slots_and_no_rows(dev):
    offs = torch.zeros(3, dtype=torch.int64, device=dev)
    x = torch.zeros(0, 8, device=dev, requires_grad=True)
    w = torch.ones(2, 4, 8, device=dev, requires_grad=True)
    y = grouped_linear(x, w, offs)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert dx.shape == (0, 8) and torch.equal(dw, torch.zeros_like(w))
