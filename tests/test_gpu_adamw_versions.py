"""The step is a write in place to autograd: graphs from before it do not go on with new weights."""

import numpy as np
import pytest
import torch

from hi2_amd.experts import grouped_linear
from hi2_amd.optim import AdamW


def test_versions_are_counted():
    """On the host: those with a gradient's address, once each; inference tensors have no count."""
    from hi2_amd import _tensors

    with torch.inference_mode():
        frozen = torch.zeros(3)
    ps = [torch.zeros(2), torch.zeros(3, requires_grad=True), frozen]
    before = [p._version for p in ps[:2]]
    addresses = np.array([0, 64, 64], dtype=np.uint64)
    _tensors.stepped(ps, addresses.ctypes.data)
    assert [p._version for p in ps[:2]] == [before[0], before[1] + 1]
    _tensors.stepped([], 0)
    with pytest.raises(RuntimeError, match="not a tensor"):
        _tensors.stepped([3], addresses.ctypes.data)
    with pytest.raises(TypeError):
        _tensors.stepped((), 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_backward_of_a_graph_from_before_the_step(dev, dtype, bits):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(6, 16, generator=g).to(dtype).to(dev).requires_grad_(True)
    w, v = (torch.nn.Parameter(torch.randn(2, 8, 16, generator=g).to(dtype).to(dev))
            for _ in range(2))
    offs = torch.tensor([0, 2, 6], device=dev)
    opt = AdamW([w, v], lr=0.1, state_bits=bits)
    kept = grouped_linear(x, v, offs)
    want, = torch.autograd.grad(kept, x, torch.ones_like(kept), retain_graph=True)
    y = grouped_linear(x, w, offs)
    y.backward(torch.ones_like(y), retain_graph=True)
    counts = w._version, v._version
    opt.step()
    assert (w._version, v._version) == (counts[0] + 1, counts[1])
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward(torch.ones_like(y))
    # v had no gradient and took no step
    assert torch.equal(torch.autograd.grad(kept, x, torch.ones_like(kept))[0], want)
    # a graph made anew takes the new weights
    y = grouped_linear(x, w, offs)
    y.backward(torch.ones_like(y))


@pytest.mark.gpu
def test_a_refused_step_counts_nothing(dev):
    a = torch.ones(300, device=dev, requires_grad=True)
    b = torch.ones(70, dtype=torch.bfloat16, device=dev, requires_grad=True)
    opt = AdamW([a, b])
    a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
    b.data = torch.ones(71, dtype=torch.bfloat16, device=dev)
    before = a._version
    with pytest.raises(RuntimeError, match="changed after construction"):
        opt.step()
    assert a._version == before
