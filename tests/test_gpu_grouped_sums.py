"""The tokens' gradient over slots: float32 sums of what the slots have, rounded once."""

import numpy as np
import pytest
import torch

from hi2_amd.experts import grouped_linear

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def routing(counts, tokens, top_k, seed):
    """(offs, rows, slots) of slots dealt to experts by counts."""
    rng = np.random.default_rng(seed)
    offs = np.concatenate([[0], np.cumsum(counts)])
    order = rng.permutation(tokens * top_k)
    assert offs[-1] == tokens * top_k
    slots = np.empty(tokens * top_k, np.int64)
    slots[order] = np.arange(tokens * top_k)
    return [torch.from_numpy(np.ascontiguousarray(v)).cuda() for v in
            (offs, order // top_k, slots.reshape(tokens, top_k))]


def grad_x(x, w, offs, rows, slots, dy):
    xr = x.clone().requires_grad_(True)
    return torch.autograd.grad(grouped_linear(xr, w, offs, rows, slots), xr, dy)[0]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("k", [8, 9, 72])
def test_slots_that_cancel(dev, dtype, k):
    """One slot has 1 + 2^-12, which neither 16-bit type holds, the other -1: their sum is 2^-12."""
    t = TYPES[dtype]
    offs, rows, slots = torch.tensor([0, 1, 2]), torch.tensor([0, 0]), torch.tensor([[0, 1]])
    w = torch.zeros(2, 16, k)
    w[:, :2] = 1.0
    dy = torch.zeros(2, 16)
    dy[0, 0], dy[0, 1], dy[1, 0] = 1.0, 2.0 ** -12, -1.0
    got = grad_x(torch.zeros(1, k, dtype=t).cuda(), w.to(t).cuda(), offs.cuda(), rows.cuda(),
                 slots.cuda(), dy.to(t).cuda())
    assert torch.equal(got, torch.full_like(got, 2.0 ** -12))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("n,k,counts,top_k", [
    (64, 96, [3, 0, 40, 21], 4),          # one tile an expert
    (40, 1001, [300, 45, 0, 39], 3),      # rows of odd length
    (4096, 130, [33, 97], 2),             # a contraction cut along its length
    (64, 1024, [9000, 0, 7031, 353], 4),  # many tiles, the last ones partial
    (72, 1100, [5000] * 6 + [4950, 5150], 5),  # the larger tiles, odd edges, half row tiles
    (64, 1024, [64] * 300, 8),            # many short ranges
])
def test_one_rounding(dev, dtype, n, k, counts, top_k):
    """Off by half a step of the type, and the float32 sums' own roundings: n products of a slot and
    top_k slots, each addition by up to a step (2^-23) of the magnitudes' sum."""
    t, e = TYPES[dtype], len(counts)
    offs, rows, slots = routing(counts, sum(counts) // top_k, top_k, 1)
    g = torch.Generator().manual_seed(2)
    x = torch.zeros(sum(counts) // top_k, k, dtype=t).cuda()
    w = (0.05 * torch.randn(e, n, k, generator=g)).to(t).cuda()
    dy = torch.randn(sum(counts), n, generator=g).to(t).cuda()
    got = grad_x(x, w, offs, rows, slots, dy)
    d, size = (torch.empty(sum(counts), k, dtype=torch.float64, device="cuda") for _ in range(2))
    o = offs.tolist()
    for i in range(e):
        at = slice(o[i], o[i + 1])
        d[at] = dy[at].double() @ w[i].double()
        size[at] = dy[at].double().abs() @ w[i].double().abs()
    want, size = d[slots].sum(1), size[slots].sum(1)
    f = torch.finfo(t)
    bound = (n + top_k + 8) * 2.0 ** -23 * size
    bound = bound * (1 + f.eps / 2) + f.eps / 2 * want.abs() + f.tiny * f.eps / 2
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())
    assert torch.equal(grad_x(x, w, offs, rows, slots, dy), got)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_slots_of_no_expert_add_zeros(dev, dtype):
    """A token one of whose slots lies behind the last range takes the other's gradient alone."""
    t = TYPES[dtype]
    offs = torch.tensor([0, 40, 40, 150]).cuda()
    slots = torch.stack([torch.arange(150), torch.arange(299, 149, -1)], 1)
    rows = torch.empty(300, dtype=torch.int64)
    rows[slots] = torch.arange(150)[:, None]
    g = torch.Generator().manual_seed(3)
    x, w = (torch.randn(s, generator=g).to(t).cuda() for s in ((150, 88), (3, 48, 88)))
    dy = torch.randn(300, 48, generator=g).to(t).cuda()
    dy[150:] = float("nan")
    got = grad_x(x, w, offs, rows.cuda(), slots.cuda(), dy)
    alone = grad_x(x, w, offs, rows[:150].cuda(), slots[:, :1].contiguous().cuda(), dy[:150])
    assert torch.equal(got, alone)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_no_slots_at_all(dev, dtype):
    """Slots outside give rows of NaN, also where there are none."""
    t, none = TYPES[dtype], torch.zeros(0, dtype=torch.int64).cuda()
    x, w = torch.ones(1, 40, dtype=t).cuda(), torch.ones(2, 8, 40, dtype=t).cuda()
    got = grad_x(x, w, torch.zeros(3, dtype=torch.int64).cuda(), none,
                 torch.zeros(1, 2, dtype=torch.int64).cuda(), torch.zeros(0, 8, dtype=t).cuda())
    assert got.shape == x.shape and torch.isnan(got).all()
