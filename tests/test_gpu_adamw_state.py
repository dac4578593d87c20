"""AdamW's state taken over by parameters of other types or sizes."""

import copy

import pytest
import torch

from hi2_amd.optim import AdamW

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def make(types, values, sizes=(300, 70, 5)):
    ps = [torch.nn.Parameter(torch.full((n,), 1.0, dtype=t).cuda()) for t, n in zip(types, sizes)]
    with torch.no_grad():
        for p, v in zip(ps, values):
            p.fill_(v)
    return ps, AdamW(ps, lr=0.25, weight_decay=0.0, betas=(0.5, 0.75))


@pytest.mark.parametrize("saved,loaded", [
    ((F32, BF16, F32), (F32, F32, F32)), ((F32, F32, F32), (F32, BF16, F32)),
    ((BF16, F32, BF16), (F32, F16, F32)), ((F16, BF16, F32), (F32, BF16, F16)),
])
@pytest.mark.parametrize("through_host", [False, True])
def test_counts_follow_their_parameters(dev, saved, loaded, through_host):
    """Parameters that have taken different numbers of steps keep them in a resume in other types:
    the next step is that of an optimizer of those types from the start."""
    values, taken = (1.0, 2.0, -1.0), (3, 1, 2)
    ps, opt = make(saved, values)
    qs, plain = make(loaded, values)
    for i in range(3):
        for p, q, n in zip(ps, qs, taken):
            for v in (p, q):
                v.grad = torch.full_like(v, 0.5) if i < n else None
        opt.step(), plain.step()
    state = copy.deepcopy(opt.state_dict())
    if through_host:
        state["state"] = {k: v.cpu() if isinstance(v, torch.Tensor) else v
                          for k, v in state["state"].items()}
    rs, other = make(loaded, values)
    other.load_state_dict(state)
    for r, q in zip(rs, qs):
        r.data.copy_(q.data)
        r.grad, q.grad = torch.full_like(r, 0.25), torch.full_like(q, 0.25)
    other.step(), plain.step()
    for r, q in zip(rs, qs):
        assert torch.equal(r, q)
    assert all(torch.equal(a, b) for a, b in zip(other.moments(), plain.moments()))


def test_a_state_of_other_sizes_is_refused(dev):
    """Also where they end in the same block of 256."""
    _, opt = make((F32, F32, F32), (1, 1, 1))
    _, other = make((F32, F32, F32), (1, 1, 1), (300, 70, 6))
    with pytest.raises(ValueError, match="other parameters"):
        other.load_state_dict(opt.state_dict())


def test_a_state_without_sizes_and_types(dev):
    """As states were before they named them: taken over by the same parameters."""
    ps, opt = make((F32, BF16, F32), (1, 2, 3))
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    ps[1].grad = None
    opt.step()
    state = copy.deepcopy(opt.state_dict())
    del state["state"]["sizes"], state["state"]["types"]
    _, other = make((F32, BF16, F32), (1, 2, 3))
    other.load_state_dict(state)
    assert torch.equal(other.state_dict()["state"]["steps"], opt.state_dict()["state"]["steps"])
    assert all(torch.equal(a, b) for a, b in zip(other.moments(), opt.moments()))


def test_empty_parameters_have_no_count(dev):
    ps, opt = make((BF16, F32, F32), (1, 2, 3), (0, 70, 5))
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    qs, other = make((F32, F32, BF16), (1, 2, 3), (0, 70, 5))
    other.load_state_dict(opt.state_dict())
    assert other.state_dict()["state"]["steps"].tolist() == [1, 1]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_between_parameters_there_are_zeros(dev, dtype, bits):
    """Also in the masters, and where eps is 0."""
    ps = [torch.nn.Parameter(torch.ones(n, dtype=dtype).cuda()) for n in (301, 255, 4097, 6, 512)]
    opt = AdamW(ps, lr=0.5, eps=0.0, state_bits=bits, master=True)
    for i in range(2):
        for p in ps:
            p.grad = torch.full_like(p, 0.5 - i)
        opt.step()
    between = torch.ones(opt.master.numel(), dtype=torch.bool, device="cuda")
    for p, a in zip(ps, opt.starts):
        between[a:a + p.numel()] = False
        assert torch.isfinite(p).all() and torch.equal(opt.master[a:a + p.numel()].to(dtype), p)
    for buffer in (opt.master, *opt.moments()):
        assert not buffer[between].any()


def test_no_copy_without_the_moments(dev):
    """A pickle held the options alone, and what was read back had no state to step with."""
    import pickle

    _, opt = make((F32, F32, F32), (1, 2, 3))
    for take in (copy.copy, copy.deepcopy, pickle.dumps):
        with pytest.raises(TypeError, match="state_dict"):
            take(opt)
    assert "lr" in repr(opt)
