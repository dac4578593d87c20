"""The AdamW step over many tensors: bit for bit against its definition in float32 operations (IEEE
numpy on the host), and that definition against 64 bits."""

import copy

import numpy as np
import pytest
import torch

from hi2_amd.optim import AdamW

B = 256
F = np.float32
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- the definition, in float32 (numpy rounds every operation by itself) ---------------------
def hold(x, steps):
    """Magnitudes [n] as codes and units of blocks of 256."""
    blocks = x.reshape(-1, B)
    d = blocks.max(1, keepdims=True) * F(1.0 / steps ** 2)
    d = np.where(d >= F(2.0 ** -126), d, F(0))
    r = np.divide(F(1), d, out=np.zeros_like(d), where=d > 0)
    z = (blocks * r).astype(np.float64)
    # the nearest code by counting the borders (c + 1/2)^2 at or below z
    c = np.searchsorted((np.arange(steps) + 0.5) ** 2, z.ravel(), side="right").reshape(z.shape)
    return c.astype(np.int64), d


def held_m(m):
    c, d = hold(np.abs(m), 127)
    c = np.where(m.reshape(-1, B) < 0, -c, c)
    return ((c * np.abs(c)).astype(F) * d).ravel()


def held_v(v):
    s = np.sqrt(v)
    c, d = hold(s, 255)
    c = np.where((c == 0) & (s.reshape(-1, B) > 0), 1, c)
    s = ((c * c).astype(F) * d).ravel()
    return s * s


def adamw(p, g, m, v, t, lr, wd, b1=0.9, b2=0.999, eps=1e-8):
    """One step of flat float32 arrays; t counts it."""
    c1, c2 = 1.0 - b1 ** t, 1.0 - b2 ** t
    m = m * F(b1) + g * F(1.0 - b1)
    v = v * F(b2) + (g * g) * F(1.0 - b2)
    q = m / (np.sqrt(v) * F(1.0 / np.sqrt(c2)) + F(eps))
    return p * F(1.0 - lr * wd) - q * F(lr / c1), m, v


def test_definition_against_64_bits():
    rng = np.random.default_rng(0)
    p, g, m, v = (rng.standard_normal(4096) for _ in range(4))
    v = v * v
    p1, m1, v1 = adamw(*(a.astype(F) for a in (p, g, m, v)), 7, 1e-2, 0.1)
    m2, v2 = 0.9 * m + 0.1 * g, 0.999 * v + 0.001 * g * g
    p2 = p * (1 - 1e-3) - 1e-2 * (m2 / (1 - 0.9 ** 7)) / (np.sqrt(v2 / (1 - 0.999 ** 7)) + 1e-8)
    u = 2.0 ** -24
    # four roundings of inputs, factors, products and the sum each, on the sum of magnitudes
    assert (np.abs(m1 - m2) <= 8 * u * (0.9 * np.abs(m) + 0.1 * np.abs(g))).all()
    assert (np.abs(v1 - v2) <= 8 * u * v2).all()
    step = 1e-2 * (np.abs(0.9 * m) + np.abs(0.1 * g)) / (1 - 0.9 ** 7) / np.sqrt(
        v2 / (1 - 0.999 ** 7))
    assert (np.abs(p1 - p2) <= 8 * u * np.abs(p) + 24 * u * step).all()


def test_codes_keep_what_they_promise():
    rng = np.random.default_rng(1)
    m = (rng.standard_normal(64 * B) * np.exp(3 * rng.standard_normal(64 * B))).astype(F)
    top = np.abs(m).reshape(-1, B).max(1).repeat(B)
    # a code's square is off by at most c + 1/4 units of top / 127^2 where c^2 is the value
    c = np.sqrt(np.abs(m) / top) * 127
    assert (np.abs(held_m(m) - m) <= (c + 0.26) * top / 127 ** 2 + 1e-6 * np.abs(m)).all()
    v = m * m
    assert (held_v(v) > 0).all()
    assert not held_v(np.zeros(B, F)).any() and not held_m(np.zeros(B, F)).any()
    once = held_m(m)
    assert (np.abs(held_m(once) - once) <= 4 * 2.0 ** -24 * np.abs(once)).all()


# ---- the kernel ------------------------------------------------------------------------------
SIZES = [1, 3, 255, 256, 257, 4095, 4096, 4097, 20000, 64, 37 * 129]


def flat(t, dtype=None):
    return t.detach().cpu().float().numpy().ravel().astype(F)


def make(sizes, dtype, seed, **options):
    g = torch.Generator().manual_seed(seed)
    ps = [torch.nn.Parameter((0.1 * torch.randn(n, generator=g)).to(dtype).cuda())
          for n in sizes]
    return ps, AdamW(ps, **options)


def grads(ps, seed, scale=1e-2):
    g = torch.Generator().manual_seed(seed)
    for p in ps:
        s = scale * torch.exp(torch.randn(1, generator=g))
        p.grad = (s * torch.randn(p.shape, generator=g)).to(p.dtype).cuda()


def pad(x):
    out = np.zeros(-(-len(x) // B) * B, F)
    out[:len(x)] = x
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_steps_bit_for_bit(dev, dtype, bits, master):
    t = TYPES[dtype]
    ps, opt = make(SIZES, t, 1, lr=3e-3, weight_decay=0.1, state_bits=bits, master=master)
    mine = [pad(flat(p)) for p in ps]
    m, v = [np.zeros_like(a) for a in mine], [np.zeros_like(a) for a in mine]
    for step in range(1, 5):
        grads(ps, 10 + step)
        opt.step()
        gm, gv = (x.cpu().numpy() for x in opt.moments())
        for i, (p, a) in enumerate(zip(ps, opt.starts)):
            q, m[i], v[i] = adamw(mine[i], pad(flat(p.grad)), m[i], v[i], step, 3e-3, 0.1)
            if bits == 8:
                m[i], v[i] = held_m(m[i]), held_v(v[i])
            n = p.numel()
            stored = torch.from_numpy(q[:n]).to(t)
            assert torch.equal(p.detach().cpu(), stored), (step, n)
            mine[i] = q if t == torch.float32 or master else pad(flat(stored))
            assert np.array_equal(gm[a:a + len(m[i])], m[i]), (step, n)
            assert np.array_equal(gv[a:a + len(v[i])], v[i]), (step, n)
            if opt.master is not None:
                assert np.array_equal(opt.master[a:a + n].cpu().numpy(), q[:n])


@pytest.mark.gpu
def test_types_groups_and_missing_gradients(dev):
    """Two types in three groups of their own options; a parameter without a gradient keeps its
    value, its moments and its count."""
    g = torch.Generator().manual_seed(0)
    a, b, c, d = (torch.nn.Parameter(torch.randn(s, generator=g).to(t).cuda()) for s, t in
                  (((40, 30), torch.float32), ((500,), torch.bfloat16), ((7, 9), torch.float32),
                   ((0,), torch.float32)))
    opt = AdamW([dict(params=[a, d], lr=1e-2), dict(params=[b], betas=(0.5, 0.9), eps=1e-4),
                 dict(params=[c], weight_decay=0.0)], lr=1e-3, weight_decay=0.05)
    grads([a, b, c], 1)
    before = flat(a).copy()
    opt.step()
    pa, ma, va = adamw(before, flat(a.grad), 0 * before, 0 * before, 1, 1e-2, 0.05)
    assert np.array_equal(flat(a), pa)
    kept = [flat(x).copy() for x in (a, c)]
    a.grad = None
    opt.param_groups[2]["lr"] = 0.5
    opt.step()
    assert np.array_equal(flat(a), kept[0]) and not np.array_equal(flat(c), kept[1])
    m, _ = opt.moments()
    assert np.array_equal(m[:1200].cpu().numpy(), ma)
    grads([a], 3)
    opt.step()
    want, _, _ = adamw(pa, flat(a.grad), ma, va, 2, 1e-2, 0.05)  # its second step
    assert np.array_equal(flat(a), want)
    opt.zero_grad()
    opt.step()  # nothing to do
    assert np.array_equal(flat(a), want)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_and_groups(dev, bits):
    """More tensors and groups than one launch takes."""
    sizes = [1 + (37 * i) % 700 for i in range(450)]
    g = torch.Generator().manual_seed(0)
    ps = [torch.nn.Parameter(torch.randn(n, generator=g).cuda()) for n in sizes]
    groups = [dict(params=ps[i:i + 10], lr=1e-3 * (1 + i // 10)) for i in range(0, 450, 10)]
    opt = AdamW(groups, weight_decay=0.1, state_bits=bits)
    before = [flat(p).copy() for p in ps]
    grads(ps, 1)
    opt.step()
    for i, p in enumerate(ps):
        want, _, _ = adamw(before[i], flat(p.grad), 0 * before[i], 0 * before[i], 1,
                           1e-3 * (1 + i // 10), 0.1)
        assert np.array_equal(flat(p), want), i


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(TYPES))
def test_views_of_any_alignment(dev, dtype):
    t = TYPES[dtype]
    base, gbase = torch.zeros(3000, dtype=t).cuda(), torch.zeros(3000, dtype=t).cuda()
    base.copy_(torch.randn(3000, generator=torch.Generator().manual_seed(0)))
    gbase.copy_(torch.randn(3000, generator=torch.Generator().manual_seed(1)))
    guard = base.clone()
    spans = [(1, 700), (703, 1300), (1301, 1302), (1500, 2999)]
    ps = [torch.nn.Parameter(base[a:b]) for a, b in spans]
    for p, (a, b) in zip(ps, spans):
        p.grad = gbase[a - 1:b - 1]
    opt = AdamW(ps, lr=1e-2)
    opt.step()
    for a, b in spans:
        x = guard[a:b].float().cpu().numpy()
        want, _, _ = adamw(x, flat(gbase[a - 1:b - 1]), 0 * x, 0 * x, 1, 1e-2, 1e-2)
        assert torch.equal(base[a:b].cpu(), torch.from_numpy(want).to(t))
        guard[a:b] = base[a:b]
    assert torch.equal(base, guard)  # nothing else was written


@pytest.mark.gpu
def test_gradients_that_are_not_contiguous(dev):
    p = torch.nn.Parameter(torch.randn(30, 50).cuda())
    p.grad = torch.randn(50, 30).cuda().t()
    x = flat(p).copy()
    opt = AdamW([p])
    opt.step()
    want, _, _ = adamw(x, flat(p.grad), 0 * x, 0 * x, 1, 1e-3, 1e-2)
    assert np.array_equal(flat(p), want)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_nan_and_infinity(dev, bits):
    """They show, and stay in their element (with 8 bits: in their block of 256)."""
    p = torch.nn.Parameter(torch.zeros(1024).cuda())
    opt = AdamW([p], lr=1e-2, weight_decay=0.0, state_bits=bits)
    p.grad = torch.ones(1024).cuda()
    p.grad[300], p.grad[600] = float("nan"), float("inf")
    opt.step()
    bad = torch.isnan(p.detach()).nonzero().ravel().tolist()
    assert bad == [300, 600]
    m, v = opt.moments()
    if bits == 32:
        assert torch.isnan(m).nonzero().ravel().tolist() == [300] and torch.isinf(v[600])
    else:
        assert torch.isnan(m[256:768]).all() and torch.isnan(v[256:768]).all()
        assert torch.isfinite(m[:256]).all() and torch.isfinite(v[768:]).all()
    # gradients of zero and the smallest ones
    q = torch.nn.Parameter(torch.ones(512).cuda())
    opt = AdamW([q], lr=1e-2, weight_decay=0.0, state_bits=bits)
    q.grad = torch.zeros(512).cuda()
    q.grad[256:] = 1e-42
    for _ in range(3):
        opt.step()
    assert torch.isfinite(q).all() and torch.equal(q.detach(), torch.ones(512).cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count_on(dev, bits):
    """A step captured in a graph: replays give what eager steps give, the learning rate read from
    its tensor in each."""
    lr = torch.tensor(1e-2).cuda()
    ps, opt = make([5000, 77], torch.float32, 3, lr=lr, state_bits=bits)
    qs, eager = make([5000, 77], torch.float32, 3, lr=1e-2, state_bits=bits)
    grads(ps, 50)
    for p, q in zip(ps, qs):
        q.grad = p.grad.clone()
    opt.step(), eager.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for i in range(4):
        g = torch.Generator().manual_seed(60 + i)
        for p, q in zip(ps, qs):
            p.grad.copy_(torch.randn(p.shape, generator=g))
            q.grad.copy_(p.grad)
        rate = float(torch.tensor(1e-2 / (1 + i)))
        lr.fill_(rate)
        eager.param_groups[0]["lr"] = rate
        graph.replay()
        eager.step()
        torch.cuda.synchronize()
        for p, q in zip(ps, qs):
            assert torch.equal(p, q), i
        for a, b in zip(opt.moments(), eager.moments()):
            assert torch.equal(a, b), i


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_state_goes_round(dev, bits):
    ps, opt = make([700, 300], torch.bfloat16, 1, state_bits=bits, master=True)
    for i in range(3):
        grads(ps, i)
        opt.step()
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    other = AdamW(qs, lr=5.0, state_bits=bits, master=True)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    assert other.param_groups[0]["lr"] == opt.param_groups[0]["lr"]
    # the same through float32 moments, from the one width to the other and back
    m, v = (x.clone() for x in opt.moments())
    third = AdamW([torch.nn.Parameter(p.detach().clone()) for p in ps], state_bits=32)
    third.load_moments(m, v, step=3)
    assert all(torch.equal(a, b) for a, b in zip(third.moments(), (m, v)))
    grads(ps, 9)
    for p, q in zip(ps, qs):
        q.grad = p.grad.clone()
    opt.step(), other.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))
    assert torch.equal(opt.master, other.master)
    assert all(torch.equal(a, b) for a, b in zip(opt.moments(), other.moments()))
    junk = torch.full_like(m, 7.0)
    other.load_moments(junk, junk)
    assert not other.moments()[0][700:768].any()


@pytest.mark.gpu
def test_scheduler_and_closure(dev):
    p = torch.nn.Parameter(torch.ones(10).cuda())
    opt = AdamW([p], lr=1.0)
    sched = torch.optim.lr_scheduler.StepLR(opt, 1, 0.1)

    def closure():
        opt.zero_grad()
        loss = (p * p).sum()
        loss.backward()
        return loss

    assert float(opt.step(closure)) == 10.0
    sched.step()
    assert abs(opt.param_groups[0]["lr"] - 0.1) < 1e-12


@pytest.mark.gpu
def test_refusals(dev):
    p = torch.nn.Parameter(torch.zeros(8, 4).cuda())
    for match, args in [("state_bits", dict(state_bits=16)), ("lr -1", dict(lr=-1.0)),
                        ("betas", dict(betas=(1.0, 0.9))), ("eps", dict(eps=-1e-8)),
                        ("weight_decay", dict(weight_decay=-1.0)),
                        ("one float32", dict(lr=torch.tensor(1e-3)))]:
        with pytest.raises(ValueError, match=match):
            AdamW([p], **args)
    with pytest.raises(ValueError, match="float32, float16"):
        AdamW([torch.nn.Parameter(torch.zeros(4, dtype=torch.float64).cuda())])
    with pytest.raises(ValueError, match="not contiguous"):
        AdamW([torch.nn.Parameter(torch.zeros(4, 6).cuda().t())])
    with pytest.raises(RuntimeError, match="MI355X only"):
        AdamW([torch.nn.Parameter(torch.zeros(4))])
    opt = AdamW([p])
    with pytest.raises(RuntimeError, match="cannot be added"):
        opt.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(4).cuda())]))
    p.grad = torch.zeros(8, 4).cuda()
    p.data = torch.zeros(4, 4).cuda()
    with pytest.raises(RuntimeError, match="changed after construction"):
        opt.step()
    p.data = torch.zeros(8, 4).half().cuda()
    with pytest.raises(RuntimeError, match="changed after construction"):
        opt.step()
    q = torch.nn.Parameter(torch.zeros(64).cuda())
    a, b = AdamW([q]), AdamW([q], state_bits=8)
    with pytest.raises(ValueError, match="another width"):
        a.load_state_dict(b.state_dict())
    with pytest.raises(ValueError, match="expected float32"):
        a.load_moments(torch.zeros(64).cuda(), torch.zeros(64).cuda())
    with pytest.raises(RuntimeError, match="no masters"):
        a.load_masters()
