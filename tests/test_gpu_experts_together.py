"""Training steps of an MoE layer as they are run: latents decoded, tokens routed, the experts' MLP and
its gradients, AdamW; and the products and the activation against differences and far apart in
memory."""

from types import SimpleNamespace

import pytest
import torch

from hi2_amd.experts import experts_mlp, gated, grouped_linear
from hi2_amd.moe import route
from hi2_amd.optim import AdamW

pytestmark = pytest.mark.gpu


def _fake_quantised(n, k, dev, seed):
    """A fake-quantised Linear of two ladders with a transform."""
    g = torch.Generator(device=dev).manual_seed(seed)
    order = torch.randperm(n, generator=g, device=dev)
    groups = []
    for rows, nbits, block in ((order[: n // 2], 4, 32), (order[n // 2:], 8, 64)):
        m = rows.numel()
        consts = torch.stack([torch.full((m,), -0.15, device=dev),
                              torch.full((m,), 2e-4, device=dev),
                              torch.full((m,), 1e-4, device=dev)], 1).half()
        lo, st = (torch.rand(m, k // block, generator=g, device=dev) * 255 for _ in range(2))
        groups.append(SimpleNamespace(rows=rows.sort().values, consts=consts, nbits=nbits,
                                      block=block, lo_u=lo.requires_grad_(),
                                      step_u=st.requires_grad_()))
    latent = (torch.randn(n, k, generator=g, device=dev) * 0.05).requires_grad_()
    return SimpleNamespace(
        latent=latent, unit=torch.ones(0, device=dev), groups=groups,
        had=(torch.rand(k // 16, generator=g, device=dev) < 0.5).to(torch.uint8),
        col_scale=(torch.rand(k, generator=g, device=dev) + 0.5).half(), has_had=True,
        has_scale=True)


def _leaves(fq):
    return [fq.latent] + [p for g in fq.groups for p in (g.lo_u, g.step_u)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_distilled_experts_take_their_steps(dev, dtype):
    """Three steps of an MoE layer's distillation: the gradients of the decoded weights are those of
    the same layer in 64 bits, what reaches the latents is the decode's gradient of them, and every
    parameter takes AdamW's step of its gradient."""
    from hi2_amd.qad_kernel import original

    experts, top_k, hidden, inter, tokens = 4, 2, 128, 64, 90
    layers = [[_fake_quantised(n, k, dev, 10 * i + e) for e in range(experts)]
              for i, (n, k) in enumerate(((inter, hidden), (inter, hidden), (hidden, inter)))]
    params = [p for layer in layers for fq in layer for p in _leaves(fq)]
    lr, b1, b2, eps, wd = 1e-3, 0.9, 0.999, 1e-8, 1e-2
    opt = AdamW(params, lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd)
    g = torch.Generator().manual_seed(3)
    state = [[v.new_zeros(v.shape, dtype=torch.float64) for _ in range(3)] for v in params]
    for step in (1, 2, 3):
        x = torch.randn(tokens, hidden, generator=g).to(dev).to(dtype)
        logits = torch.randn(tokens, experts, generator=g).to(dev)
        dy = torch.randn(tokens, hidden, generator=g).to(dev).to(dtype)
        routing = route(logits, top_k)
        decoded = [[original(fq) for fq in layer] for layer in layers]
        weights = [torch.stack(layer).to(dtype) for layer in decoded]
        for w in weights + [w for layer in decoded for w in layer]:
            w.retain_grad()
        y = experts_mlp(x, routing, *weights)
        opt.zero_grad()
        y.backward(dy)
        # the layer in 64 bits
        w64 = [w.detach().double().requires_grad_(True) for w in weights]
        h = torch.nn.functional.silu(torch.matmul(w64[0], x.double().T)) * \
            torch.matmul(w64[1], x.double().T)
        every = torch.matmul(w64[2], h).permute(2, 0, 1)
        picked = every.gather(1, routing.index[..., None].expand(-1, -1, hidden))
        want = (picked * routing.weights.detach().double().view(tokens, top_k, 1)).sum(1)
        # (up to seven roundings on the way, each half a step of its values, as norms at most added)
        rel = 8 * torch.finfo(dtype).eps / 2 + 1e-6
        assert float((y.detach().double() - want).norm()) <= rel * float(want.norm())
        for got, ref in zip(weights, torch.autograd.grad(want, w64, dy.double())):
            assert float((got.grad.double() - ref).norm()) <= rel * float(ref.norm())
        # through the decode
        for layer, outs, w in zip(layers, decoded, weights):
            for e, (fq, out) in enumerate(zip(layer, outs)):
                assert torch.equal(out.grad, w.grad[e].to(out.dtype))
                again = torch.autograd.grad(original(fq), _leaves(fq), out.grad)
                assert all(torch.equal(p.grad, a) for p, a in zip(_leaves(fq), again))
        # the step: m, v and the magnitude of what was added up for m, which bounds its roundings
        before = [p.detach().double().clone() for p in params]
        opt.step()
        for p, p0, (m, v, big) in zip(params, before, state):
            d = p.grad.double()
            m.mul_(b1).add_((1 - b1) * d)
            big.mul_(b1).add_((1 - b1) * d.abs())
            v.mul_(b2).add_((1 - b2) * d * d)
            root = v.sqrt() / (1 - b2 ** step) ** 0.5 + eps
            move = lr / (1 - b1 ** step)
            expected = p0 * (1 - lr * wd) - move * m / root
            # m: three roundings a step; the quotient: v's three a step, halved by the root, and 8
            u = 2.0 ** -24
            bound = u * (3 * p0.abs() + move / root * (3 * step * big + (2 * step + 8) * m.abs()))
            assert bool(((p.detach().double() - expected).abs() <= bound + 1e-30).all())
    m, v = opt.moments()
    for p, at, (m64, v64, big) in zip(params, opt.starts, state):
        got = m[at:at + p.numel()].view(p.shape).double()
        assert bool(((got - m64).abs() <= 9 * 2.0 ** -24 * big + 1e-38).all())


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
def test_gated_gradients_against_differences(dev, act):
    """Central differences, element by element: off by the third derivative (below 2 of each
    activation away from relu's corner) and by the values' roundings (8 at most) over the step."""
    g = torch.Generator().manual_seed(1)
    gate, up = ((2 * torch.randn(33, 70, generator=g)).to(dev) for _ in range(2))
    h = 2.0 ** -6
    a, b = gate.clone().requires_grad_(True), up.clone().requires_grad_(True)
    out = gated(a, b, act)
    d_gate, d_up = torch.autograd.grad(out, (a, b), torch.ones_like(out))
    for got, hi, lo, bend in ((d_gate, gated(gate + h, up, act), gated(gate - h, up, act), up.abs()),
                              (d_up, gated(gate, up + h, act), gated(gate, up - h, act), 0 * up)):
        want = (hi.double() - lo.double()) / (2 * h)
        # the step itself is rounded too: gate + h is off by half a step of the sum
        noise = 2.0 ** -24 * (8 * out.detach().abs() + 8 * (gate.abs() + up.abs() + 1) *
                              (1 + up.abs()) * 1.2) / h
        off = (got.double() - want).abs()
        keep = gate.abs() > 2 * h if act == "relu" else torch.ones_like(gate, dtype=torch.bool)
        assert bool((off <= h * h / 3 * bend + noise)[keep].all())


def test_product_gradients_against_differences(dev):
    """The product is linear in x and in w, so a difference along a direction is the gradient's
    product with it but for the sums' roundings."""
    g = torch.Generator().manual_seed(2)
    logits = torch.randn(50, 6, generator=g).to(dev)
    r = route(logits, 3)
    x, w = torch.randn(50, 40, generator=g).to(dev), torch.randn(6, 24, 40, generator=g).to(dev)
    dy = torch.randn(150, 24, generator=g).to(dev)
    xr, wr = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(grouped_linear(xr, wr, r.offs, r.rows, r.slots), (xr, wr), dy)

    def value(a, b):
        return float((grouped_linear(a, b, r.offs, r.rows).double() * dy.double()).sum())

    ux, uw = torch.randn(x.shape, generator=g).to(dev), torch.randn(w.shape, generator=g).to(dev)
    # sums of 40 (and 24, 3 and a range's) products, each rounding a step of the magnitudes' sum
    size = float((grouped_linear(x.abs() + ux.abs(), w.abs() + uw.abs(), r.offs, r.rows).double() *
                  dy.abs().double()).sum())
    for got, want in (((dx.double() * ux).sum(), value(x + ux, w) - value(x - ux, w)),
                      ((dw.double() * uw).sum(), value(x, w + uw) - value(x, w - uw))):
        assert abs(float(got) - want / 2) <= 200 * 2.0 ** -23 * size


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_farther_apart_than_32_bits_of_offsets(dev, dtype):
    """Tokens 2.3 GB apart: their rows are brought together first, in the order of the slots."""
    width = 2300000000 // 1100 // dtype.itemsize // 8 * 8
    far = torch.empty(1100, width, dtype=dtype, device=dev)[:, 8:96]
    g = torch.Generator().manual_seed(4)
    x = torch.randn(1100, 88, generator=g).to(dtype).to(dev)
    far.copy_(x)
    r = route(torch.randn(1100, 5, generator=g).to(dev), 2)
    w = torch.randn(5, 72, 88, generator=g).to(dtype).to(dev)
    dy = torch.randn(2200, 72, generator=g).to(dtype).to(dev)
    rows = r.rows.clone()
    rows[7] = 1100
    out = []
    for v in (far, x):
        a, b = v.detach().requires_grad_(True), w.clone().requires_grad_(True)
        y = grouped_linear(a, b, r.offs, rows, r.slots)
        out.append((y, *torch.autograd.grad(y, (a, b), dy)))
    assert torch.isnan(out[1][0][7]).all()
    for got, want in zip(*out):
        assert torch.equal(torch.nan_to_num(got, 1e9), torch.nan_to_num(want, 1e9))


@pytest.mark.parametrize("slots", [30, 700])
def test_weights_past_32_bits_of_offsets(dev, slots):
    """4.7 GB of weights: the last expert's are where they should be, and so is their gradient."""
    e, n, k = 70, 8192, 4096
    t = torch.bfloat16
    w = torch.empty(e, n, k, dtype=t, device=dev)
    g = torch.Generator().manual_seed(5)
    for i in (0, e - 1):
        w[i] = (torch.randn(n, k, generator=g) * 0.05).to(t)
    w.requires_grad_(True)
    offs = torch.zeros(e + 1, dtype=torch.int64)
    offs[1:e] = 9
    offs[e] = slots
    offs = offs.to(dev)
    x = torch.randn(slots, k, generator=g).to(t).to(dev).requires_grad_(True)
    dy = torch.randn(slots, n, generator=g).to(t).to(dev)
    y = grouped_linear(x, w, offs)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert not dw[1:e - 1].any()
    # float32 sums of 16-bit products, each addition a step of the magnitudes' sum, then a rounding
    for i, at in ((0, slice(0, 9)), (e - 1, slice(9, slots))):
        a, b, d = x.detach()[at].double(), w.detach()[i].double(), dy[at].double()
        for got, want, size, length in (
                (y[at], a @ b.T, a.abs() @ b.abs().T, k), (dx[at], d @ b, d.abs() @ b.abs(), n),
                (dw[i], d.T @ a, d.abs().T @ a.abs(), slots)):
            bound = 2.0 ** -8 * want.abs() + (length + 8) * 2.0 ** -23 * 1.01 * size + 1e-38
            assert bool(((got.detach().double() - want).abs() <= bound).all())


def test_a_step_is_taken_whole_or_not(dev):
    """A parameter that no longer fits refuses the step before any other has taken it."""
    a = torch.ones(300, device=dev, requires_grad=True)
    b = torch.ones(70, dtype=torch.bfloat16, device=dev, requires_grad=True)
    opt = AdamW([a, b], lr=0.1)
    a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
    b.data = torch.ones(71, dtype=torch.bfloat16, device=dev)
    with pytest.raises(RuntimeError, match="changed after construction"):
        opt.step()
    assert bool((a == 1).all()) and not opt.moments()[0].any()


def test_parameters_that_share_memory_are_refused(dev):
    base = torch.zeros(100, device=dev)
    a, b = base[:60].requires_grad_(True), base[59:].requires_grad_(True)
    with pytest.raises(ValueError, match="share memory"):
        AdamW([a, b])
    with pytest.raises(ValueError, match="share memory|some parameters appear in more"):
        AdamW([dict(params=[a]), dict(params=[base[:60].requires_grad_(True)])])
    AdamW([a, base[60:].requires_grad_(True)])


def test_a_state_is_taken_over_whole_or_not(dev):
    def make(lr):
        ps = [torch.ones(5, device=dev, requires_grad=True) for _ in range(2)]
        return AdamW([dict(params=[ps[0]], lr=lr), dict(params=[ps[1]])])

    tensor = torch.full((1,), 0.25, device=dev)
    opt, other = make(tensor), make(torch.full((1,), 0.5, device=dev))
    bad = other.state_dict()
    bad["param_groups"][1]["eps"] = -1.0
    with pytest.raises(ValueError, match="eps"):
        opt.load_state_dict(bad)
    assert float(tensor) == 0.25 and opt.param_groups[1]["eps"] == 1e-8
    good = other.state_dict()
    good["param_groups"][0]["lr"] = good["param_groups"][0]["lr"].cpu()
    opt.load_state_dict(good)
    assert opt.param_groups[0]["lr"] is tensor and float(tensor) == 0.5


@pytest.mark.parametrize("tokens", [0, 1])
def test_few_or_no_tokens(dev, tokens):
    g = torch.Generator().manual_seed(8)
    gate, up, down = ((torch.randn(s, generator=g) * 0.1).bfloat16().to(dev).requires_grad_(True)
                      for s in ((3, 32, 64), (3, 32, 64), (3, 64, 32)))
    x = torch.randn(tokens, 64, generator=g).bfloat16().to(dev).requires_grad_(True)
    r = route(torch.randn(tokens, 3, generator=g).to(dev), 2)
    y = experts_mlp(x, r, gate, up, down)
    grads = torch.autograd.grad(y, (x, gate, up, down), torch.ones_like(y))
    assert y.shape == x.shape and grads[0].shape == x.shape
    used = [False] * 3
    for e in r.index.flatten().tolist():
        used[e] = True
    for v in grads[1:]:
        assert [bool(v[e].any()) for e in range(3)] == used and torch.isfinite(v).all()


def test_gated_in_the_graph(dev):
    """One input with a gradient, none used, an expanded gradient, a graph kept, second derivatives
    refused, an input changed in between, another stream."""
    g = torch.Generator().manual_seed(9)
    a, b = (torch.randn(40, 24, generator=g).to(dev) for _ in range(2))
    ar, br = a.clone().requires_grad_(True), b.clone().requires_grad_(True)
    both = torch.autograd.grad(gated(ar, br).sum(), (ar, br))
    want = torch.autograd.grad(gated(ar, br), (ar, br), torch.ones_like(a))
    assert all(torch.equal(x, y) for x, y in zip(both, want))
    only, = torch.autograd.grad(gated(ar, b).sum(), ar)
    other, = torch.autograd.grad(gated(a, br).sum(), br)
    assert torch.equal(only, both[0]) and torch.equal(other, both[1])
    y = gated(ar, br)
    first = torch.autograd.grad(y.sum(), ar, retain_graph=True)[0]
    assert torch.equal(first, torch.autograd.grad(y.sum(), ar)[0])
    with pytest.raises(RuntimeError, match="second time|freed"):
        torch.autograd.grad(y.sum(), ar)
    d, = torch.autograd.grad(gated(ar, br).sum(), ar, create_graph=True)
    assert torch.equal(d, both[0])
    with pytest.raises(RuntimeError, match="twice"):
        d.sum().backward()
    y = gated(ar, br)
    with torch.no_grad():
        ar.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
    del y
    three = torch.randn(2, 3, 5, generator=g).half().to(dev).requires_grad_(True)
    z = gated(three, three * 2, "relu")
    assert z.shape == three.shape and torch.autograd.grad(z.sum(), three)[0].shape == three.shape
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ys = torch.autograd.grad(gated(ar, br), (ar, br), torch.ones_like(a))
    torch.cuda.current_stream().wait_stream(side)
    now = torch.autograd.grad(gated(ar, br), (ar, br), torch.ones_like(a))
    assert all(torch.equal(x, y) for x, y in zip(ys, now))
