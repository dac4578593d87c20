"""What the packed products promise at the edges of their arguments, on the MI355X."""

import ctypes

import numpy as np
import pytest
import torch

from packed_data import act64, bound, packed_tensor, stored
from test_gpu_packed import F, MIX, N, _experts, tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("slots", [1, 16, 17, 200])
@pytest.mark.parametrize("k", [128, 8320])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_slots_of_an_empty_batch_are_nan(own, slots, k, dt, dev):
    """Indices into a batch of no rows (whose data pointer is null) all lie outside it."""
    from hi2_amd.packed import PackedExperts, experts_linear

    print("empty batch", own, slots, k, dt, flush=True)
    plan = PackedExperts(_experts(3, 48, k, 5, own)[0], dev)
    assert (plan.transform is None) == own
    x = torch.empty(0, k, dtype=F[dt], device=dev)
    assert x.data_ptr() == 0
    offs = torch.tensor([0, slots // 2, slots // 2, slots], device=dev)
    rows = torch.arange(slots, device=dev) - 1
    out = experts_linear(x, plan, offs, rows)
    assert out.shape == (slots, 48) and torch.isnan(out).all()
    assert experts_linear(x, plan, torch.zeros(4, dtype=torch.int64, device=dev)).shape == (0, 48)


@pytest.mark.parametrize("own", [False, True])
def test_activations_of_an_empty_batch_are_nan(own, dev):
    from hi2_amd import _lib
    from hi2_amd.packed import PackedExperts

    plan = PackedExperts(_experts(2, 32, 192, 5, own)[0], dev)
    planes = torch.ones(40, plan.kp // 128, 2, 128, dtype=torch.float16, device=dev)
    scale = torch.ones(40, device=dev)
    desc = _lib.ActivationsDesc(planes.data_ptr(), scale.data_ptr(), 40, plan.kp, 2, 0)
    src, offs = torch.arange(40, device=dev), torch.tensor([0, 20, 40], device=dev)
    _lib.call("hi2x_packed_activations", dev, ctypes.byref(plan.desc), None, 2, 192, 0,
              _lib.ptr(src), _lib.ptr(offs), ctypes.byref(desc))
    assert torch.isnan(scale).all() and not planes.any()


def mlp64(x, r, gate, up, down, act="relu"):
    """The gated MLP in float64: gate, up and down each (tensors, decoded weights)."""
    index, w = N(r.index).astype(int), N(r.weights)
    out = np.zeros((len(x), down[1][0].shape[0]))
    for e in range(len(gate[0])):
        tok, c = np.nonzero(index == e)
        if not len(tok):
            continue
        a = act64(stored(N(x)[tok], gate[0][e]) @ gate[1][e].T, act)
        a = a * (stored(N(x)[tok], up[0][e]) @ up[1][e].T)
        np.add.at(out, tok, w[tok, c][:, None] * (stored(a, down[0][e]) @ down[1][e].T))
    return out


def huge_row(t, w, row):
    """Row `row` of INT4 in steps of about 5000, codes up to 11: its weights are finite, the
    ladder's last step is not."""
    k = t.shape[1]
    assert t.row_nbits[row] == 4
    t.row_consts[row] = torch.tensor([0.0, 0.0, 19.6]).half()
    blocks = slice(2 * int(t.param_off[row]), 2 * int(t.param_off[row + 1]))
    t.blk_params[blocks] = 255
    words = t.codes[int(t.code_off[row]):int(t.code_off[row + 1])]
    words &= int(np.uint32(0xBBBBBBBB).view(np.int32))
    codes = (words.numpy().view(np.uint32)[:, None] >> (4 * np.arange(8, dtype=np.uint32))) & 15
    step = np.float64(np.float16(np.float32(255 * np.float64(np.float16(19.6)))))
    w[row] = (codes.reshape(k) * step).astype(np.float16).astype(np.float64)
    assert np.isfinite(w[row]).all() and np.isinf(np.float16(15 * step))


def test_mlp_of_weights_below_an_infinite_step(dev):
    """A ladder whose last steps overflow fp16 and are not used: every weight and result is
    finite, in one call as in its parts."""
    from hi2_amd.moe import route
    from hi2_amd.packed import PackedExperts, moe_mlp

    t, e, k, h, i = 60, 3, 2, 128, 64
    gs, us, ds = _experts(e, i, h, 100), _experts(e, i, h, 200), _experts(e, h, i, 300)
    for ts, ws in (gs, us, ds):
        huge_row(ts[1], ws[1], int(torch.nonzero(ts[1].row_nbits == 4)[0]))
    plans = [PackedExperts(s[0], dev) for s in (gs, us, ds)]
    x = tokens(t, h, torch.bfloat16, 4, dev)
    r = route(torch.randn(t, e, generator=torch.Generator().manual_seed(3)).to(dev), k)
    got, want = N(moe_mlp(x, r, *plans, activation="relu")), mlp64(x, r, gs, us, ds)
    assert np.isfinite(got).all()
    # the roundings of the tokens, the hidden values and the result, as in the other MLP tests
    assert np.linalg.norm(got - want) < 2.0 ** -8 * np.linalg.norm(want)


def decoded(t):
    """The weights of a tensor by the format's definition, float64."""
    n, k = t.shape
    w = np.zeros((n, k))
    params, words = t.blk_params.numpy().reshape(-1, 2), t.codes.numpy().view(np.uint32)
    for r in range(n):
        nb, b = int(t.row_nbits[r]), int(t.row_block[r])
        c = t.row_consts[r].numpy().astype(np.float64)
        v = words[int(t.code_off[r]):int(t.code_off[r + 1])]
        codes = (v[:, None] >> (nb * np.arange(32 // nb, dtype=np.uint32))) & (2 ** nb - 1)
        u = params[int(t.param_off[r]):int(t.param_off[r + 1])]
        lo = (u[:, 0] * c[1] + c[0]).astype(np.float32).astype(np.float16).astype(np.float64)
        st = (u[:, 1] * c[2]).astype(np.float32).astype(np.float16).astype(np.float64)
        w[r] = (lo[:, None] + codes.reshape(-1, b) * st[:, None]).astype(np.float16).reshape(-1)
    return w


@pytest.mark.parametrize("channel", [0.0, 1e5, 1e7])
def test_mlp_of_experts_of_unlike_magnitude(channel, dev):
    """Experts with weights of 1e-3 and of 5e4 side by side, and tokens with a channel that
    dwarfs the others and meets zero weights: every token's result is as exact as another's."""
    from hi2_amd.moe import route
    from hi2_amd.packed import PackedExperts, moe_mlp

    t, e, h, i = 90, 3, 256, 128
    sides = []
    for n, k, seed in ((i, h, 100), (i, h, 200), (h, i, 300)):
        ts, _ = _experts(e, n, k, seed)
        for j, size in enumerate((1.0, 2.0 ** 18, 2.0 ** -6)):
            consts = ts[j].row_consts.double() * size
            ts[j].row_consts = consts.half()
            ts[j].had[:] = 0
            if k == h:  # columns 0 to 63 are zero: lo = u lo_scale + 0 and step 0 at u = 0
                consts[:, 1], consts[:, 0] = consts[:, 0] / 255, 0.0
                ts[j].row_consts = consts.half()
                for r in range(n):
                    b = 64 // int(ts[j].row_block[r])
                    a = 2 * int(ts[j].param_off[r])
                    ts[j].blk_params[a:a + 2 * b] = 0
        ws = [decoded(q) for q in ts]
        assert all(np.isfinite(v).all() for v in ws)
        sides.append((ts, ws))
    assert np.abs(sides[0][1][1]).max() > 2e4 and np.abs(sides[0][1][2]).max() < 4e-3
    x = tokens(t, h, torch.float32, 4, dev)
    x[:, 5] = channel
    x = x.bfloat16()
    index = torch.arange(t, device=dev) % e
    logits = torch.zeros(t, e, device=dev)
    logits[torch.arange(t, device=dev), index] = 4.0
    r = route(logits, 1)
    got = N(moe_mlp(x, r, *(PackedExperts(s[0], dev) for s in sides), activation="relu"))
    want = mlp64(x, r, *sides)
    off = np.linalg.norm(got - want, axis=1) / np.linalg.norm(want, axis=1)
    # a token's own roundings: its values, the hidden ones, the result, 2^-9 or less each as rms
    assert off.max() < 2.0 ** -7, off.reshape(-1, e).max(0)


@pytest.mark.parametrize("h,i", [(8064, 64), (64, 8064), (4096, 2064), (528, 1040)])
def test_mlp_of_wide_rows(h, i, dev):
    """The widest rows that the experts hand on in slot order, and widths beside the steps of
    the kernels that read them."""
    from hi2_amd.moe import route
    from hi2_amd.packed import PackedExperts, moe_mlp

    t, e, k = 24, 2, 1
    classes = [(2, 16), (4, 16)]
    sides = [_experts(e, n, m, s, classes=classes) for n, m, s in ((i, h, 1), (i, h, 2), (h, i, 3))]
    plans = [PackedExperts(s[0], dev) for s in sides]
    x = tokens(t, h, torch.bfloat16, 4, dev)
    r = route(torch.randn(t, e, generator=torch.Generator().manual_seed(3)).to(dev), k)
    got, want = N(moe_mlp(x, r, *plans, residual=x)), mlp64(x, r, *sides, act="silu") + N(x)
    assert np.isfinite(got).all()
    # each element: the result's rounding, and that of the tokens, the hidden values and what
    # is handed on, 2^-11 each, of sums whose terms cancel: as the row's norm, with margin
    off = np.abs(got - want) - 2.0 ** -8 * np.abs(want)
    assert off.max() < 2.0 ** -8 * np.abs(want).max()


@pytest.mark.parametrize("t,e,h,i", [(9000, 4, 512, 256), (1500, 16, 320, 192)])
def test_every_element_of_a_large_mlp(t, e, h, i, dev):
    """Large and middle tiles, element by element."""
    from hi2_amd.moe import route
    from hi2_amd.packed import PackedExperts, moe_mlp

    sides = _experts(e, i, h, 1), _experts(e, i, h, 2), _experts(e, h, i, 3)
    plans = [PackedExperts(s[0], dev) for s in sides]
    x = tokens(t, h, torch.bfloat16, 4, dev)
    r = route(torch.randn(t, e, generator=torch.Generator().manual_seed(3)).to(dev), 2)
    got, want = N(moe_mlp(x, r, *plans, residual=x)), mlp64(x, r, *sides, act="silu") + N(x)
    assert np.isfinite(got).all()
    # the result's rounding, and 2^-11 of each term of sums that cancel: as each row's largest
    off = np.abs(got - want) - 2.0 ** -8 * np.abs(want)
    assert (off <= 2.0 ** -7 * np.abs(want).max(1, keepdims=True)).all()


@pytest.mark.parametrize("rest", [5, 300])
def test_more_rows_than_a_grid_holds(rest, dev):
    """Rows beyond 65535 tiles of 64 go in parts, with their factor, bias and residual."""
    from hi2_amd.packed import PackedLinear, packed_linear

    n, k, part = 16, 64, 65535 * 64
    t = part + rest
    p, w = packed_tensor(n, k, [(4, 64)], 2)
    x = torch.zeros(t, k, dtype=torch.bfloat16, device=dev)
    mul = torch.zeros(t, n, dtype=torch.float16, device=dev)
    res = torch.zeros(t, n, device=dev)
    at = torch.tensor([0, 1, part - 1, part, part + 1, t - 1], device=dev)
    x[at] = tokens(len(at), k, torch.bfloat16, 3, dev)
    mul[at] = torch.randn(len(at), n, generator=torch.Generator().manual_seed(1)).half().to(dev)
    res[at] = torch.randn(len(at), n, generator=torch.Generator().manual_seed(2)).to(dev)
    got = packed_linear(x, PackedLinear(p, dev), mul=mul, residual=res)
    want = stored(N(x[at]), p) @ w.T * N(mul[at]) + N(res[at])
    xs = stored(N(x[at]), p)
    lim = bound(want, torch.bfloat16, torch.bfloat16, xs, w, np.abs(N(mul[at]))) + \
        2.0 ** -21 * np.abs(N(res[at]))
    assert (np.abs(N(got[at]) - want) <= lim).all()
    got[at] = 0
    assert not got.any()


def relative(got, want):
    return np.linalg.norm(N(got) - want) / np.linalg.norm(want)


@pytest.mark.parametrize("t", [1, 8, 14, 90, 300])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("out", ["f32", "f16"])
def test_results_wider_than_bf16_keep_the_activations_bits(t, dt, out, dev):
    """Rotated and smoothed activations of 16 bits take two planes where the result shows it."""
    from hi2_amd.packed import PackedLinear, activations, packed_linear

    n, k = 96, 256
    p, w = packed_tensor(n, k, MIX, 9, smooth=True)
    plan = PackedLinear(p, dev)
    x = tokens(t, k, F[dt], 3, dev)
    want = stored(N(x), p) @ w.T
    got = packed_linear(x, plan, out_dtype=F[out])
    # two planes leave 2^-22 of a value, sums in float32 about sqrt(k / 2) 2^-25 of the result;
    # an fp16 result is at most half an ulp from its value.  (One plane: about 2^-13.)
    lim = 2.0 ** -19 if out == "f32" else 2.0 ** -11.5
    assert relative(got, want) < lim
    if out == "f16":  # nothing beyond the result's own rounding
        own = np.linalg.norm(want.astype(np.float16) - want) / np.linalg.norm(want)
        assert relative(got, want) < own * (1 + 2.0 ** -7)
    a = activations(x, plan, out_dtype=F[out])
    assert relative(packed_linear(a, plan, out_dtype=F[out]), want) < lim


def test_activations_made_for_bf16_results_refuse_wider_ones(dev):
    from hi2_amd.packed import PackedLinear, activations, packed_linear

    p, _ = packed_tensor(32, 128, MIX, 9)
    plan = PackedLinear(p, dev)
    x = tokens(4, 128, torch.bfloat16, 3, dev)
    a = activations(x, plan)
    assert packed_linear(a, plan).dtype == torch.bfloat16
    with pytest.raises(ValueError, match="out_dtype"):
        packed_linear(a, plan, out_dtype=torch.float32)
    p.had[:] = 0  # bfloat16 values that nothing transforms are whole in one plane
    plain = PackedLinear(p, dev)
    got = packed_linear(activations(x, plain), plain, out_dtype=torch.float32)
    assert torch.equal(got, packed_linear(x, plain, out_dtype=torch.float32))


def test_gradient_of_the_mlps_weights_keeps_the_activations_bits(dev):
    """The routing's weights have a float32 gradient, from float32 parts: nothing in it is left
    to the 11 bits of one plane."""
    from dataclasses import replace

    from hi2_amd.moe import route
    from hi2_amd.packed import PackedExperts, moe_mlp

    t, e, k, h, i = 50, 4, 2, 128, 64
    sides = _experts(e, i, h, 100), _experts(e, i, h, 200), _experts(e, h, i, 300)
    plans = [PackedExperts(s[0], dev) for s in sides]
    x = tokens(t, h, torch.bfloat16, 4, dev)
    r = route(torch.randn(t, e, generator=torch.Generator().manual_seed(3)).to(dev), k)
    weights = r.weights.clone().requires_grad_(True)
    out = moe_mlp(x, replace(r, weights=weights), *plans, activation="relu")
    c = torch.randn(t, h, generator=torch.Generator().manual_seed(6)).bfloat16().to(dev)
    out.backward(c)
    want = np.zeros((t, k))
    for j in range(k):
        only = torch.zeros_like(r.weights)
        only[:, j] = 1.0
        want[:, j] = (N(c) * mlp64(x, replace(r, weights=only), *sides)).sum(1)
    assert relative(weights.grad, want) < 2.0 ** -17


@pytest.mark.parametrize("k,t", [(192, 8), (1040, 8), (8256, 8), (17024, 8), (17024, 40),
                                 (16384, 14), (4160, 100), (2064, 700)])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_every_column_counts_in_both_planes(k, t, dt, dev):
    """One value a row, in the first and last columns and at the chunks' edges: the product is
    its column times the value, bit for bit, with values that one plane cannot hold."""
    from hi2_amd.packed import PackedLinear, packed_linear

    n = 40
    p, w = packed_tensor(n, k, [(2, 16), (4, 16), (8, 16)], 11, had=0.0)
    edges = [k - 1, 0, k - 16, k - 2, 127, k // 128 * 128 - 1, k - 15, k - 8]
    cols = (edges + list(range(k - 1, -1, -max(1, k // t))))[:t]
    cols += [k - 1] * (t - len(cols))
    # 13 bits with the weight's 11: exact in float32
    value = 1.0 + 2.0 ** -12 if dt == "f32" else 1.0 + 2.0 ** -7
    x = torch.zeros(t, k, dtype=F[dt], device=dev)
    x[torch.arange(t, device=dev), torch.tensor(cols, device=dev)] = value
    got = packed_linear(x, PackedLinear(p, dev), out_dtype=torch.float32)
    assert np.array_equal(N(got), w.T[cols] * value)


def dual(t):
    from torch.autograd import forward_ad

    return forward_ad.make_dual(t, torch.ones_like(t))


def test_forward_mode_tangents_are_refused(dev):
    """None of these has a forward-mode derivative: a tangent is refused, not dropped."""
    from torch.autograd import forward_ad

    from hi2_amd.moe import route
    from hi2_amd.packed import (PackedExperts, PackedLinear, activations, combine,
                                experts_linear, moe_mlp, packed_linear)

    p, _ = packed_tensor(128, 128, MIX, 9)
    one, ex = PackedLinear(p, dev), PackedExperts([p, p], dev)
    x = torch.randn(6, 128, device=dev)
    logits = torch.randn(6, 2, device=dev)
    r = route(logits, 1)
    y = torch.randn(6, 8, device=dev)
    calls = [lambda d: route(d(logits), 1), lambda d: route(logits, 1, bias=d(logits[0])),
             lambda d: packed_linear(d(x), one), lambda d: packed_linear(x, one, mul=d(x)),
             lambda d: packed_linear(x, one, bias=d(x[0])), lambda d: activations(d(x), one),
             lambda d: experts_linear(x, ex, r.offs, r.rows, residual=d(x)),
             lambda d: combine(d(y), r.slots, r.weights),
             lambda d: combine(y, r.slots, d(r.weights)),
             lambda d: combine(y, r.slots, r.weights, residual=d(y)),
             lambda d: moe_mlp(d(x), r, ex, ex, ex), lambda d: moe_mlp(x, r, ex, ex, ex, residual=d(x))]
    for call in calls:
        with forward_ad.dual_level():
            call(lambda v: v)
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(dual)


def test_residuals_of_another_shape_are_refused(dev):
    from hi2_amd.moe import route
    from hi2_amd.packed import PackedExperts, combine, moe_mlp

    p, _ = packed_tensor(128, 128, MIX, 9)
    ex = PackedExperts([p, p], dev)
    x = torch.randn(2, 3, 128, device=dev)
    r = route(torch.randn(6, 2, device=dev), 1)
    y, res = torch.randn(6, 8, device=dev), torch.randn(6, 8, device=dev)
    want = combine(y, r.slots, r.weights, residual=res)
    for ok in (res.view(2, 3, 8), res.t().contiguous().t()):
        assert torch.equal(combine(y, r.slots, r.weights, residual=ok), want)
    for bad in (res.t(), res.reshape(-1), res[:5], res.view(6, 4, 2)):
        with pytest.raises(ValueError, match="residual"):
            combine(y, r.slots, r.weights, residual=bad)
    want = moe_mlp(x, r, ex, ex, ex, residual=x)
    assert torch.equal(moe_mlp(x, r, ex, ex, ex, residual=x.view(6, 128)), want)
    for bad in (x.view(6, 128).t(), x.reshape(-1), x[:1]):
        with pytest.raises(ValueError, match="residual"):
            moe_mlp(x, r, ex, ex, ex, residual=bad)


def repeated(kind, t, k, rows, g):
    """Slots that name rows several times: at random, one row only, in pairs far apart."""
    if kind == "random":
        return torch.randint(0, rows, (t, k), generator=g)
    if kind == "one":
        return torch.full((t, k), rows // 2)
    half = torch.arange(t * k // 2)
    return torch.cat([half, half, torch.zeros(t * k % 2, dtype=torch.int64)]).view(t, k) % rows


@pytest.mark.parametrize("kind", ["random", "one", "pairs"])
@pytest.mark.parametrize("t,k,rows,n", [(1, 3, 2, 5), (40, 2, 30, 260), (300, 8, 2400, 64),
                                        (70, 3, 1, 33), (129, 4, 90, 1)])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_rows_named_several_times_sum_their_gradients(kind, t, k, rows, n, dt, dev):
    from hi2_amd.packed import combine

    print("repeated", kind, t, k, rows, n, dt, flush=True)
    g = torch.Generator().manual_seed(t)
    y = torch.randn(rows, n, generator=g).to(F[dt]).to(dev).requires_grad_(True)
    slots = repeated(kind, t, k, rows, g).to(dev)
    w = torch.rand(t, k, generator=g).to(dev).requires_grad_(True)
    c = torch.randn(t, n, generator=g).to(F[dt]).to(dev)
    grads = [torch.autograd.grad(combine(y, slots, w), (y, w), c) for _ in range(2)]
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    s, gc, wd = N(slots).astype(int), N(c), N(w)
    want, mass = np.zeros((rows, n)), np.zeros((rows, n))
    for j in range(k):
        np.add.at(want, s[:, j], wd[:, j, None] * gc)
        np.add.at(mass, s[:, j], np.abs(wd[:, j, None] * gc))
    most = np.bincount(s.reshape(-1), minlength=rows)[:, None]  # float32 products and sums
    unit = {"bf16": 2.0 ** -8, "f32": 2.0 ** -23}[dt]
    assert (np.abs(N(grads[0][0]) - want) <= unit * np.abs(want) + 2 * most * 2.0 ** -24 * mass).all()
    terms = gc[:, None] * N(y)[s]
    lim = (n + 8) * 2.0 ** -24 * np.abs(terms).sum(-1)
    assert (np.abs(N(grads[0][1]) - terms.sum(-1)) <= lim).all()


def test_scanned_counts_of_64_token_workgroups(dev):
    """Above 1024 workgroups of 64 tokens the counts are scanned by a launch of their own."""
    from hi2_amd.moe import route, route_order

    x = torch.randn(70_000, 96, generator=torch.Generator().manual_seed(1)).to(dev)
    r = route(x, 8)
    assert torch.equal(r.index, x.sort(dim=-1, descending=True, stable=True).indices[:, :8])
    rows, offs = route_order(r.index, 96)
    assert torch.equal(r.rows, rows) and torch.equal(r.offs, offs)
    assert torch.equal(r.rows[r.slots], torch.arange(70_000, device=dev)[:, None].expand(-1, 8))


def test_threads_route_over_different_groups(dev):
    """Two threads whose routers want different amounts of LDS of one kernel."""
    from concurrent.futures import ThreadPoolExecutor

    from hi2_amd.moe import route

    def runs(e, groups):
        with torch.cuda.device(dev), torch.cuda.stream(torch.cuda.Stream()):
            x = torch.randn(64, e, generator=torch.Generator().manual_seed(e)).to(dev)
            first = route(x, 4, groups=groups, top_groups=groups // 2)
            same = [torch.equal(route(x, 4, groups=groups, top_groups=groups // 2).slots,
                                first.slots) for _ in range(100)]
            torch.cuda.current_stream().synchronize()
            return all(same)

    with ThreadPoolExecutor(2) as pool:
        assert all(pool.map(runs, (256, 200), (64, 50)))
