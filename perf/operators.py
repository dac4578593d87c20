"""The measured workloads of running an encoded model: the products by packed weights, the
router and the experts' products, what a program that serves or scores the quantised
checkpoint has this package do.

=========  ===============================================================================
kind       one pass
=========  ===============================================================================
linear     ``packed_linear``: ``act(T(x) Wq^T + bias) * mul + residual`` with ``Wq`` the
           packed INT2/INT4/INT8 rows of one tensor and ``T`` its smoothing and rotation
route      ``moe.route``: scores, expert groups, top-k, weights and the expert order of
           the routed slots; with ``grad`` also the gradient of the weights to the logits
experts    ``moe.route`` and ``packed.moe_mlp``: a gated MLP of packed experts over the
           routed tokens and its weighted sum
=========  ===============================================================================

Tokens are unit normal with 1 % of the channels twenty times larger, the ladders' constants
give weights of about N(0, 0.03^2), and rows are split at random between the classes.
"""

import math
from types import SimpleNamespace

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
GROUP = 16


def _linear(n, k, t, dtype="bf16", int2=0.3, int8=0.0, b2=32, b4=64, b8=64, had=1.0,
            smooth=False, bias=False, act="none", mul=False, residual=False, **more):
    return dict(kind="linear", n=n, k=k, t=t, dtype=dtype, int2=int2, int8=int8, b2=b2, b4=b4,
                b8=b8, had=had, smooth=smooth, bias=bias, act=act, mul=mul, residual=residual,
                **more)


def _route(t, e, k, scoring="softmax", bias=False, groups=1, top_groups=1, dtype="f32",
           renorm=True, grad=False, **more):
    return dict(kind="route", t=t, e=e, k=k, scoring=scoring, bias=bias, groups=groups,
                top_groups=top_groups, dtype=dtype, renorm=renorm, grad=grad, **more)


def _experts(t, e, k, hidden, inter, dtype="bf16", int2=0.3, int8=0.0, residual=True, **more):
    return dict(kind="experts", t=t, e=e, k=k, hidden=hidden, inter=inter, dtype=dtype,
                int2=int2, int8=int8, residual=residual, **more)


def listed():
    return [
        # k_proj / v_proj of an 8B block, one token: the smallest product of a decode step
        _linear(1024, 4096, 1, bias=True, name="linear_1024x4096_t1"),
        # down_proj of an 8B block, one token, added to the residual stream
        _linear(4096, 14336, 1, residual=True, name="linear_4096x14336_t1"),
        # gate_proj of a 70B layer over a small batch of sequences, one token each
        _linear(28672, 8192, 13, int2=0.25, int8=0.03, act="silu",
                name="linear_28672x8192_t13"),
        # a small Linear over a calibration sample, half precision, smoothing vector
        _linear(2048, 2048, 512, dtype="f16", int2=0.0, smooth=True, bias=True, act="gelu",
                name="linear_2048x2048_t512_f16"),
        # down_proj over a ragged prompt, some groups unrotated
        _linear(4096, 14336, 1000, had=0.9, residual=True, name="linear_4096x14336_t1000"),
        # up_proj of an 8B block over a long prompt, times the activated gate
        _linear(14336, 4096, 4096, mul=True, name="linear_14336x4096_t4096"),
        # one token of a 64-expert layer: latency
        _route(1, 64, 8, dtype="bf16", name="route_64_t1"),
        # a 64-expert layer's calibration batch
        _route(16384, 64, 8, name="route_64_t16384"),
        # many experts in groups, a balance bias, sigmoid scores
        _route(4096, 256, 8, scoring="sigmoid", bias=True, groups=8, top_groups=4,
               name="route_256_t4096_groups"),
        # the router's training direction
        _route(8192, 64, 8, dtype="bf16", grad=True, name="route_64_t8192_grad"),
        # an MoE layer, one token: eight experts' weights
        _experts(1, 64, 8, 2048, 1024, name="experts_64_t1"),
        # the same layer over a calibration batch
        _experts(16384, 64, 8, 2048, 1024, name="experts_64_t16384"),
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _mult(x, m):
    return max(m, int(x) // m * m)


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "route", "route", "experts", "experts"])
    if kind == "linear":
        b2, b4, b8 = rng.choice([16, 32, 64]), rng.choice([16, 32, 64]), rng.choice([32, 64])
        k = _mult(_log(rng, 256, 14336), 64)
        n = int(_log(rng, 64, min(28672, 14336 * 8192 / k)))
        t = int(_log(rng, 1, min(4096, 14336.0 * 4096 * 4096 / (n * k))))
        return _linear(n, k, t, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                       int2=round(rng.uniform(0.0, 0.6), 2), int8=rng.choice([0.0, 0.03, 0.2]),
                       b2=b2, b4=b4, b8=b8, had=rng.choice([1.0, 1.0, 0.9, 0.0]),
                       smooth=rng.random() < 0.3, bias=rng.random() < 0.3,
                       act=rng.choice(["none", "none", "silu", "gelu", "gelu_tanh", "relu"]),
                       mul=rng.random() < 0.3, residual=rng.random() < 0.4)
    if kind == "route":
        groups = rng.choice([1, 1, 4, 8])
        e = groups * rng.randint(4, 256 // groups)
        top_groups = rng.randint(1, groups)
        grad = rng.random() < 0.4
        # (one renormalised expert has the weight 1: no gradient)
        k = rng.randint(2 if grad else 1, min(16, e // groups * top_groups))
        scoring = rng.choice(["softmax", "sigmoid"])
        return _route(int(_log(rng, 1, 16384)), e, k, scoring=scoring,
                      bias=rng.random() < 0.5, groups=groups, top_groups=top_groups,
                      dtype=rng.choice(["f32", "bf16", "f16"]), renorm=rng.random() < 0.7, grad=grad)
    e = rng.choice([8, 16, 60, 64, 128])
    hidden, inter = _mult(_log(rng, 256, 2048), 64), _mult(_log(rng, 128, 1024), 64)
    return _experts(int(_log(rng, 1, 8192)), e, rng.randint(1, 8), hidden, inter,
                    dtype=rng.choice(["bf16", "bf16", "f16"]), int2=round(rng.uniform(0, 0.6), 2),
                    int8=rng.choice([0.0, 0.1]), residual=rng.random() < 0.7)


# ---- inputs -------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(1000003 * (seed + 1))


def _tokens(t, k, g, dtype):
    x = torch.randn(t, k, generator=g, device=DEV)
    x[:, torch.randperm(k, generator=g, device=DEV)[: -(-k // 100)]] *= 20.0
    return x.to(dtype)


def _uniform(shape, lo, hi, g):
    return torch.rand(shape, generator=g, device=DEV) * (hi - lo) + lo


def _packed(e, n, k, classes, g):
    """The flat buffers of ``e`` tensors [n, k] one after the other: ``classes`` is a list
    of (share of the rows, nbits, block), a random choice of rows each in every tensor."""
    nbits = torch.empty(e, n, dtype=torch.int64, device=DEV)
    block = torch.empty(e, n, dtype=torch.int64, device=DEV)
    order = torch.rand(e, n, generator=g, device=DEV).argsort(dim=1)
    at = 0
    for i, (share, nb, b) in enumerate(classes):
        to = n if i == len(classes) - 1 else min(n, at + int(round(share * n)))
        nbits.scatter_(1, order[:, at:to], nb)
        block.scatter_(1, order[:, at:to], b)
        at = to
    nbits, block = nbits.reshape(-1), block.reshape(-1)
    zero = torch.zeros(1, dtype=torch.int64, device=DEV)
    code_off = torch.cat([zero, (nbits * k // 32).cumsum(0)])
    param_off = torch.cat([zero, (k // block).cumsum(0)])
    codes = torch.randint(-2 ** 31, 2 ** 31, (int(code_off[-1]),), generator=g, device=DEV,
                          dtype=torch.int32)
    params = torch.randint(64, 256, (2 * int(param_off[-1]),), generator=g, device=DEV,
                           dtype=torch.uint8)
    # lo = lo_min + u lo_scale around -0.05, step so that the ladder spans about 0.1
    lo_min = _uniform((e * n,), -0.07, -0.06, g)
    lo_scale = _uniform((e * n,), 0.01, 0.03, g) / 255
    step = _uniform((e * n,), 0.12, 0.16, g) / 255 / (2.0 ** nbits - 1)
    consts = torch.stack([lo_min, lo_scale, step], 1).half()
    return SimpleNamespace(codes=codes, code_off=code_off, params=params, param_off=param_off,
                           consts=consts, nbits=nbits, block=block, e=e, n=n, k=k)


def _flags(share, k, g):
    return (torch.rand(k // GROUP, generator=g, device=DEV) < share).to(torch.uint8)


def _tensors(p, had, smooth):
    """The tensors of ``p`` as the package's ``HI2Tensor``s."""
    from hi2_amd.format import HI2Tensor

    co, po = p.code_off.cpu(), p.param_off.cpu()
    out = []
    for i in range(p.e):
        a, b = i * p.n, (i + 1) * p.n
        out.append(HI2Tensor(
            codes=p.codes[int(co[a]):int(co[b])], code_off=(co[a:b + 1] - co[a]).int(),
            blk_params=p.params[2 * int(po[a]):2 * int(po[b])],
            param_off=(po[a:b + 1] - po[a]).int(), row_consts=p.consts[a:b],
            row_nbits=p.nbits[a:b].to(torch.uint8).cpu(),
            row_block=p.block[a:b].to(torch.uint8).cpu(), had=had, shape=(p.n, p.k),
            col_scale=smooth))
    return out


def _logits(case, g):
    t, e = case["t"], case["e"]
    popular = -0.4 * torch.log(torch.randperm(e, generator=g, device=DEV) + 1.0)
    return (1.5 * torch.randn(t, e, generator=g, device=DEV) + popular).to(
        DTYPES[case["dtype"]])


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    s = SimpleNamespace(kind=kind, case=case)
    if kind == "route":
        s.logits = _logits(case, g)
        s.bias = _uniform((case["e"],), -0.1, 0.1, g) if case["bias"] else None
        s.grad = torch.randn(case["t"], case["k"], generator=g, device=DEV)
        s.want = s.logits.clone().requires_grad_(True)
        return s
    dtype = DTYPES[case["dtype"]]
    if kind == "linear":
        n, k, t = case["n"], case["k"], case["t"]
        s.w = _packed(1, n, k, [(case["int2"], 2, case["b2"]), (case["int8"], 8, case["b8"]),
                                (1.0, 4, case["b4"])], g)
        s.had = _flags(case["had"], k, g)
        s.smooth = _uniform((k,), 0.5, 2.0, g).half() if case["smooth"] else None
        s.x = _tokens(t, k, g, dtype)
        s.bias = (0.1 * torch.randn(n, generator=g, device=DEV)).to(dtype) \
            if case["bias"] else None
        s.mul = torch.randn(t, n, generator=g, device=DEV).to(dtype) if case["mul"] else None
        s.residual = torch.randn(t, n, generator=g, device=DEV).to(dtype) \
            if case["residual"] else None
        if own:
            from hi2_amd.packed import PackedLinear

            s.plan = PackedLinear(_tensors(s.w, s.had, s.smooth)[0], DEV)
        return s
    e, h, i = case["e"], case["hidden"], case["inter"]
    classes = [(case["int2"], 2, 32), (case["int8"], 8, 64), (1.0, 4, 64)]
    s.gate, s.up = _packed(e, i, h, classes, g), _packed(e, i, h, classes, g)
    s.down = _packed(e, h, i, classes, g)
    s.had_in, s.had_mid = _flags(1.0, h, g), _flags(1.0, i, g)
    s.x = _tokens(case["t"], h, g, dtype)
    s.logits = _logits(case, g)
    s.residual = torch.randn(case["t"], h, generator=g, device=DEV).to(dtype) \
        if case["residual"] else None
    if own:
        from hi2_amd.packed import PackedExperts

        s.plans = [PackedExperts(_tensors(p, f, None), DEV) for p, f in
                   ((s.gate, s.had_in), (s.up, s.had_in), (s.down, s.had_mid))]
    return s


# ---- the plain forms ----------------------------------------------------------------------
def _h16(dtype):
    h = torch.ones(1, 1, dtype=dtype, device=DEV)
    for _ in range(4):
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    return h / 4.0


def _stored(x, had, smooth):
    """The activations in the weights' basis: ``x / s``, flagged groups rotated (32 bits)."""
    x = x.float()
    if smooth is not None:
        x = x / smooth.float()
    groups = x.reshape(*x.shape[:-1], -1, GROUP)
    return torch.where(had.bool()[:, None], groups @ _h16(torch.float32), groups).reshape(x.shape)


def _class_rows(p, rows, nb, b):
    """The decoded weights of ``rows``, all of one class, float32."""
    k = p.k
    words = p.codes[p.code_off[rows][:, None] + torch.arange(k * nb // 32, device=DEV)]
    shifts = torch.arange(0, 32, nb, device=DEV, dtype=torch.int32)
    code = ((words[:, :, None] >> shifts) & (2 ** nb - 1)).reshape(len(rows), k // b, b).float()
    byte = p.params.reshape(-1, 2)[p.param_off[rows][:, None] + torch.arange(k // b, device=DEV)]
    c = p.consts[rows].float()
    lo = (byte[:, :, 0].float() * c[:, 1:2] + c[:, 0:1]).half().float()
    step = (byte[:, :, 1].float() * c[:, 2:3]).half().float()
    return (code * step[:, :, None] + lo[:, :, None]).half().float().reshape(len(rows), k)


def _weights(p, tensors=None):
    """The decoded weights [e, n, k] of the tensors asked for, float32."""
    t = torch.arange(p.e, device=DEV) if tensors is None else tensors
    rows = (t[:, None] * p.n + torch.arange(p.n, device=DEV)).reshape(-1)
    out = torch.empty(len(rows), p.k, device=DEV)
    kinds = p.nbits[rows] * 256 + p.block[rows]
    for kind in torch.unique(kinds).tolist():
        at = (kinds == kind).nonzero()[:, 0]
        out[at] = _class_rows(p, rows[at], kind // 256, kind % 256)
    return out.reshape(len(t), p.n, p.k)


def _act(y, act):
    if act == "relu":
        return torch.where(y > 0, y, torch.zeros_like(y))
    if act == "silu":
        return y / (1 + torch.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    return y


def _plain_linear(s):
    y = _stored(s.x, s.had, s.smooth) @ _weights(s.w)[0].T
    if s.bias is not None:
        y = y + s.bias.float()
    y = _act(y, s.case["act"])
    if s.mul is not None:
        y = y * s.mul.float()
    if s.residual is not None:
        y = y + s.residual.float()
    return y.to(s.x.dtype)


def _scores(logits, scoring):
    """The scores of float32 logits; the softmax's sum is taken in 64 bits, so that the
    order of its terms does not show in the experts chosen."""
    if scoring == "sigmoid":
        return 1 / (1 + torch.exp(-logits))
    e = torch.exp(logits - logits.amax(-1, keepdim=True))
    return e / e.double().sum(-1, keepdim=True).to(e.dtype)


def _choose(logits, scores, bias, k, groups, top_groups):
    """The experts of each token, ties to the lowest index: by the logits themselves
    (the scores' order, without their rounding), by score + bias where there is one."""
    t, e = logits.shape
    choice = logits if bias is None else scores + bias
    if groups > 1 and top_groups < groups:
        by = choice.reshape(t, groups, e // groups)
        # a group is as good as its best expert, with a bias as its best two together
        best = by.sort(dim=-1, descending=True).values
        good = best[..., 0] if bias is None or e == groups else best[..., 0] + best[..., 1]
        kept = good.sort(dim=-1, descending=True, stable=True).indices[:, :top_groups]
        keep = torch.zeros(t, groups, dtype=torch.bool, device=logits.device)
        keep.scatter_(1, kept, True)
        choice = torch.where(keep[..., None], by, -math.inf).reshape(t, e)
    return choice.sort(dim=-1, descending=True, stable=True).indices[:, :k]


def _weigh(scores, index, renorm):
    w = scores.gather(1, index)
    return w / w.sum(-1, keepdim=True) if renorm else w


def _order(index, e):
    """(rows, offs, slots): the token of each routed slot in expert order (stable), the
    experts' ranges, and each (token, choice)'s slot."""
    flat = index.reshape(-1)
    order = flat.sort(dim=0, stable=True).indices
    offs = (flat[:, None] == torch.arange(e, device=DEV)).sum(0).cumsum(0) \
        if flat.numel() * e <= 1 << 22 else torch.bincount(flat, minlength=e).cumsum(0)
    slots = torch.empty_like(order)
    slots[order] = torch.arange(len(flat), device=DEV)
    return (order // index.shape[1], torch.cat([offs.new_zeros(1), offs]),
            slots.reshape(index.shape))


def _plain_route(s):
    c = s.case
    logits = s.logits.float()
    scores = _scores(logits, c["scoring"])
    index = _choose(logits, scores, s.bias, c["k"], c["groups"], c["top_groups"])
    w = _weigh(scores, index, c["renorm"])
    rows, offs, slots = _order(index, c["e"])
    out = dict(index=index, weights=w, rows=rows, offs=offs, slots=slots)
    if c["grad"]:
        # the gradient at the scores of the chosen experts, then through the scores
        g = s.grad
        if c["renorm"]:
            total = scores.gather(1, index).sum(-1, keepdim=True)
            g = (g - (g * w).sum(-1, keepdim=True)) / total
        at = torch.zeros_like(scores).scatter_(1, index, g)
        if c["scoring"] == "sigmoid":
            d = at * scores * (1 - scores)
        else:
            d = scores * (at - (at * scores).sum(-1, keepdim=True))
        out["dlogits"] = d.to(s.logits.dtype)
    return out


def _plain_experts(s):
    c = s.case
    logits = s.logits.float()
    scores = _scores(logits, "softmax")
    index = _choose(logits, scores, None, c["k"], 1, 1)
    w = _weigh(scores, index, True)
    rows, offs, slots = _order(index, c["e"])
    counts = offs[1:] - offs[:-1]
    # the experts that have tokens, each one's slots padded to the longest
    live = counts.nonzero()[:, 0]
    pad = torch.arange(int(counts.max()), device=DEV)
    at = offs[live][:, None] + pad
    ok = pad < counts[live][:, None]
    at = torch.where(ok, at, torch.zeros_like(at))
    x = _stored(s.x, s.had_in, None)[rows[at]]
    gate = torch.bmm(x, _weights(s.gate, live).transpose(1, 2).contiguous())
    up = torch.bmm(x, _weights(s.up, live).transpose(1, 2).contiguous())
    h = _stored(_act(gate, "silu") * up, s.had_mid, None)
    y = torch.bmm(h, _weights(s.down, live).transpose(1, 2).contiguous())
    flat = torch.empty(len(rows), c["hidden"], device=DEV)
    flat[at[ok]] = y[ok]
    out = (flat[slots] * w[:, :, None]).sum(1)
    if s.residual is not None:
        out = out + s.residual.float()
    return out.to(s.x.dtype)


# ---- one pass -----------------------------------------------------------------------------
def run(s):
    if not own:
        return {"linear": _plain_linear, "route": _plain_route,
                "experts": _plain_experts}[s.kind](s)
    c = s.case
    if s.kind == "linear":
        from hi2_amd.packed import packed_linear

        return packed_linear(s.x, s.plan, bias=s.bias, activation=c["act"], mul=s.mul,
                             residual=s.residual)
    from hi2_amd.moe import route

    if s.kind == "route":
        r = route(s.want if c["grad"] else s.logits, c["k"], scoring=c["scoring"], bias=s.bias,
                  groups=c["groups"], top_groups=c["top_groups"], renormalise=c["renorm"])
        out = dict(index=r.index, weights=r.weights, rows=r.rows, offs=r.offs, slots=r.slots)
        if c["grad"]:
            out["dlogits"], = torch.autograd.grad(r.weights, s.want, s.grad)
        return out
    from hi2_amd.packed import moe_mlp

    r = route(s.logits, c["k"])
    return moe_mlp(s.x, r, *s.plans, residual=s.residual)


# ---- the definition in 64 bits --------------------------------------------------------------
def _exact_weights(p, tensor):
    """Tensor ``tensor`` of ``p``, [n, k] float64, each code taken from its bit position."""
    rows = torch.arange(tensor * p.n, (tensor + 1) * p.n, device=DEV)
    col = torch.arange(p.k, device=DEV)
    out = []
    for r in rows.split(max(1, (1 << 24) // p.k)):
        nb, b = p.nbits[r][:, None], p.block[r][:, None]
        bit = col * nb
        word = p.codes[p.code_off[r][:, None] + bit // 32].long()
        code = (word >> (bit % 32)) & (2 ** nb - 1)
        blk = 2 * (p.param_off[r][:, None] + col // b)
        c = p.consts[r].double()
        lo = (p.params[blk].double() * c[:, 1:2] + c[:, 0:1]).float().half().double()
        step = (p.params[blk + 1].double() * c[:, 2:3]).float().half().double()
        out.append((lo + code * step).half().double())
    return torch.cat(out)


def _exact_stored(x, had, smooth):
    x = x.double()
    if smooth is not None:
        x = x / smooth.double()
    v = x.reshape(len(x), -1, GROUP)
    h = _h16(torch.float64)
    turned = sum(v[..., i:i + 1] * h[i] for i in range(GROUP))
    return torch.where(had[:, None] != 0, turned, v).reshape(x.shape)


def _exact_act(y, act):
    if act == "relu":
        return y.clamp_min(0)
    if act == "silu":
        return y * torch.special.expit(y)
    if act == "gelu":
        return y * 0.5 * torch.special.erfc(-y / math.sqrt(2))
    if act == "gelu_tanh":
        return y * torch.special.expit(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
    return y


def _exact_route(case, logits, bias):
    v = logits.double()
    if case.get("scoring", "softmax") == "sigmoid":
        p = torch.special.expit(v)
    else:
        p = torch.exp(v - torch.logsumexp(v, -1, keepdim=True))
    t, e = v.shape
    key = v if bias is None else p + bias.double()
    groups, top_groups = case.get("groups", 1), case.get("top_groups", 1)
    if top_groups < groups:
        by = key.reshape(t, groups, -1)
        good = by.topk(1 if bias is None or e == groups else 2, -1).values.sum(-1)
        # how many groups go before each one
        before = (good[:, None, :] > good[:, :, None]) | (
            (good[:, None, :] == good[:, :, None]) & torch.tril(torch.ones(
                groups, groups, dtype=torch.bool, device=DEV), -1))
        key = by.masked_fill((before.sum(-1) >= top_groups)[..., None], -math.inf).reshape(t, e)
    index = torch.argsort(-key, dim=-1, stable=True)[:, :case["k"]]
    w = torch.take_along_dim(p, index, 1)
    total = w.sum(-1, keepdim=True)
    return p, index, (w / total if case.get("renorm", True) else w), total


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "linear":
        y = _exact_stored(s.x, s.had, s.smooth) @ _exact_weights(s.w, 0).T
        if s.bias is not None:
            y = y + s.bias.double()
        y = _exact_act(y, case["act"])
        if s.mul is not None:
            y = y * s.mul.double()
        return y if s.residual is None else y + s.residual.double()
    if case["kind"] == "route":
        p, index, w, total = _exact_route(case, s.logits, s.bias)
        out = dict(index=None, weights=w, rows=None, offs=None, slots=None)
        if case["grad"]:
            leaf = s.logits.double().requires_grad_(True)
            q = torch.sigmoid(leaf) if case["scoring"] == "sigmoid" else torch.softmax(leaf, -1)
            v = torch.take_along_dim(q, index, 1)
            v = v / v.sum(-1, keepdim=True) if case["renorm"] else v
            out["dlogits"], = torch.autograd.grad((v * s.grad.double()).sum(), leaf)
        return out
    _, index, w, _ = _exact_route(case, s.logits, None)
    x = _exact_stored(s.x, s.had_in, None)
    out = torch.zeros(case["t"], case["hidden"], dtype=torch.float64, device=DEV)
    if s.residual is not None:
        out += s.residual.double()
    for e in range(case["e"]):
        tok, j = (index == e).nonzero(as_tuple=True)
        if len(tok) == 0:
            continue
        a = x[tok]
        gate, up = a @ _exact_weights(s.gate, e).T, a @ _exact_weights(s.up, e).T
        mid = _exact_stored(_exact_act(gate, "silu") * up, s.had_mid, None)
        out.index_add_(0, tok, w[tok, j][:, None] * (mid @ _exact_weights(s.down, e).T))
    return out


# ---- what a pass cannot do without ----------------------------------------------------------
def _packed_bytes(n, k, case):
    b2, b4, b8 = case.get("b2", 32), case.get("b4", 64), case.get("b8", 64)
    n2, n8 = int(round(case["int2"] * n)), int(round(case["int8"] * n))
    n4 = n - n2 - n8
    return k * (n2 * (2 / 8 + 2 / b2) + n4 * (4 / 8 + 2 / b4) + n8 * (1 + 2 / b8)) + 6 * n


def work(case):
    t = case["t"]
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if case["kind"] == "linear":
        n, k = case["n"], case["k"]
        return {"bytes": _packed_bytes(n, k, case) + size * (
            t * k + t * n * (1 + case["mul"] + case["residual"]) + n * case["bias"]),
            "flops": 2.0 * t * n * k}
    e, k = case["e"], case["k"]
    if case["kind"] == "route":
        # index, rows and slots of 8 bytes, weights of 4; the gradient in and out
        return {"bytes": t * e * size * (2 if case["grad"] else 1) + t * k * (
            28 + 4 * case["grad"]) + 8 * (e + 1), "flops": 8.0 * t * e}
    h, i, slots = case["hidden"], case["inter"], t * case["k"]
    live = e * (1 - (1 - k / e) ** t)
    return {"bytes": live * (2 * _packed_bytes(i, h, case) + _packed_bytes(h, i, case)) + size * (
        t * h * (2 + case["residual"])) + t * e * size, "flops": 6.0 * slots * h * i}
