"""The measured workloads of training a model's weights: the products of an MoE layer's experts
with their gradients, the gated activation between them, and the AdamW step over all of a
layer's tensors.

=========  ===============================================================================
kind       one pass
=========  ===============================================================================
grouped    ``experts.grouped_linear``: every expert's product ``x[rows] w[e]^T`` over the
           routed slots; with ``grad`` also the gradients of the tokens and of the weights
gated      ``experts.gated``: ``act(gate) * up``; with ``grad`` also both gradients
adamw      ``optim.AdamW.step`` over all tensors at once, moments in 32 or in 8 bits, and
           the moments as the values they stand for
=========  ===============================================================================

Tokens are unit normal with 1 % of the channels twenty times larger, weights N(0, 0.03^2), and
experts are chosen by logits that prefer some of them.  Parameters, gradients and moments lie one
tensor after the other, each from a multiple of 256 elements on.
"""

import math
from types import SimpleNamespace

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BLOCK = 256
BETA1, BETA2, EPS = 0.9, 0.999, 1e-8
# (learning rate, weight decay) of the weights and of what belongs to them (ladders, norms)
GROUPS = ((1e-4, 0.01), (1e-3, 0.0))


def _grouped(t, e, k, n, width, dtype="bf16", gather=True, grad=False, **more):
    return dict(kind="grouped", t=t, e=e, k=k, n=n, width=width, dtype=dtype, gather=gather,
                grad=grad, **more)


def _gated(rows, width, dtype="bf16", act="silu", halves=False, grad=False, **more):
    return dict(kind="gated", rows=rows, width=width, dtype=dtype, act=act, halves=halves,
                grad=grad, **more)


def _adamw(tensors, rows, width, small=0, dtype="f32", bits=32, master=False, t=100, **more):
    """``tensors`` weights of ``rows`` x ``width`` and beside each ``small`` vectors of its
    ladder blocks (one value to 64 weights)."""
    return dict(kind="adamw", tensors=tensors, rows=rows, width=width, small=small, dtype=dtype,
                bits=bits, master=master, t=t, **more)


def listed():
    return [
        # the gate projection of a 64-expert layer for one token: eight experts' weights, latency
        _grouped(1, 64, 8, 1024, 2048, name="grouped_64_t1"),
        # its down projection over a small decode batch, rows already in slot order
        _grouped(37, 64, 8, 2048, 1024, gather=False, name="grouped_64_t37_down"),
        # a training step of a layer of eight wide experts over a ragged batch
        _grouped(1000, 8, 2, 14336, 4096, dtype="f16", grad=True, name="grouped_8_t1000_f16_grad"),
        # odd sizes in full precision, as a small distillation run has them
        _grouped(777, 60, 4, 520, 1001, dtype="f32", grad=True, name="grouped_60_t777_f32_grad"),
        # the 64-expert layer over a training batch
        _grouped(16384, 64, 8, 1024, 2048, grad=True, name="grouped_64_t16384_grad"),
        # between the products of one token's experts: latency
        _gated(8, 1024, name="gated_8x1024"),
        # between wide experts, gate and up the halves of one product's rows
        _gated(2000, 14336, dtype="f16", act="gelu_tanh", halves=True, grad=True,
               name="gated_2000x14336_f16_grad"),
        # the 64-expert layer's training batch
        _gated(131072, 1024, grad=True, name="gated_131072x1024_grad"),
        # one distilled Linear: its latent and its ladders' bytes
        _adamw(1, 1024, 4096, small=2, name="adamw_1024x4096"),
        # a block's wide Linears in 8-bit states, with their ladders
        _adamw(3, 14336, 4096, small=2, bits=8, name="adamw_3x14336x4096_8bit"),
        # every expert of a layer in bfloat16 with 32-bit masters
        _adamw(192, 1024, 2048, dtype="bf16", master=True, name="adamw_192x1024x2048_bf16"),
        # many small tensors of odd sizes in half precision and 8-bit states
        _adamw(100, 37, 129, small=3, dtype="f16", bits=8, t=0, name="adamw_100x37x129_f16_8bit"),
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def draw(rng):
    kind = rng.choice(["grouped", "grouped", "grouped", "gated", "adamw", "adamw"])
    if kind == "grouped":
        e = rng.choice([4, 8, 16, 60, 64, 128])
        k = rng.randint(1, min(e, 8))
        step = rng.choice([1, 8, 64])
        n = max(step, int(_log(rng, 64, 14336)) // step * step)
        most = min(14336.0, 8 * 14336 * 4096.0 / (e * n))
        width = max(step, int(_log(rng, min(64, most / 2), most)) // step * step)
        dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f16", "f32"])
        slots = 16384 * 8 * 1024 * 2048.0 / (n * width * (8 if dtype == "f32" else 1))
        t = int(_log(rng, 1, max(2.0, min(16384.0, slots / k))))
        # (what the padded plain form holds stays within some gigabytes)
        t = max(1, min(t, int(2e9 / (k * max(n, width)))))
        return _grouped(t, e, k, n, width, dtype=dtype, gather=rng.random() < 0.6,
                        grad=rng.random() < 0.5)
    if kind == "gated":
        step = rng.choice([1, 8, 64])
        width = max(step, int(_log(rng, 64, 14336)) // step * step)
        rows = int(_log(rng, 1, min(131072.0, 131072 * 1024.0 / width)))
        return _gated(rows, width, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                      act=rng.choice(["silu", "silu", "gelu", "gelu_tanh", "relu"]),
                      halves=rng.random() < 0.4, grad=rng.random() < 0.6)
    tensors = int(_log(rng, 1, 200))
    total = _log(rng, 3e3 * tensors, 17e7)
    width = int(_log(rng, 16, min(14336.0, total / tensors)))
    rows = max(1, int(total / tensors / width))
    dtype = rng.choice(["f32", "f32", "bf16", "f16"])
    return _adamw(tensors, rows, width, small=rng.choice([0, 2, 3]), dtype=dtype,
                  bits=rng.choice([32, 8]), master=dtype != "f32" and rng.random() < 0.5,
                  t=rng.choice([0, 1, 100, 20000]))


# ---- inputs -------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(1000003 * (seed + 1))


def _normal(shape, g, scale, dtype):
    return (scale * torch.randn(shape, generator=g, device=DEV)).to(dtype)


def _routing(case, g):
    """(offs, rows, slots) of a routed batch: the experts' ranges of slots, the token of each
    slot (in token order within an expert), the slot of each (token, choice)."""
    t, e, k = case["t"], case["e"], case["k"]
    popular = -0.4 * torch.log(torch.randperm(e, generator=g, device=DEV) + 1.0)
    logits = 1.5 * torch.randn(t, e, generator=g, device=DEV) + popular
    flat = logits.topk(k, dim=-1).indices.reshape(-1)
    order = flat.sort(stable=True).indices
    slots = torch.empty_like(order)
    slots[order] = torch.arange(t * k, device=DEV)
    offs = torch.zeros(e + 1, dtype=torch.int64, device=DEV)
    offs[1:] = torch.bincount(flat, minlength=e).cumsum(0)
    return offs, order // k, slots.reshape(t, k)


def _sizes(case):
    """The elements of each tensor, the weights first, then what belongs to them, and the index
    of the first of those."""
    weights, blocks = case["rows"] * case["width"], max(1, case["rows"] * case["width"] // 64)
    sizes = [weights] * case["tensors"] + [blocks] * (case["tensors"] * case["small"])
    return sizes, case["tensors"]


def _padded(n):
    return -(-n // BLOCK) * BLOCK


def prepare(case, seed):
    g = _gen(seed)
    s = SimpleNamespace(kind=case["kind"], case=case)
    dtype = DTYPES[case["dtype"]]
    if s.kind == "grouped":
        t, e, k, n, width = (case[c] for c in ("t", "e", "k", "n", "width"))
        s.offs, s.rows, s.slots = _routing(case, g)
        if not case["gather"]:
            s.rows = s.slots = None
        x = torch.randn(t if case["gather"] else t * k, width, generator=g, device=DEV)
        x[:, torch.randperm(width, generator=g, device=DEV)[: -(-width // 100)]] *= 20.0
        s.x = x.to(dtype).requires_grad_(case["grad"])
        s.w = torch.empty(e, n, width, dtype=dtype, device=DEV).normal_(0.0, 0.03, generator=g)
        s.w.requires_grad_(case["grad"])
        s.dy = _normal((t * k, n), g, 0.1, dtype) if case["grad"] else None
        return s
    if s.kind == "gated":
        rows, width = case["rows"], case["width"]
        if case["halves"]:
            s.gate, s.up = _normal((rows, 2 * width), g, 2.0, dtype).split(width, 1)
        else:
            s.gate, s.up = (_normal((rows, width), g, 2.0, dtype) for _ in range(2))
        s.gate, s.up = (v.detach().requires_grad_(case["grad"]) for v in (s.gate, s.up))
        s.dh = _normal((rows, width), g, 0.1, dtype) if case["grad"] else None
        return s
    sizes, weights = _sizes(case)
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + _padded(n))
    live = torch.zeros(starts[-1], dtype=torch.bool, device=DEV)
    for a, n in zip(starts, sizes):
        live[a:a + n] = True
    # channels' gradients differ by orders of magnitude; the moments are those of such gradients
    sigma = 1e-3 * torch.exp(1.5 * torch.randn(starts[-1] // BLOCK, 1, generator=g, device=DEV))

    def values(scale):
        return (scale * torch.randn(starts[-1] // BLOCK, BLOCK, generator=g,
                                    device=DEV)).reshape(-1) * live

    s.grad = values(sigma).to(dtype)
    s.p = values(0.03).to(dtype)
    s.master = s.p.float() if case["master"] else None
    s.m = values(0.3 * sigma) * min(case["t"], 1)
    s.v = values(sigma).square() * min(case["t"], 1)
    s.t, s.cut = case["t"], starts[weights]
    if own:
        from hi2_amd.optim import AdamW

        views = [(s.p[a:a + n], s.grad[a:a + n]) for a, n in zip(starts, sizes)]
        s.params = [torch.nn.Parameter(p) for p, _ in views]
        for p, (_, d) in zip(s.params, views):
            p.grad = d
        s.opt = AdamW([dict(params=ps, lr=lr, weight_decay=wd) for ps, (lr, wd) in
                       zip((s.params[:weights], s.params[weights:]), GROUPS) if ps],
                      betas=(BETA1, BETA2), eps=EPS, state_bits=case["bits"],
                      master=case["master"])
        s.opt.load_moments(s.m, s.v, step=s.t)
    elif case["bits"] == 8:
        s.m, s.v = _held_m(s.m), _held_v(s.v)
    return s


# ---- the plain forms ----------------------------------------------------------------------
def _pad(s):
    """The experts that have slots, the slots of each padded to the longest, and which are."""
    counts = s.offs[1:] - s.offs[:-1]
    live = counts.nonzero()[:, 0]
    pad = torch.arange(int(counts.max()), device=DEV)
    ok = pad < counts[live][:, None]
    at = torch.where(ok, s.offs[live][:, None] + pad, torch.zeros_like(pad))
    return live, at, ok


def _plain_grouped(s):
    c, dtype = s.case, s.x.dtype
    with torch.no_grad():
        live, at, ok = _pad(s)
        src = at if s.rows is None else s.rows[at]
        x = s.x.float()[src] * ok[..., None]
        w = s.w[live].float()
        slots = c["t"] * c["k"]
        y = torch.empty(slots, c["n"], dtype=dtype, device=DEV)
        y[at[ok]] = torch.bmm(x, w.transpose(1, 2).contiguous())[ok].to(dtype)
        if not c["grad"]:
            return y
        dy = s.dy.float()[at] * ok[..., None]
        dw = torch.zeros_like(s.w)
        dw[live] = torch.bmm(dy.transpose(1, 2).contiguous(), x).to(dtype)
        d = torch.empty(slots, c["width"], device=DEV)
        d[at[ok]] = torch.bmm(dy, w)[ok]
        dx = d if s.slots is None else d[s.slots].sum(1)
        return dict(y=y, dx=dx.to(dtype), dw=dw)


def _act(x, act):
    """The activation of float32 values and its derivative."""
    if act == "relu":
        return torch.where(x > 0, x, torch.zeros_like(x)), (x > 0).float()
    if act == "silu":
        p = 1 / (1 + torch.exp(-x))
        return x * p, p * (1 + x * (1 - p))
    if act == "gelu":
        # (the upper tail by erfc: 1 + erf loses it where the argument is far below zero)
        p = 0.5 * torch.erfc(-x * math.sqrt(0.5))
        return x * p, p + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)
    a = math.sqrt(2 / math.pi)
    p = 1 / (1 + torch.exp(-2 * a * (x + 0.044715 * x * x * x)))
    return x * p, p + x * p * (1 - p) * 2 * a * (1 + 0.134145 * x * x)


def _plain_gated(s):
    c, dtype = s.case, s.gate.dtype
    with torch.no_grad():
        up = s.up.float()
        h, slope = _act(s.gate.float(), c["act"])
        out = (h * up).to(dtype)
        if not c["grad"]:
            return out
        dh = s.dh.float()
        return dict(h=out, dgate=(dh * up * slope).to(dtype), dup=(dh * h).to(dtype))


def _held(x, steps):
    """Magnitudes as 8 bits to a block of 256 hold them: c^2 d with whole c up to ``steps``,
    d the block's largest divided by steps^2 (32 bits), c the nearest to sqrt(x / d)."""
    x = x.reshape(-1, BLOCK)
    d = x.amax(1, keepdim=True) * (1.0 / steps ** 2)
    d = torch.where(d >= 2.0 ** -126, d, torch.zeros_like(d))
    r = torch.where(d > 0, 1.0 / d.double(), torch.zeros_like(d, dtype=torch.float64)).float()
    # (the borders (c + 1/2)^2 are exact in 32 bits; the root in 64 keeps to their sides)
    c = torch.floor(torch.sqrt((x * r).double()) + 0.5).float()
    return c, d


def _held_m(m):
    c, d = _held(m.abs(), 127)
    return torch.copysign(c * c * d, m.reshape(-1, BLOCK)).reshape(-1)


def _held_v(v):
    """The second moments by their roots; a root that is not zero keeps at least the code 1."""
    root = _root(v)
    c, d = _held(root, 255)
    c = torch.where(root.reshape(-1, BLOCK) > 0, c.clamp_min(1.0), c)
    root = (c * c * d).reshape(-1)
    return root * root


def _root(v):
    return torch.sqrt(v.double()).float()


def _plain_adamw(s):
    c = s.case
    s.t += 1
    correct1, correct2 = 1 - BETA1 ** s.t, 1 - BETA2 ** s.t
    g = s.grad.float()
    m = s.m * BETA1 + g * (1 - BETA1)
    v = s.v * BETA2 + (g * g) * (1 - BETA2)
    quotient = m / (_root(v) * (1 / math.sqrt(correct2)) + EPS)
    p = s.p.float() if s.master is None else s.master
    p = torch.cat([p[a:b] * (1 - lr * wd) - quotient[a:b] * (lr / correct1) for a, b, (lr, wd) in
                   zip((0, s.cut), (s.cut, len(p)), GROUPS)])
    s.p = p.to(s.p.dtype)
    s.m, s.v = (m, v) if c["bits"] == 32 else (_held_m(m), _held_v(v))
    out = dict(p=s.p, m=s.m, v=s.v)
    if s.master is not None:
        out["master"] = s.master = p
    return out


# ---- one pass -----------------------------------------------------------------------------
def run(s):
    if not own:
        return {"grouped": _plain_grouped, "gated": _plain_gated, "adamw": _plain_adamw}[s.kind](s)
    c = s.case
    if s.kind == "grouped":
        from hi2_amd.experts import grouped_linear

        y = grouped_linear(s.x, s.w, s.offs, rows=s.rows, slots=s.slots)
        if not c["grad"]:
            return y
        dx, dw = torch.autograd.grad(y, (s.x, s.w), s.dy)
        return dict(y=y, dx=dx, dw=dw)
    if s.kind == "gated":
        from hi2_amd.experts import gated

        h = gated(s.gate, s.up, activation=c["act"])
        if not c["grad"]:
            return h
        dgate, dup = torch.autograd.grad(h, (s.gate, s.up), s.dh)
        return dict(h=h, dgate=dgate, dup=dup)
    s.opt.step()
    m, v = s.opt.moments()
    out = dict(p=s.p, m=m, v=v)
    if c["master"]:
        out["master"] = s.opt.master
    return out


# ---- the definition in 64 bits --------------------------------------------------------------
def _exact_act(x, act):
    """The activation in 64 bits and its derivative."""
    if act == "relu":
        return x.clamp_min(0), torch.heaviside(x, torch.zeros((), dtype=x.dtype, device=DEV))
    if act == "silu":
        p = torch.special.expit(x)
        return x * p, p + x * p * torch.special.expit(-x)
    if act == "gelu":
        p = torch.special.ndtr(x)
        return x * p, p + x * torch.exp(-x.square() / 2) / math.sqrt(2 * math.pi)
    a = math.sqrt(2 / math.pi)
    th = torch.tanh(a * (x + 0.044715 * x ** 3))
    p = torch.special.expit(2 * a * (x + 0.044715 * x ** 3))
    return x * p, p + 0.5 * x * (1 - th.square()) * a * (1 + 3 * 0.044715 * x.square())


def exact(case, seed):
    s = prepare(case, seed)
    if s.kind == "grouped":
        slots, offs = case["t"] * case["k"], s.offs.tolist()
        x, w = s.x.detach(), s.w.detach()
        y = torch.zeros(slots, case["n"], dtype=torch.float64, device=DEV)
        dx = torch.zeros(x.shape, dtype=torch.float64, device=DEV)
        # (the weights' gradient of the large layers would not fit beside the rest in 64 bits)
        dw = torch.zeros(w.shape, dtype=torch.float64 if w.numel() < 2e8 else torch.float32,
                         device=DEV)
        for e in range(case["e"]):
            at = torch.arange(offs[e], offs[e + 1], device=DEV)
            src = at if s.rows is None else s.rows[at]
            a, b = x[src].double(), w[e].double()
            y[at] = a @ b.T
            if case["grad"]:
                d = s.dy[at].double()
                dw[e] = (d.T @ a).to(dw.dtype)
                dx.index_add_(0, src, d @ b)
        return dict(y=y, dx=dx, dw=dw) if case["grad"] else y
    if s.kind == "gated":
        gate, up = s.gate.detach().double(), s.up.detach().double()
        h, slope = _exact_act(gate, case["act"])
        if not case["grad"]:
            return h * up
        dh = s.dh.double()
        return dict(h=h * up, dgate=dh * up * slope, dup=dh * h)
    t = case["t"] + 1
    g = s.grad.double()
    m = BETA1 * s.m.double() + (1 - BETA1) * g
    v = BETA2 * s.v.double() + (1 - BETA2) * g.square()
    p = (s.p if s.master is None else s.master).double()
    first = torch.arange(len(p), device=DEV) < s.cut
    lr, wd = (torch.where(first, *(torch.tensor(GROUPS[i][j], dtype=torch.float64, device=DEV)
                                   for i in range(2))) for j in range(2))
    p = p - lr * wd * p - lr * (m / (1 - BETA1 ** t)) / (
        torch.sqrt(v / (1 - BETA2 ** t)) + EPS)
    # (codes of 8 bits jump where a value passes a border, which 32 bits and 64 do not share)
    held = case["bits"] == 8
    out = dict(p=p, m=None if held else m, v=None if held else v)
    if case["master"]:
        out["master"] = p
    return out


# ---- what a pass cannot do without ----------------------------------------------------------
def work(case):
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if case["kind"] == "grouped":
        t, e, k, n, width = (case[c] for c in ("t", "e", "k", "n", "width"))
        slots, live = t * k, e * (1 - (1 - k / e) ** t)
        x = t if case["gather"] else slots
        both = 2 if case["grad"] else 1  # tokens and results, and their gradients
        return {"bytes": size * (both * (x * width + slots * n) + live * n * width +
                                 (e * n * width if case["grad"] else 0)) +
                8 * (e + 1 + slots * case["gather"] * both),
                "flops": 2.0 * slots * n * width * (3 if case["grad"] else 1)}
    if case["kind"] == "gated":
        n = case["rows"] * case["width"]
        return {"bytes": size * n * (6 if case["grad"] else 3),
                "flops": n * (30.0 if case["grad"] else 12.0)}
    n = sum(_sizes(case)[0])
    states = 16 if case["bits"] == 32 else 4 + 16 / BLOCK + 8  # 8: and the values they stand for
    return {"bytes": n * (3 * size + states + (8 if case["master"] else 0)),
            "flops": n * (15.0 if case["bits"] == 32 else 40.0)}
