"""Argument checks of the packed products', the router's and the weighted sum's C entries, and
of their Python side: they come before any HIP call, so they run on a host without a GPU."""

import ctypes

import pytest
import torch

from hi2_amd import _lib

FAKE = 1 << 20  # an aligned address that no check reads through


def packed(n=64, k=128, experts=1, **more):
    kp = -(-k // 128) * 128
    d = _lib.Packed(FAKE, FAKE, FAKE, FAKE, experts, n, k, kp, 4 * experts, 4)
    d.had, d.largest = FAKE, FAKE
    for key, value in more.items():
        setattr(d, key, value)
    return d


def epilogue(**more):
    e = _lib.Epilogue(out=FAKE, ld_out=64)
    for key, value in more.items():
        setattr(e, key, value)
    return e


def refused(name, match, *args):
    rc = getattr(_lib.lib(), name)(*args)
    assert rc == _lib.EINVAL and match in _lib.last_error(), (rc, _lib.last_error())


def linear(w=None, x=FAKE, dtype=2, ldx=128, x_rows=4, planes=1, src=None, offs=None, slots=4,
           epi=None):
    w = packed() if w is None else w
    return (ctypes.byref(w), x, dtype, ldx, x_rows, planes, src, offs, slots,
            ctypes.byref(epi or epilogue()), None, 0, None)


@pytest.mark.parametrize("match,args", [
    ("columns a multiple of 16", dict(w=packed(k=120))),
    ("padded columns", dict(w=packed(kp=256))),
    ("too large", dict(w=packed(experts=7001))),
    ("null buffer", dict(w=packed(codes=None))),
    ("256-byte aligned", dict(w=packed(params=FAKE + 16))),
    ("without ranges", dict(w=packed(experts=2))),
    ("dtype 3", dict(dtype=3)),
    ("bad shape", dict(ldx=120)),
    ("null activations", dict(x=None)),
    ("16 bytes", dict(x=FAKE + 8)),
    ("16 bytes", dict(ldx=130)),
    ("3 planes", dict(planes=3)),
    ("5 rows of 4", dict(slots=5)),
    ("bad rows", dict(slots=-1)),
    ("activation 9", dict(epi=epilogue(act=9))),
    ("dtype 7", dict(epi=epilogue(dt_out=7))),
    ("null output", dict(epi=epilogue(out=None))),
    ("rows overlap", dict(epi=epilogue(ld_out=63))),
    ("rows overlap", dict(epi=epilogue(mul=FAKE, ld_mul=1))),
])
def test_packed_linear_refuses(match, args):
    refused("hi2x_packed_linear", match, *linear(**args))


def test_nothing_to_do_and_sizes():
    lib = _lib.lib()
    assert lib.hi2x_packed_linear(*linear(slots=0)) == 0
    w = packed()
    size = lib.hi2x_packed_workspace_bytes
    assert size(ctypes.byref(w), 4, 1, 0, 4, 0, 0) == 0  # few rows need none
    assert size(ctypes.byref(w), 100, 2, 0, 100, 0, 0) >= 100 * 128 * 2 * 2 + 100 * 4
    assert size(ctypes.byref(w), 100, 3, 0, 100, 0, 0) == -1
    assert size(None, 100, 1, 0, 100, 0, 0) == -1
    assert size(ctypes.byref(w), 100, 1, 0, -1, 0, 0) == -1
    assert lib.hi2x_route_workspace_bytes(-1, 8) == -1
    assert lib.hi2x_route_workspace_bytes(8, 513) == -1
    assert lib.hi2x_route_workspace_bytes(64, 8) == 0


def test_activations_refuse():
    w = packed()

    def act(**more):
        a = _lib.ActivationsDesc(FAKE, FAKE, 4, 128, 1, 0)
        for key, value in more.items():
            setattr(a, key, value)
        return ctypes.byref(a)

    def given(a, slots=4, src=None):
        return (ctypes.byref(w), a, src, None, slots, ctypes.byref(epilogue()), None, 0, None)

    name = "hi2x_packed_linear_activations"
    refused(name, "null argument", *given(None))
    refused(name, "padded columns", *given(act(kp=256)))
    refused(name, "0 planes", *given(act(nplanes=0)))
    refused(name, "rows of 4", *given(act(), slots=6))
    refused(name, "not aligned", *given(act(planes=FAKE + 128)))
    refused(name, "4 GiB", *given(act(rows=1 << 25), src=FAKE))
    name = "hi2x_packed_activations"
    x = (ctypes.byref(w), FAKE, 2, 128, 4, None, None)
    refused(name, "null output", *x, None, None)
    refused(name, "planes not aligned", *x, act(planes=FAKE + 2), None)
    refused(name, "6 rows of 4", *x, act(rows=6), None)
    own = packed(experts=2, per_expert=1)
    refused(name, "without ranges", ctypes.byref(own), FAKE, 2, 128, 4, None, None, act(), None)


def test_layout_and_mlp_refuse():
    w = packed(largest=None)
    refused("hi2x_packed_layout", "null buffer", ctypes.byref(w), *[FAKE] * 5, None)
    gate, down, wrong = packed(64, 128), packed(128, 64), packed(64, 64)

    def mlp(g, u, d, dtype=2, act=2, top_k=2, rows=FAKE):
        return (*(ctypes.byref(p) for p in (g, u, d)), FAKE, dtype, 128, 4, top_k, 1, 1, 1, act,
                rows, FAKE, FAKE, FAKE, None, 0, FAKE, 2, None, 0, None)

    name = "hi2x_moe_mlp"
    refused(name, "same experts", *mlp(gate, gate, wrong))
    refused(name, "bad shape", *mlp(gate, gate, down, top_k=0))
    refused(name, "dtype 4", *mlp(gate, gate, down, dtype=4))
    refused(name, "activation -1", *mlp(gate, gate, down, act=-1))
    refused(name, "null buffer", *mlp(gate, gate, down, rows=None))
    size = _lib.lib().hi2x_moe_mlp_workspace_bytes
    assert size(*(ctypes.byref(p) for p in (gate, gate, wrong)), 4, 2, 1, 1, 1) == -1
    few = size(*(ctypes.byref(p) for p in (gate, gate, down)), 4, 2, 1, 1, 1)
    assert few >= 8 * (64 + 64 + 128) * 4


def test_route_and_combine_refuse():
    def route(t=4, e=8, k=2, scoring=0, groups=1, top_groups=1, dtype=0, ld=8):
        return (FAKE, dtype, ld, t, e, k, scoring, None, groups, top_groups, 1, 1.0, FAKE, FAKE,
                FAKE, FAKE, FAKE, None, 0, None)

    for more in (dict(e=513, ld=513), dict(k=9), dict(k=0), dict(scoring=2), dict(dtype=5),
                 dict(ld=7), dict(groups=3), dict(groups=4, top_groups=5), dict(t=-1)):
        assert _lib.lib().hi2x_route(*route(**more)) == _lib.EINVAL, more
        assert "route" in _lib.last_error()

    def combine(dt=0, rows=4, n=16, t=2, k=2, y=FAKE, out=FAKE):
        return (y, dt, rows, n, FAKE, FAKE, t, k, None, 0, out, 0, None)

    for more in (dict(dt=3), dict(n=-1), dict(k=0), dict(y=None), dict(out=None)):
        refused("hi2x_moe_combine", "moe_combine", *combine(**more))
    assert _lib.lib().hi2x_moe_combine(*combine(t=0)) == 0

    def back(dt=0, y=FAKE, t=2, k=2, dw=FAKE):
        return (FAKE, dt, y, 0, 4, 16, FAKE, FAKE, t, k, dw, None, None)

    for more in (dict(dt=3), dict(y=None), dict(k=0), dict(t=-1)):
        refused("hi2x_moe_combine_backward", "moe_combine_backward", *back(**more))
    assert _lib.lib().hi2x_moe_combine_backward(*back(dw=None)) == 0


def test_python_refuses_tensors_of_the_host():
    from hi2_amd.moe import route
    from hi2_amd.packed import PackedLinear, combine

    with pytest.raises(RuntimeError, match="MI355X"):
        route(torch.zeros(2, 4), 2)
    with pytest.raises(RuntimeError, match="MI355X"):
        combine(torch.zeros(4, 8), torch.zeros(2, 2, dtype=torch.int64), torch.ones(2, 2))
    with pytest.raises(RuntimeError, match="MI355X"):
        PackedLinear(None, "cpu")
