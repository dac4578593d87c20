"""Argument checks of the training operators' C entries: they come before any HIP call, so they run
on a host without a GPU."""

import ctypes

import numpy as np
import pytest
import torch

from hi2_amd import _lib
from hi2_amd.optim import _TENSOR

FAKE = 1 << 20  # an aligned address that no check reads through


def refused(name, match, *args):
    rc = getattr(_lib.lib(), name)(*args)
    assert rc == _lib.EINVAL and match in _lib.last_error(), (rc, _lib.last_error())


def linear(x=FAKE, dtype=2, ldx=64, x_rows=8, w=FAKE, experts=2, n=32, k=64, rows=FAKE, offs=FAKE,
           slots=8, out=FAKE):
    return x, dtype, ldx, x_rows, w, experts, n, k, rows, offs, slots, out, None, 0, None


@pytest.mark.parametrize("match,args", [
    ("dtype 3", dict(dtype=3)),
    ("0 experts", dict(experts=0)),
    ("7001 experts", dict(experts=7001)),
    ("weights of 0 x 64", dict(n=0)),
    ("weights of 32 x 1048576", dict(k=1 << 20, ldx=1 << 20)),
    ("bad rows", dict(slots=-1)),
    ("bad rows", dict(slots=1 << 31)),
    ("8 rows for 9 slots", dict(rows=None, slots=9)),
    ("overlap", dict(ldx=63)),
    ("2^21 elements apart", dict(ldx=1 << 21)),
    ("null buffer", dict(x=None)),
    ("null buffer", dict(w=None)),
    ("null buffer", dict(offs=None)),
    ("null buffer", dict(out=None)),
    ("too many results", dict(n=(1 << 20) - 1, x_rows=(1 << 31) - 1, slots=(1 << 31) - 1)),
])
def test_grouped_linear_refuses(match, args):
    refused("hi2x_grouped_linear", match, *linear(**args))


def grad_x(dy=FAKE, dtype=2, ldy=32, w=FAKE, experts=2, n=32, k=64, offs=FAKE, slots=8,
           slots_of=FAKE, t=4, top_k=2, dx=FAKE, ws=None, size=0):
    return dy, dtype, ldy, w, experts, n, k, offs, slots, slots_of, t, top_k, dx, ws, size, None


@pytest.mark.parametrize("match,args", [
    ("dtype -1", dict(dtype=-1)),
    ("bad routing", dict(top_k=0)),
    ("bad r", dict(t=-1)),
    ("overlap", dict(ldy=31)),
    ("null buffer", dict(dy=None)),
    ("null buffer", dict(dx=None)),
    ("workspace of 16 bytes", dict(ws=FAKE, size=16)),
    ("256-byte aligned", dict(ws=FAKE + 16, size=1 << 20)),
])
def test_grouped_grad_x_refuses(match, args):
    refused("hi2x_grouped_grad_x", match, *grad_x(**args))


def grad_w(dy=FAKE, dtype=2, ldy=32, x=FAKE, ldx=64, x_rows=8, experts=2, n=32, k=64, rows=FAKE,
           offs=FAKE, slots=8, dw=FAKE):
    return dy, dtype, ldy, x, ldx, x_rows, experts, n, k, rows, offs, slots, dw, None, 0, None


@pytest.mark.parametrize("match,args", [
    ("overlap", dict(ldx=60)),
    ("overlap", dict(ldy=30)),
    ("null buffer", dict(dw=None)),
    ("null buffer", dict(x=None)),
    ("8 rows for 7 slots", dict(rows=None, slots=7)),
])
def test_grouped_grad_w_refuses(match, args):
    refused("hi2x_grouped_grad_w", match, *grad_w(**args))


def test_workspace_query_refuses():
    size = _lib.lib().hi2x_grouped_workspace_bytes
    assert size(3, 0, 1, 1, 1, 1, 1, 1, 0, 1, 1) == -1
    assert size(0, 5, 1, 1, 1, 1, 1, 1, 0, 1, 1) == -1
    assert size(1, 0, 1, 1, 0, 1, 1, 1, 0, 1, 1) == -1
    assert size(1, 2, 100, 128, 4, 64, 128, 200, 1, 1, 1) >= 200 * 128 * 2
    # copies: of unaligned operands, and of rows beyond an index's reach
    plain = size(0, 2, 100, 128, 4, 64, 128, 200, 1, 1, 1)
    assert plain < 1 << 20
    assert size(0, 2, 100, 128, 4, 64, 128, 200, 1, 0, 1) >= plain + 100 * 128 * 2
    assert size(0, 2, 100, 128, 4, 64, 127, 300, 1, 1, 0) >= plain + 4 * 64 * 128 * 2
    assert size(0, 2, 100, 128, 4, 64, 127, 200, 1, 1, 0) == 0  # (a few slots take them as they are)
    assert size(0, 2, 1 << 20, 1 << 12, 4, 64, 4096, 300, 1, 1, 1) >= 300 * 4096 * 2


def gated(gate=FAKE, ldg=64, up=FAKE, ldu=64, rows=4, n=64, dtype=2, act=2, out=FAKE, ldo=64):
    return gate, ldg, up, ldu, rows, n, dtype, act, out, ldo, None


@pytest.mark.parametrize("match,args", [
    ("dtype 3", dict(dtype=3)), ("activation 5", dict(act=5)), ("bad shape", dict(rows=-1)),
    ("null buffer", dict(gate=None)), ("null buffer", dict(out=None)), ("overlap", dict(ldg=63)),
    ("overlap", dict(ldo=63)), ("too many", dict(rows=1 << 35, ldg=65, n=64)),
])
def test_gated_refuses(match, args):
    refused("hi2x_gated", match, *gated(**args))


def test_gated_backward_refuses():
    ok = [FAKE, 64, FAKE, 64, FAKE, 64, 4, 64, 2, 2, FAKE, 64, FAKE, 64, None]
    for at, value, match in [(0, None, "null"), (2, None, "null"), (10, None, "null"),
                             (12, None, "null"), (1, 60, "overlap"), (11, 60, "overlap"),
                             (8, 4, "dtype 4")]:
        args = list(ok)
        args[at] = value
        refused("hi2x_gated_backward", match, *args)


def adamw(tensors=((100, 0, 0, 0), (5000, 256, 1, 0)), dtype=0, bits=32, groups=1, m=FAKE, v=FAKE,
          mu=FAKE, vu=FAKE, master=None, steps=FAKE, done=FAKE, table=FAKE, count=None,
          params=(FAKE, FAKE), grads=(FAKE, FAKE)):
    host = np.zeros(len(tensors), dtype=_TENSOR)
    for i, t in enumerate(tensors):
        host[i] = (*t, 0)
    adamw.keep = host, (ctypes.c_void_p * 2)(*params), (ctypes.c_void_p * 2)(*grads), \
        (_lib.AdamwGroup * 2)()
    return (host.ctypes.data, table, adamw.keep[1], adamw.keep[2],
            len(tensors) if count is None else count, dtype, bits, adamw.keep[3], groups, m, v, mu,
            vu, master, steps, done, None)


@pytest.mark.parametrize("match,args", [
    ("bad counts", dict(count=-1)),
    ("dtype 3", dict(dtype=3)),
    ("moments of 16 bits", dict(bits=16)),
    ("master of float32", dict(master=FAKE)),
    ("null argument", dict(m=None)),
    ("null argument", dict(steps=None)),
    ("null argument", dict(table=None)),
    ("null argument", dict(bits=8, mu=None)),
    ("not aligned", dict(m=FAKE + 4)),
    ("overlaps", dict(tensors=((100, 0, 0, 0), (5000, 0, 1, 0)))),
    ("overlaps", dict(tensors=((100, 0, 0, 0), (5000, 260, 1, 0)))),
    ("overlaps", dict(tensors=((0, 0, 0, 0), (5000, 256, 0, 0)))),
    ("chunks of tensor 1", dict(tensors=((100, 0, 0, 0), (5000, 256, 2, 0)))),
    ("group 1 of tensor 1", dict(tensors=((100, 0, 0, 0), (5000, 256, 1, 1)))),
    ("group 0 of tensor 1", dict(tensors=((100, 0, 0, 1), (5000, 256, 1, 0)), groups=2)),
    ("null parameter 1", dict(params=(FAKE, None))),
])
def test_adamw_refuses(match, args):
    refused("hi2x_adamw_step", match, *adamw(**args))


def test_adamw_conversions_refuse():
    refused("hi2x_adamw_hold", "null", FAKE, FAKE, 4, FAKE, FAKE, None, FAKE, None)
    refused("hi2x_adamw_hold", "aligned", FAKE + 4, FAKE, 4, FAKE, FAKE, FAKE, FAKE, None)
    refused("hi2x_adamw_moments", "blocks", FAKE, FAKE, FAKE, FAKE, -1, FAKE, FAKE, None)


def test_addresses_of_tensors_are_checked():
    from hi2_amd import _tensors

    sizes, out = np.array([4], dtype=np.int64), np.zeros((2, 1), dtype=np.uint64)
    more = sizes.ctypes.data, 0, 0, out[0].ctypes.data, out[1].ctypes.data
    assert _tensors.addresses([], *more) == []
    for bad in ([torch.zeros(4)], [torch.zeros(5)], [torch.zeros(4, dtype=torch.float64)], [3]):
        with pytest.raises(RuntimeError, match="AdamW"):
            _tensors.addresses(bad, *more)
    with pytest.raises(TypeError):
        _tensors.addresses((), *more)
    with pytest.raises(ValueError, match="dtype 3"):
        _tensors.addresses([], sizes.ctypes.data, 3, 0, 0, 0)
