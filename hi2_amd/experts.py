"""Training the experts of an MoE layer on the MI355X: products grouped by expert with their
gradients, and the gated activation between them.

The packed experts of :mod:`hi2_amd.packed` are frozen; these are the products of weights that
learn, the experts' own or what :func:`hi2_amd.qad_kernel.original` decodes from latents, over the
routed slots of :func:`hi2_amd.moe.route` (``hi2/moe.py:83-100``).

* :func:`grouped_linear`: ``x[rows] w[e]^T`` for every expert's slots, with gradients to the tokens
  and to the weights.
* :func:`gated`: ``act(gate) * up``, with both gradients.
* :func:`experts_mlp`: the gated MLP of experts and its weighted sum, from these and
  :func:`hi2_amd.packed.combine`.

Inputs are float32, float16 or bfloat16; sums are float32 and every result is rounded once to its
inputs' type."""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .optim import _tensors
from .packed import ACTIVATIONS, DTYPES, combine

__all__ = ["grouped_linear", "gated", "experts_mlp"]

_LINEAR, _GRAD_X, _GRAD_W = 0, 1, 2


def _rows(x: torch.Tensor) -> torch.Tensor:
    """``x [rows, n]`` as the kernels take it: neighbours in a row next to each other, rows not
    overlapping (expanded and transposed tensors are copied)."""
    if x.shape[1] > 1 and x.stride(1) != 1 or x.shape[0] > 1 and x.stride(0) < x.shape[1]:
        return x.contiguous()
    return x


def _near_rows(x: torch.Tensor) -> torch.Tensor:
    """The same for the grouped products, whose rows are less than 2^21 elements apart (as those of
    ``h[:, -1]`` of long sequences are not: they are copied)."""
    if x.shape[0] > 1 and x.stride(0) >= 1 << 21:
        return x.contiguous()
    return _rows(x)


def _pitch(x: torch.Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _aligned(x: torch.Tensor) -> bool:
    return (x.data_ptr() | _pitch(x) * x.element_size()) % 16 == 0


def _type_of(what: str, **tensors) -> int:
    """The one type of the tensors."""
    first = next(iter(tensors.values())).dtype
    if first not in DTYPES:
        raise ValueError(f"{what}: {next(iter(tensors))} is {first} (float32, float16 or bfloat16)")
    for name, t in tensors.items():
        if t.dtype != first:
            raise ValueError(f"{what}: {name} is {t.dtype}, expected {first} as the others")
    return DTYPES[first]


def _workspace(dev, *args):
    size = _lib.lib().hi2x_grouped_workspace_bytes(*args)
    if size < 0:
        raise RuntimeError(f"hi2x_grouped_workspace_bytes: {_lib.last_error()}")
    return (torch.empty(size, dtype=torch.uint8, device=dev), size) if size else (None, 0)


def _linear(x, w, offs, rows, slots):
    e, n, k = w.shape
    dt = DTYPES[x.dtype]
    out = torch.empty(slots, n, dtype=x.dtype, device=x.device)
    if slots and n:
        ws, size = _workspace(x.device, _LINEAR, dt, x.shape[0], _pitch(x), e, n, k, slots,
                              rows is not None, _aligned(x), _aligned(w.view(e * n, k)))
        _lib.call("hi2x_grouped_linear", x.device, x.data_ptr(), dt, _pitch(x), x.shape[0],
                  w.data_ptr(), e, n, k, _lib.ptr(rows), offs.data_ptr(), slots, out.data_ptr(),
                  _lib.ptr(ws), size)
    return out


class _Grouped(torch.autograd.Function):
    """The product with gradients to x and w."""

    @staticmethod
    def forward(ctx, x, w, offs, rows, slots_of, slots):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, w, offs, rows, slots_of)
        return _linear(x, w, offs, rows, slots)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        if grad is None:
            return (None,) * 6
        # (saved tensors' hooks may give them back in other strides than they were saved with)
        x, w, offs, rows, slots_of = ctx.saved_tensors
        x, w, offs = _near_rows(x), w.contiguous(), offs.contiguous()
        rows, slots_of = (v if v is None else v.contiguous() for v in (rows, slots_of))
        e, n, k = w.shape
        dev, dt, slots = x.device, DTYPES[x.dtype], grad.shape[0]
        grad = _near_rows(grad)
        dx = dw = None
        if ctx.needs_input_grad[0]:
            dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
            top_k = 0 if slots_of is None else slots_of.shape[1]
            if x.shape[0]:
                ws, size = _workspace(dev, _GRAD_X, dt, x.shape[0], k, e, n, k, slots,
                                      slots_of is not None, _aligned(grad),
                                      _aligned(w.view(e * n, k)))
                _lib.call("hi2x_grouped_grad_x", dev, grad.data_ptr(), dt, _pitch(grad),
                          w.data_ptr(), e, n, k, offs.data_ptr(), slots, _lib.ptr(slots_of),
                          x.shape[0], top_k, dx.data_ptr(), _lib.ptr(ws), size)
        if ctx.needs_input_grad[1]:
            dw = torch.empty(e, n, k, dtype=w.dtype, device=dev)
            ws, size = _workspace(dev, _GRAD_W, dt, x.shape[0], _pitch(x), e, n, k, slots,
                                  rows is not None, _aligned(grad), _aligned(x))
            _lib.call("hi2x_grouped_grad_w", dev, grad.data_ptr(), dt, _pitch(grad), x.data_ptr(),
                      _pitch(x), x.shape[0], e, n, k, _lib.ptr(rows), offs.data_ptr(), slots,
                      dw.data_ptr(), _lib.ptr(ws), size)
        return dx, dw, None, None, None, None


def _index(what, name, t, shape):
    if t.dtype != torch.int64 or (shape is not None and tuple(t.shape) != shape):
        raise ValueError(f"{what}: {name} is {t.dtype} {tuple(t.shape)}, expected int64"
                         f"{'' if shape is None else f' {shape}'}")
    return t.contiguous()


def grouped_linear(x: torch.Tensor, w: torch.Tensor, offs: torch.Tensor,
                   rows: torch.Tensor | None = None, slots: torch.Tensor | None = None
                   ) -> torch.Tensor:
    """``[S, N]``: row j is ``x[rows[j]] w[e]^T`` for the slots j of expert e's range
    ``offs[e]:offs[e + 1]`` (row j of ``x [T, K]`` itself without ``rows``), with ``w [E, N, K]``.

    ``offs`` (E + 1 entries, ascending, 0 to S), ``rows [S]`` and ``slots [T, k]`` are those of
    :func:`hi2_amd.moe.route`, int64 on the device, and are never read by the host.  A row outside
    x is taken as a row of NaN; a slot outside all ranges gets zeros, so that a batch may be padded
    behind its last range.

    x and w have gradients where they require them: an expert without slots gets zeros.  With
    ``rows``, x's takes ``slots``, the slots of each token, and is the float32 sum over them, in
    their order, of what each slot has.  Everything is of one type; 1 to 7000 experts, N and K below
    2^20, S and T below 2^31."""
    if x.dim() != 2 or w.dim() != 3 or w.shape[2] != x.shape[1]:
        raise ValueError(f"grouped_linear: x {tuple(x.shape)} and w {tuple(w.shape)}, expected "
                         "[T, K] and [E, N, K]")
    dev = _lib.require_gpu(x, w, offs, rows, slots)
    _lib.refuse_tangents("grouped_linear", x, w)
    _type_of("grouped_linear", x=x, w=w)
    e, n, k = w.shape
    if e < 1 or n < 1 or k < 1:
        raise ValueError(f"grouped_linear: w of shape {tuple(w.shape)} is empty")
    offs = _index("grouped_linear", "offs", offs, (e + 1,))
    if rows is not None:
        rows = _index("grouped_linear", "rows", rows, (rows.numel(),))
    count = x.shape[0] if rows is None else rows.numel()
    if slots is not None:
        if rows is None:
            raise ValueError("grouped_linear: slots without rows")
        if slots.dim() != 2 or slots.shape[0] != x.shape[0] or slots.shape[1] < 1:
            raise ValueError(f"grouped_linear: slots {tuple(slots.shape)} for {x.shape[0]} tokens")
        slots = _index("grouped_linear", "slots", slots, None)
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad):
        if x.requires_grad and rows is not None and slots is None:
            raise ValueError("grouped_linear: with rows, the gradient of x takes slots")
        return _Grouped.apply(_near_rows(x), w.contiguous(), offs, rows, slots, count)
    return _linear(_near_rows(x), w.contiguous(), offs, rows, count)


_gated_graph = None


def _bind():
    """The host extension's activation with its gradients, on the library's entries."""
    global _gated_graph
    module, lib = _tensors(), _lib.lib()
    module.bind(*(ctypes.cast(f, ctypes.c_void_p).value for f in (
        lib.hi2x_gated, lib.hi2x_gated_backward, lib.hi2x_last_error)))
    _gated_graph = module.gated
    return _gated_graph


def _gated(gate, up, act):
    rows, n = gate.shape
    out = torch.empty(rows, n, dtype=gate.dtype, device=gate.device)
    if rows and n:
        _lib.call("hi2x_gated", gate.device, gate.data_ptr(), _pitch(gate), up.data_ptr(),
                  _pitch(up), rows, n, DTYPES[gate.dtype], act, out.data_ptr(), n)
    return out


def gated(gate: torch.Tensor, up: torch.Tensor, activation: str = "silu") -> torch.Tensor:
    """``activation(gate) * up`` of two tensors of one shape ``[..., N]`` and type (rows may be
    strided, as the halves of one product's rows are), with gradients to both where they require
    them: in float32, rounded once.  ``activation`` one of none, relu, silu, gelu (erf) and
    gelu_tanh."""
    _lib.require_gpu(gate, up)
    _lib.refuse_tangents("gated", gate, up)
    if gate.shape != up.shape or gate.dim() < 1:
        raise ValueError(f"gated: gate {tuple(gate.shape)} and up {tuple(up.shape)}: one shape "
                         "[..., N] expected")
    _type_of("gated", gate=gate, up=up)
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation {activation!r} ({', '.join(ACTIVATIONS)})")
    shape = gate.shape
    if gate.dim() != 2:
        rows = gate.numel() // shape[-1] if shape[-1] else 0
        gate, up = gate.reshape(rows, shape[-1]), up.reshape(rows, shape[-1])
    gate, up = _rows(gate), _rows(up)
    if torch.is_grad_enabled() and (gate.requires_grad or up.requires_grad):
        out = (_gated_graph or _bind())(gate, up, act)
    else:
        out = _gated(gate, up, act)
    return out if len(shape) == 2 else out.view(shape)


def experts_mlp(x: torch.Tensor, routing, gate: torch.Tensor, up: torch.Tensor,
                down: torch.Tensor, activation: str = "silu", residual=None) -> torch.Tensor:
    """The gated MLP of experts over routed tokens,
    ``residual + sum_j w_j down(activation(gate(x)) * up(x))``, for ``x [..., K]``, the
    :class:`hi2_amd.moe.Routing` of its tokens, ``gate`` and ``up [E, I, K]`` and ``down [E, K, I]``,
    as x's shape and type; the differentiable form of :func:`hi2_amd.packed.moe_mlp`.  The parts
    are :func:`grouped_linear`, :func:`gated` and :func:`hi2_amd.packed.combine` and hand on values
    of x's type; x, the weights, the routing's weights and the residual have gradients where they
    require them."""
    if routing is None:
        raise TypeError("experts_mlp takes a Routing")
    if x.dim() < 1:
        raise ValueError("experts_mlp: x is a scalar, expected [..., K]")
    if gate.dim() != 3 or gate.shape != up.shape or \
            tuple(down.shape) != (gate.shape[0], gate.shape[2], gate.shape[1]):
        raise ValueError(f"experts_mlp: gate {tuple(gate.shape)}, up {tuple(up.shape)} and down "
                         f"{tuple(down.shape)}: [E, I, K] twice and [E, K, I] expected")
    if x.shape[-1] != gate.shape[2]:
        raise ValueError(f"experts_mlp: x {tuple(x.shape)}, expected {gate.shape[2]} columns")
    _type_of("experts_mlp", x=x, gate=gate, up=up, down=down)
    flat = x.reshape(-1, x.shape[-1])
    r = routing
    if r.slots.dim() != 2 or r.slots.shape[0] != flat.shape[0]:
        raise ValueError(f"experts_mlp: routing of {r.slots.shape[0]} tokens for {flat.shape[0]}")
    if r.rows.numel() != r.slots.numel():
        raise ValueError(f"experts_mlp: routing of {r.rows.numel()} rows for {r.slots.numel()} "
                         "slots")
    g = grouped_linear(flat, gate, r.offs, r.rows, r.slots)
    u = grouped_linear(flat, up, r.offs, r.rows, r.slots)
    y = grouped_linear(gated(g, u, activation), down, r.offs)
    return combine(y, r.slots, r.weights, residual, x.dtype).view(x.shape)
