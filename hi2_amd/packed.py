"""Running an encoded model on the MI355X: products by packed tensors.

``hi2.format.reference_linear`` (``hi2/format.py:195-249``) defines what a packed tensor
computes: ``y = T(x) Wq^T`` with ``Wq = fp16(lo + code * step)`` per ladder block and ``T``
the smoothing and rotation of the activations (``H16(x / col_scale)`` on the flagged
16-column groups).  Here the packed rows are never unpacked to memory: the codes are laid
out once per tensor in the order the matrix instructions take them and decoded in
registers on the way.

* :class:`PackedLinear`: one tensor, laid out.  :func:`packed_linear` multiplies by it with
  bias, activation, factor and residual in the epilogue, from one token to long prompts.
* :class:`PackedExperts`: the experts of one projection of an MoE layer.
  :func:`experts_linear` multiplies every expert's routed slots in one launch, in the order
  :func:`hi2_amd.moe.route` gives; :func:`combine` is the weighted sum over each token's
  experts; :func:`moe_mlp` runs a gated MLP of them.
* :func:`activations`: the transformed activations, for tensors that share their input
  (q, k, v; gate, up) to be multiplied one after the other.

Inputs are float32, float16 or bfloat16; products are summed in float32 and rounded once,
to ``out_dtype``.  Their transformed activations have 22 bits, for bfloat16 results of
bfloat16 inputs 11 (an eighth of the result's rounding).  The products have no gradient (the codes are integers; inputs that
require one are refused while gradients are recorded); :func:`combine` has, and
:func:`moe_mlp` to the routing's weights, so that a router can be trained on frozen experts.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass

import numpy as np
import torch

from . import _lib
from .format import GROUP, HI2Tensor

__all__ = ["PackedLinear", "PackedExperts", "Activations", "activations", "packed_linear",
           "experts_linear", "combine", "moe_mlp"]

CHUNK = 128  # columns are padded to whole chunks
FRAG = 16  # rows of one matrix-instruction fragment
CLASSES = [(nb, b) for nb in (2, 4, 8) for b in (16, 32, 64)]
DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}

_CLASS_AT = np.full((256, 256), -1, np.int64)  # class of [nbits, block]
for _i, (_nb, _b) in enumerate(CLASSES):
    _CLASS_AT[_nb, _b] = _i

_SEGMENT = np.dtype([("codes", np.int64), ("params", np.int64), ("frag0", np.int32),
                     ("frags", np.int32), ("nbits", np.int32), ("block", np.int32)])


def _classes_of(t: HI2Tensor, what: str) -> np.ndarray:
    """The class index of each row of ``t``, checked against its shape and offsets."""
    r, k = t.shape
    if k % GROUP or k < GROUP or r < 1:
        raise ValueError(f"{what}: shape {tuple(t.shape)} (columns a multiple of {GROUP})")
    nb8, blk8 = t.row_nbits.cpu().numpy(), t.row_block.cpu().numpy()
    if nb8.shape != (r,) or blk8.shape != (r,):
        raise ValueError(f"{what}: {nb8.size} row widths and {blk8.size} blocks for {r} rows")
    nb, blk = nb8.astype(np.int64), blk8.astype(np.int64)
    cls = _CLASS_AT[nb, blk] if 0 <= min(nb.min(), blk.min()) and \
        max(nb.max(), blk.max()) < 256 else np.full(r, -1)
    if cls.min() < 0:
        at = int(np.argmax(cls < 0))
        raise ValueError(f"{what}: row {at} is INT{nb[at]} in blocks of {blk[at]}")
    if (k % blk).any():
        raise ValueError(f"{what}: K={k} is not a multiple of every row's block")
    code_off = np.concatenate([[0], np.cumsum(k * nb // 32)])
    param_off = np.concatenate([[0], np.cumsum(k // blk)])
    if t.code_off.numel() != r + 1 or t.param_off.numel() != r + 1 or \
            not np.array_equal(t.code_off.cpu().numpy(), code_off) or \
            not np.array_equal(t.param_off.cpu().numpy(), param_off):
        raise ValueError(f"{what}: offsets do not follow from the rows' widths and blocks")
    if t.codes.numel() != code_off[-1] or t.blk_params.numel() != 2 * param_off[-1] or \
            t.row_consts.shape != (r, 3):
        raise ValueError(f"{what}: buffers do not match the offsets")
    if t.codes.dtype != torch.int32 or t.blk_params.dtype != torch.uint8 or \
            t.row_consts.dtype != torch.float16:
        raise ValueError(f"{what}: codes int32, blk_params uint8 and row_consts float16 expected")
    if t.had.numel() != k // GROUP:
        raise ValueError(f"{what}: had has {t.had.numel()} entries, expected {k // GROUP}")
    if t.col_scale is not None and t.col_scale.numel() != k:
        raise ValueError(f"{what}: col_scale has {t.col_scale.numel()} entries, expected {k}")
    return cls


class _Packed:
    """One or more tensors of one shape, laid out on the device (``hi2x_packed_layout``)."""

    def __init__(self, tensors: list[HI2Tensor], device="cuda"):
        dev = torch.device(device)
        if dev.type != "cuda":
            raise RuntimeError(f"hi2_amd.packed runs on the MI355X; got device {dev}")
        if dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        tensors = list(tensors)
        if not tensors:
            raise ValueError("no tensor to lay out")
        n, k = (int(v) for v in tensors[0].shape)
        for i, t in enumerate(tensors):
            if tuple(t.shape) != (n, k):
                raise ValueError(f"expert {i} has shape {tuple(t.shape)}, expected {(n, k)}")
        e = len(tensors)
        if e > 7000:
            raise ValueError(f"{e} experts (at most 7000)")
        kp = -(-k // CHUNK) * CHUNK
        self.device, self.n, self.k, self.kp, self.experts = dev, n, k, kp, e
        segs = np.zeros((e, len(CLASSES)), _SEGMENT)
        slot_rows = []
        codes_at = params_at = frag = 0
        most, tiles, starts = 0, np.zeros(3, np.int64), np.zeros(e, np.int64)
        for i, t in enumerate(tensors):
            cls = _classes_of(t, "tensor" if e == 1 else f"expert {i}")
            first = frag
            starts[i] = FRAG * frag
            cut = np.zeros(3, np.int64)
            order = np.argsort(cls, kind="stable").astype(np.int32)
            ends = np.cumsum(np.bincount(cls, minlength=len(CLASSES)))
            for c in range(len(CLASSES)):
                rows = order[ends[c - 1] if c else 0:ends[c]]
                if not rows.size:
                    continue
                nb, blk = CLASSES[c]
                f = -(-rows.size // FRAG)
                slot_rows += [rows, np.full(f * FRAG - rows.size, -1, np.int32)]
                segs[i, c] = (codes_at, params_at, frag, f, nb, blk)
                codes_at += f * (kp // CHUNK) * 256 * nb
                params_at += -(-(f * (kp // blk) * 64) // 256) * 256
                frag += f
                cut += [-(-f // 4), -(-f // 8), -(-f // 16)]
            most = max(most, frag - first)
            tiles = np.maximum(tiles, cut)
        self._codes = torch.empty(codes_at, dtype=torch.uint8, device=dev)
        self._params = torch.empty(params_at, dtype=torch.uint8, device=dev)
        rows = np.concatenate(slot_rows)
        self._rows = _lib.h2d(torch.from_numpy(rows), dev)
        self._places = None
        if 16 * most <= 8192:  # (beyond, nothing reads them)
            places = np.empty((e, n), np.uint16)
            at = np.flatnonzero(rows >= 0)
            of = np.searchsorted(starts, at, side="right") - 1  # the expert of each slot
            places[of, rows[at]] = at - starts[of]
            self._places = _lib.h2d(torch.from_numpy(places.view(np.int16)), dev)
        self._segments = _lib.h2d(torch.from_numpy(segs.reshape(-1).view(np.uint8)), dev)
        def flat(parts, dtype):
            parts = [_lib.to_device(p.reshape(-1), dev, dtype) for p in parts]
            return (parts[0] if len(parts) == 1 else torch.cat(parts)).contiguous()

        words = flat([t.codes for t in tensors], torch.int32)
        bytes_ = flat([t.blk_params for t in tensors], torch.uint8)
        consts = flat([t.row_consts for t in tensors], torch.float16)
        co = np.concatenate([[0], np.cumsum([t.codes.numel() for t in tensors])])
        po = np.concatenate([[0], np.cumsum([t.blk_params.numel() // 2 for t in tensors])])
        offs = np.stack([
            np.concatenate([t.code_off.cpu().numpy()[:-1].astype(np.int64) + a
                            for t, a in zip(tensors, co)]),
            np.concatenate([t.param_off.cpu().numpy()[:-1].astype(np.int64) + a
                            for t, a in zip(tensors, po)])])
        offs = _lib.h2d(torch.from_numpy(offs), dev)
        # the transform: one for all where every expert has the same
        seen: dict = {}  # experts often share the tensors themselves (all alive here)

        def host(v, dtype):
            if v is not None and id(v) not in seen:
                seen[id(v)] = v.reshape(-1).cpu().to(dtype).numpy()
            return None if v is None else seen[id(v)]

        had = [host(t.had, torch.uint8) for t in tensors]
        cs = [host(t.col_scale, torch.float16) for t in tensors]
        if any(c is None for c in cs) and not all(c is None for c in cs):
            cs = [np.ones(k, np.float16) if c is None else c for c in cs]
        keys = [(h.astype(bool).tobytes(), b"" if c is None else c.tobytes())
                for h, c in zip(had, cs)]
        #: the transform all tensors share, None where experts have their own
        self.transform = keys[0] if all(x == keys[0] for x in keys) else None
        #: no rotation and no smoothing at all
        self.plain = all(c is None for c in cs) and not any(h.any() for h in had)
        own = 1 if self.transform is not None else e
        self._had = _lib.h2d(torch.from_numpy(np.stack(had[:own])), dev)
        self._scale = None if cs[0] is None else \
            _lib.h2d(torch.from_numpy(np.stack(cs[:own])), dev)
        self._largest = torch.empty(1, device=dev)
        first = (_lib.Segment * len(CLASSES)).from_buffer_copy(segs[0].tobytes())
        #: hi2x_packed: the layout, the tables and the transform
        self.desc = _lib.Packed(
            self._codes.data_ptr(), self._params.data_ptr(), self._rows.data_ptr(),
            self._segments.data_ptr(), e, n, k, kp, frag, most,
            (ctypes.c_int64 * 3)(*(int(v) for v in tiles)), self._had.data_ptr(),
            None if self._scale is None else self._scale.data_ptr(), int(self.transform is None),
            self._largest.data_ptr(), None if self._places is None else self._places.data_ptr(),
            first)
        self._ref = ctypes.byref(self.desc)
        _lib.call("hi2x_packed_layout", dev, self._ref, _lib.ptr(words),
                  _lib.ptr(offs[0]), _lib.ptr(bytes_), _lib.ptr(offs[1]), _lib.ptr(consts))

    @property
    def nbytes(self) -> int:
        """Device bytes of the laid-out codes and ladder parameters."""
        return self._codes.numel() + self._params.numel()


class PackedLinear(_Packed):
    """A packed tensor (``HI2Tensor``, host or device buffers) laid out for
    :func:`packed_linear`.  The layout is made once; the tensor is not needed after it."""

    def __init__(self, tensor: HI2Tensor, device="cuda"):
        super().__init__([tensor], device)


class PackedExperts(_Packed):
    """The experts of one projection, one ``HI2Tensor`` each, all of one shape (each with
    its own rows' widths and its own transform)."""


@dataclass
class Activations:
    """Transformed activations (:func:`activations`): usable with every tensor whose
    transform is ``transform``."""

    planes: torch.Tensor  # float16 [rows, kp / 128, nplanes, 128]
    scale: torch.Tensor  # float32 [rows]
    k: int
    dtype: torch.dtype  # of the activations they were made from
    transform: tuple | None
    desc: object


def _no_grad_inputs(what, *tensors):
    _lib.refuse_tangents(what, *tensors)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad() or detach "
                           "its inputs")


def _dtype(t: torch.Tensor | torch.dtype, what: str) -> int:
    d = t if isinstance(t, torch.dtype) else t.dtype
    if d not in DTYPES:
        raise ValueError(f"{what} is {d} (float32, float16 or bfloat16)")
    return DTYPES[d]


def _rows_of(x: torch.Tensor, k: int, what: str) -> torch.Tensor:
    """``x`` as [rows, k] with unit column stride, without a copy where its strides allow."""
    if x.dim() < 1 or x.shape[-1] != k:
        raise ValueError(f"{what} has shape {tuple(x.shape)}, expected {k} columns")
    x = x.reshape(-1, k) if x.dim() != 2 else x
    if x.shape[0] > 1 and x.stride(0) < k or k > 1 and x.stride(1) != 1:
        x = x.contiguous()
    return x


def _pitch(x: torch.Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _planes(dtype: torch.dtype, w: _Packed, out_dtype: torch.dtype) -> int:
    """fp16 planes of the transformed activations.  One plane rounds each value by up to
    2^-11, which a bf16 result of bf16 values hides, but not an fp16 or fp32 one: those
    take two (22 bits), except 16-bit values that the transform leaves as they are."""
    if w.plain and dtype != torch.float32:
        return 1
    return 1 if dtype == out_dtype == torch.bfloat16 else 2


def _aligned(x: torch.Tensor) -> torch.Tensor:
    """Rows that begin at multiples of 16 bytes, as the kernels read them."""
    if _pitch(x) * x.element_size() % 16:
        x = x.contiguous()
    return x.clone() if x.data_ptr() % 16 else x


def activations(x: torch.Tensor, w: PackedLinear | PackedExperts, out_dtype=None
                ) -> Activations:
    """``T(x)`` for ``w`` and every tensor with the same transform, to be handed to
    :func:`packed_linear` or :func:`experts_linear` in the place of ``x [..., K]``.  The
    product then has one row per row of ``x``.  ``out_dtype`` is the type of the results
    (default: x's); where bfloat16 values are held to a bfloat16 result's bits, the products
    refuse a wider one."""
    _same_device(w, "activations", x)
    _no_grad_inputs("activations", x)
    if w.transform is None:
        raise ValueError("the experts have transforms of their own: give experts_linear x itself")
    dt = _dtype(x, "x")
    x = _aligned(_rows_of(x, w.k, "x"))
    rows, npl = x.shape[0], _planes(x.dtype, w, out_dtype or x.dtype)
    planes = torch.empty(rows, w.kp // CHUNK, npl, CHUNK, dtype=torch.float16, device=w.device)
    scale = torch.empty(rows, dtype=torch.float32, device=w.device)
    desc = _lib.ActivationsDesc(planes.data_ptr(), scale.data_ptr(), rows, w.kp, npl, 0)
    _lib.call("hi2x_packed_activations", w.device, w._ref, _lib.ptr(x), dt, _pitch(x), rows, None,
              None, ctypes.byref(desc))
    return Activations(planes, scale, w.k, x.dtype, w.transform, desc)


def _operand(t, slots, n, name):
    """(tensor, address, pitch, dtype) of a factor or residual."""
    if t is None:
        return None, None, 0, 0
    if t.numel() != slots * n:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {slots} rows of {n}")
    dt = _dtype(t, name)
    t = _rows_of(t, n, name)
    return t, t.data_ptr(), _pitch(t), dt


def _product(w, x, src, offs, slots, bias, activation, mul, residual, out_dtype, what):
    """The product of :func:`packed_linear` and :func:`experts_linear`; ``x`` is rows
    ``[rows, K]`` or :class:`Activations`, both on the weights' device already."""
    dev, n = w.device, w.n
    given = not isinstance(x, torch.Tensor)
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation {activation!r} ({', '.join(ACTIVATIONS)})")
    bias_p = bias_dt = 0
    if bias is not None:
        if bias.numel() != n:
            raise ValueError(f"bias has {bias.numel()} entries, expected {n}")
        bias = bias.reshape(-1).contiguous()
        bias_p, bias_dt = bias.data_ptr(), _dtype(bias, "bias")
    mul, mul_p, mul_ld, mul_dt = _operand(mul, slots, n, "mul")
    residual, res_p, res_ld, res_dt = _operand(residual, slots, n, "residual")
    out_dt = _dtype(out_dtype, "out_dtype")
    if given and x.desc.nplanes < _planes(x.dtype, w, out_dtype):
        raise ValueError(f"activations of {x.dtype} made for results of that type: give "
                         f"activations out_dtype={out_dtype}")
    dt = 0 if given else _dtype(x, "x")
    out = torch.empty(slots, n, dtype=out_dtype, device=dev)
    if not slots:
        return out
    epi = _lib.Epilogue(bias_p or None, mul_p, res_p, out.data_ptr(), mul_ld, res_ld, n, bias_dt,
                        mul_dt, res_dt, out_dt, act, 0)
    if given:
        rows, npl = x.scale.numel(), x.desc.nplanes
    else:
        x = _aligned(x)
        rows, npl = x.shape[0], _planes(x.dtype, w, out_dtype)
    size = _lib.lib().hi2x_packed_workspace_bytes(w._ref, rows, npl, given, slots,
                                                  src is not None, offs is not None)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size > 0 else None
    src_p = None if src is None else src.data_ptr()
    offs_p = None if offs is None else offs.data_ptr()
    ws_p = None if ws is None else ws.data_ptr()
    if given:
        _lib.call("hi2x_packed_linear_activations", dev, w._ref, ctypes.byref(x.desc), src_p,
                  offs_p, slots, ctypes.byref(epi), ws_p, size)
    else:
        _lib.call("hi2x_packed_linear", dev, w._ref, x.data_ptr(), dt, _pitch(x), rows, npl,
                  src_p, offs_p, slots, ctypes.byref(epi), ws_p, size)
    return out


def _same_device(w, what, *tensors):
    dev = _lib.require_gpu(*tensors)
    if dev != w.device:
        raise RuntimeError(f"{what}: inputs are on {dev}, the weights on {w.device}")


def _check_activations(x: Activations, w):
    if x.k != w.k or x.transform is None or x.transform != w.transform:
        raise ValueError("activations of another transform than the weights'")


def packed_linear(x: torch.Tensor | Activations, w: PackedLinear, bias=None,
                  activation: str = "none", mul=None, residual=None, out_dtype=None
                  ) -> torch.Tensor:
    """``activation(T(x) Wq^T + bias) * mul + residual`` for ``x [..., K]`` (or its
    :func:`activations`), as ``[..., N]`` in ``out_dtype`` (default: x's): summed in float32,
    rounded once.  ``bias [N]``, ``mul`` and ``residual`` (one row per row of x; rows may be
    strided) in any of the float types; activation one of none, relu, silu, gelu (erf) and
    gelu_tanh."""
    if not isinstance(w, PackedLinear):
        raise TypeError(f"packed_linear takes a PackedLinear, got {type(w).__name__}")
    if isinstance(x, Activations):
        _check_activations(x, w)
        _same_device(w, "packed_linear", x.planes, bias, mul, residual)
        _no_grad_inputs("packed_linear", bias, mul, residual)
        return _product(w, x, None, None, x.scale.numel(), bias, activation, mul, residual,
                        out_dtype or x.dtype, "packed_linear")
    _same_device(w, "packed_linear", x, bias, mul, residual)
    _no_grad_inputs("packed_linear", x, bias, mul, residual)
    rows = _rows_of(x, w.k, "x")
    y = _product(w, rows, None, None, rows.shape[0], bias, activation, mul, residual,
                 out_dtype or x.dtype, "packed_linear")
    return y if x.dim() == 2 else y.view(*x.shape[:-1], w.n)


def _routed(offs, rows, w, what):
    if offs.dtype != torch.int64 or offs.numel() != w.experts + 1:
        raise ValueError(f"{what}: offs is {offs.dtype} of {offs.numel()} entries, expected "
                         f"int64 of {w.experts + 1}")
    if rows is not None and rows.dtype != torch.int64:
        raise ValueError(f"{what}: rows is {rows.dtype}, expected int64")
    return offs.contiguous(), None if rows is None else rows.reshape(-1).contiguous()


def experts_linear(x: torch.Tensor | Activations, w: PackedExperts, offs: torch.Tensor,
                   rows: torch.Tensor | None = None, activation: str = "none", mul=None,
                   residual=None, out_dtype=None) -> torch.Tensor:
    """``[S, N]``: row j is expert e's product for the routed slot j of its range
    ``offs[e]:offs[e + 1]``, which reads row ``rows[j]`` of ``x`` (row j itself without
    ``rows``), with the epilogue of :func:`packed_linear`.  ``offs`` (device int64, E + 1
    entries, 0 to S) and ``rows`` (device int64; an index outside x gives a row of NaN) are
    those of :func:`hi2_amd.moe.route` and are never read by the host; the ranges must cover
    all S slots, rows outside them are left unwritten."""
    if not isinstance(w, PackedExperts):
        raise TypeError(f"experts_linear takes PackedExperts, got {type(w).__name__}")
    given = isinstance(x, Activations)
    _same_device(w, "experts_linear", offs, rows, x.planes if given else x, mul, residual)
    offs, rows = _routed(offs, rows, w, "experts_linear")
    _no_grad_inputs("experts_linear", None if given else x, mul, residual)
    if given:
        _check_activations(x, w)
    else:
        x = _rows_of(x, w.k, "x")
    slots = rows.numel() if rows is not None else (x.scale.numel() if given else x.shape[0])
    return _product(w, x, rows, offs, slots, None, activation, mul, residual,
                    out_dtype or x.dtype, "experts_linear")


def _check_residual(residual, t, n):
    """``residual`` has t rows of n, in any leading dimensions."""
    if residual is not None and (residual.numel() != t * n or residual.shape[-1:] != (n,)):
        raise ValueError(f"residual has shape {tuple(residual.shape)}, expected {(t, n)}")


class _Combine(torch.autograd.Function):
    """:func:`combine` with gradients to y, the weights and the residual."""

    @staticmethod
    def forward(ctx, y, weights, residual, slots, out_dtype):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(y, weights, slots)
        ctx.res = None if residual is None else (residual.shape, residual.dtype)
        return _combine(y, slots, weights, residual, out_dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        if grad is None:
            return (None,) * 5
        y, weights, slots = ctx.saved_tensors
        need_y, need_w, need_r = ctx.needs_input_grad[:3]
        grad = grad.contiguous()
        dw = torch.empty_like(weights) if need_w else None
        dy = torch.zeros_like(y) if need_y else None
        if need_w or need_y:
            ws = _lib.workspace(y.device, "hi2x_moe_combine_grad_workspace_bytes",
                                y.shape[0] if need_y else 0)
            _lib.call("hi2x_moe_combine_grad", y.device, _lib.ptr(grad), _dtype(grad, "grad"),
                      _lib.ptr(y), _dtype(y, "y"), y.shape[0], y.shape[1], _lib.ptr(slots),
                      _lib.ptr(weights), slots.shape[0], slots.shape[1], _lib.ptr(dw),
                      _lib.ptr(dy), _lib.ptr(ws), ws.numel())
        return dy, dw, grad.to(ctx.res[1]).view(ctx.res[0]) if need_r else None, None, None


def combine(y: torch.Tensor, slots: torch.Tensor, weights: torch.Tensor, residual=None,
            out_dtype=None) -> torch.Tensor:
    """``out[t] = residual[t] + sum_j weights[t, j] * y[slots[t, j]]`` over ``y [S, N]``, with
    ``slots`` (int64) and ``weights`` (float32) ``[T, k]`` of :func:`hi2_amd.moe.route`: summed
    in float32 in the order of j, rounded once to ``out_dtype`` (default: residual's, else
    y's).  y, the weights and the residual have gradients where they require them; a row of y
    that several slots name takes the sum of theirs, in their order."""
    _lib.require_gpu(y, slots, weights, residual)
    _lib.refuse_tangents("combine", y, weights, residual)
    if y.dim() != 2:
        raise ValueError(f"y has shape {tuple(y.shape)}, expected [S, N]")
    if slots.dim() != 2 or weights.shape != slots.shape or slots.shape[1] < 1:
        raise ValueError(f"slots {tuple(slots.shape)} and weights {tuple(weights.shape)}: one "
                         "shape [T, k] expected")
    if slots.dtype != torch.int64 or weights.dtype != torch.float32:
        raise ValueError(f"slots {slots.dtype} and weights {weights.dtype}: int64 and float32 "
                         "expected")
    t, n = slots.shape[0], y.shape[1]
    _check_residual(residual, t, n)
    y, slots, weights = y.contiguous(), slots.contiguous(), weights.contiguous()
    if torch.is_grad_enabled() and (y.requires_grad or weights.requires_grad or
                                    residual is not None and residual.requires_grad):
        return _Combine.apply(y, weights, residual, slots, out_dtype)
    return _combine(y, slots, weights, residual, out_dtype)


def _combine(y, slots, weights, residual, out_dtype):
    t, n = slots.shape[0], y.shape[1]
    res = None if residual is None else residual.contiguous()
    out_dtype = out_dtype or (y.dtype if res is None else res.dtype)
    out = torch.empty(t, n, dtype=out_dtype, device=y.device)
    if t and n:
        _lib.call("hi2x_moe_combine", y.device, _lib.ptr(y), _dtype(y, "y"), y.shape[0], n,
                  _lib.ptr(slots), _lib.ptr(weights), t, slots.shape[1], _lib.ptr(res),
                  0 if res is None else _dtype(res, "residual"), _lib.ptr(out),
                  _dtype(out_dtype, "out_dtype"))
    return out


def moe_mlp(x: torch.Tensor, routing, gate: PackedExperts, up: PackedExperts,
            down: PackedExperts, activation: str = "silu", residual=None) -> torch.Tensor:
    """The gated MLP of packed experts over routed tokens:
    ``residual + sum_j w_j down(activation(gate(x)) * up(x))`` for ``x [..., K]`` and the
    :class:`hi2_amd.moe.Routing` of its tokens, as x's shape and type.  Sums are float32 and the
    rounding to x's type is one, at the end; what the experts hand on is float32, for bfloat16
    inputs of more than a few tokens fp16 with an exponent to every 16 values (2^-11 of each,
    an eighth of the result's own rounding, and no less than 2^-39 of the largest of the 16).
    Where the routing's weights (or the residual) require a gradient they have one, from the
    parts' own calls, in float32 between them."""
    for name, p in (("gate", gate), ("up", up), ("down", down)):
        if not isinstance(p, PackedExperts):
            raise TypeError(f"{name} is {type(p).__name__}, expected PackedExperts")
    if (gate.n, gate.k, gate.experts) != (up.n, up.k, up.experts) or \
            (down.k, down.n, down.experts) != (gate.n, gate.k, gate.experts):
        raise ValueError("gate and up [I, K] and down [K, I] of the same experts expected")
    if up.device != gate.device or down.device != gate.device:
        raise RuntimeError("gate, up and down are on different devices")
    if routing is None:
        raise TypeError("moe_mlp takes a Routing")
    rows, offs = routing.rows.contiguous(), routing.offs.contiguous()
    slots, weights = routing.slots.contiguous(), routing.weights.contiguous()
    _same_device(gate, "moe_mlp", x, residual, rows, offs, slots, weights)
    _no_grad_inputs("moe_mlp", x)
    _lib.refuse_tangents("moe_mlp", weights, residual)
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation {activation!r} ({', '.join(ACTIVATIONS)})")
    flat = _aligned(_rows_of(x, gate.k, "x"))
    t = flat.shape[0]
    if slots.dim() != 2 or slots.shape[0] != t:
        raise ValueError(f"routing of {slots.shape[0]} tokens for {t}")
    if offs.numel() != gate.experts + 1:
        raise ValueError(f"routing over {offs.numel() - 1} experts for {gate.experts}")
    if weights.shape != slots.shape or rows.numel() != slots.numel() or slots.shape[1] < 1:
        raise ValueError(f"routing: weights {tuple(weights.shape)}, slots {tuple(slots.shape)} "
                         f"and {rows.numel()} rows do not belong together")
    if rows.dtype != torch.int64 or offs.dtype != torch.int64 or slots.dtype != torch.int64 or \
            weights.dtype != torch.float32:
        raise ValueError("routing: rows, offs and slots int64 and weights float32 expected")
    if residual is not None:
        _check_residual(residual, t, gate.k)
        residual = residual.reshape(t, gate.k).contiguous()
    if torch.is_grad_enabled() and (weights.requires_grad or
                                    residual is not None and residual.requires_grad):
        with torch.no_grad():
            def part(p, v, **more):
                return experts_linear(v, p, offs, out_dtype=torch.float32, **more)

            h = part(up, flat, rows=rows)
            h = part(gate, flat, rows=rows, activation=activation, mul=h)
            y = part(down, h)
        return combine(y, slots, weights, residual, x.dtype).view(x.shape)
    dt = _dtype(x, "x")
    out = torch.empty(x.shape, dtype=x.dtype, device=gate.device)
    if not t:
        return out
    # one fp16 plane of the hidden values (and fp16 between the products) is well below a bf16
    # result's own rounding, and half the products; next to an fp16 result it would show
    npl = max(_planes(x.dtype, gate, x.dtype), _planes(x.dtype, up, x.dtype))
    mid = 1 if dt == 2 else 2
    top_k = slots.shape[1]
    shared = gate.transform is not None and gate.transform == up.transform
    size = _lib.lib().hi2x_moe_mlp_workspace_bytes(gate._ref, up._ref, down._ref, t, top_k, npl,
                                                   mid, shared)
    ws = torch.empty(max(size, 1), dtype=torch.uint8, device=gate.device)
    _lib.call("hi2x_moe_mlp", gate.device, gate._ref, up._ref, down._ref, flat.data_ptr(), dt,
              _pitch(flat), t, top_k, npl, mid, shared, act, rows.data_ptr(), offs.data_ptr(),
              slots.data_ptr(), weights.data_ptr(),
              None if residual is None else residual.data_ptr(),
              0 if residual is None else _dtype(residual, "residual"), out.data_ptr(), dt,
              ws.data_ptr(), size)
    return out
