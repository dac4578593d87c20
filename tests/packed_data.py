"""Packed tensors and 64-bit references for the tests of hi2_amd.packed and moe.route."""

import math

import numpy as np
import torch

from hi2_amd.format import HI2Tensor


def packed_tensor(n, k, classes, seed, had=1.0, smooth=False, step=None):
    """A random HI2Tensor on the host and its decoded weights in float64: ``classes`` a list
    of (nbits, block), every row one of them at random (each class at least once)."""
    rng = np.random.default_rng(seed)
    cls = rng.integers(0, len(classes), n)
    cls[:len(classes)] = np.arange(len(classes))[:n]
    nbits = np.array([classes[c][0] for c in cls])
    block = np.array([classes[c][1] for c in cls])
    words, params, consts, weights = [], [], np.zeros((n, 3), np.float16), np.zeros((n, k))
    for r in range(n):
        nb, b = int(nbits[r]), int(block[r])
        codes = rng.integers(0, 2 ** nb, k)
        per = 32 // nb
        shifted = codes.reshape(-1, per).astype(np.uint64) << (nb * np.arange(per, dtype=np.uint64))
        words.append(shifted.sum(1).astype(np.uint32).view(np.int32))
        u = rng.integers(0, 256, (k // b, 2)).astype(np.uint8)
        params.append(u.reshape(-1))
        st = 0.15 / 255 / (2 ** nb - 1) if step is None else step
        consts[r] = [rng.uniform(-0.08, -0.04), rng.uniform(0.0, 0.02) / 255,
                     st * rng.uniform(0.8, 1.2)]
        c = consts[r].astype(np.float64)
        lo = (u[:, 0] * c[1] + c[0]).astype(np.float32).astype(np.float16).astype(np.float64)
        sp = (u[:, 1] * c[2]).astype(np.float32).astype(np.float16).astype(np.float64)
        w = lo[:, None] + codes.reshape(-1, b) * sp[:, None]
        weights[r] = w.astype(np.float16).astype(np.float64).reshape(-1)
    flags = (rng.random(k // 16) < had).astype(np.uint8)
    scale = torch.from_numpy(rng.uniform(0.5, 2.0, k).astype(np.float16)) if smooth else None
    zero = np.zeros(1, np.int64)
    t = HI2Tensor(
        codes=torch.from_numpy(np.concatenate(words)),
        code_off=torch.from_numpy(np.concatenate([zero, np.cumsum(k * nbits // 32)]).astype(np.int32)),
        blk_params=torch.from_numpy(np.concatenate(params)),
        param_off=torch.from_numpy(np.concatenate([zero, np.cumsum(k // block)]).astype(np.int32)),
        row_consts=torch.from_numpy(consts), row_nbits=torch.from_numpy(nbits.astype(np.uint8)),
        row_block=torch.from_numpy(block.astype(np.uint8)), had=torch.from_numpy(flags),
        shape=(n, k), col_scale=scale)
    return t, weights


def h16():
    i = np.arange(16)
    return np.where(np.bitwise_count(i[:, None] & i[None, :]) & 1, -0.25, 0.25)


def stored(x, t):
    """T(x) in float64 (x a float64 array [rows, k])."""
    if t.col_scale is not None:
        x = x / t.col_scale.numpy().astype(np.float64)
    v = x.reshape(len(x), -1, 16)
    with np.errstate(invalid="ignore"):
        return np.where(t.had.numpy()[:, None] != 0, v @ h16(), v).reshape(x.shape)


def act64(y, name):
    if name == "relu":
        return np.maximum(y, 0)
    if name == "silu":
        return y / (1 + np.exp(-y))
    if name == "gelu":
        return 0.5 * y * (1 + np.vectorize(math.erf)(y / math.sqrt(2)))
    if name == "gelu_tanh":
        return 0.5 * y * (1 + np.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    return y


UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# what the rounding of the transformed activations can cost, of each: one fp16 plane for
# 16-bit inputs (half an ulp, 2^-11 of the value), two for float32 (2^-22), besides the
# float32 sums of the transform
X_UNIT = {torch.float32: 2.0 ** -21, torch.float16: 2.0 ** -11 + 2.0 ** -21,
          torch.bfloat16: 2.0 ** -11 + 2.0 ** -21}


def bound(out, dtype, x_dtype, xs, w, slope):
    """An elementwise bound on a product's error: half an ulp of the result, the rounding of
    the activations and of float32 sums (at most one unit of 2^-23 a term) against the sum of
    magnitudes, times the steepest slope of what follows; 2^-24 for fp16's subnormals."""
    k = xs.shape[1]
    mass = np.abs(xs) @ np.abs(w).T
    tiny = 2.0 ** -24 if dtype == torch.float16 else 1e-37
    return (UNIT[dtype] * np.abs(out) + slope * (X_UNIT[x_dtype] + (k + 64) * 2.0 ** -23) * mass
            + 2.0 ** -21 * np.abs(out) + tiny)


def route64(logits, k, scoring="softmax", bias=None, groups=1, top_groups=None, renorm=True,
            scale=1.0):
    """The router by its definition, a token at a time, float64: (index, weights, scores)."""
    v = np.where(np.isnan(logits), -np.inf, logits.astype(np.float64))
    t, e = v.shape
    top_groups = top_groups or groups
    index, weights, scores = np.zeros((t, k), np.int64), np.zeros((t, k)), np.zeros((t, e))
    for i in range(t):
        if scoring == "sigmoid":
            p = 1 / (1 + np.exp(-v[i]))
        else:
            m = v[i].max()
            p = np.exp(v[i] - m) if np.isfinite(m) else np.zeros(e)
            p = p / p.sum() if p.sum() > 0 else p
        scores[i] = p
        key = v[i].copy() if bias is None else np.where(np.isneginf(v[i]), -np.inf, p + bias)
        if top_groups < groups:
            by = key.reshape(groups, -1)
            two = bias is not None and by.shape[1] > 1
            good = np.sort(by, 1)[:, -1] + (np.sort(by, 1)[:, -2] if two else 0)
            keep = np.argsort(-good, kind="stable")[:top_groups]
            out = np.ones(groups, bool)
            out[keep] = False
            rank = np.where(np.repeat(out, e // groups), 1, 0)
        else:
            rank = np.zeros(e)
        order = np.lexsort((np.arange(e), -key, rank))
        index[i] = order[:k]
        w = p[index[i]]
        if renorm:
            w = w / w.sum() if w.sum() > 0 else np.zeros(k)
        weights[i] = scale * w
    return index, weights, scores


def order64(index, e):
    """(rows, offs, slots) of a routed batch."""
    flat = index.reshape(-1)
    order = np.argsort(flat, kind="stable")
    offs = np.concatenate([[0], np.cumsum(np.bincount(flat, minlength=e))])
    slots = np.empty(flat.size, np.int64)
    slots[order] = np.arange(flat.size)
    return order // index.shape[1], offs, slots.reshape(index.shape)
