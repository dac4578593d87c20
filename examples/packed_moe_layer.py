"""An MoE layer from its weights to its outputs on packed tensors: every expert's projections
are rounded and packed (INT2 and INT4 rows), laid out once, and a batch of tokens goes through
the router, the experts' products and their weighted sum.  With ``--train`` the router's
weights then take a few steps against the unquantised layer's outputs, the experts frozen.

    python examples/packed_moe_layer.py --tokens 1024 --experts 16 --top-k 4 --train 20
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

from hi2_amd.encode import encode_rows  # noqa: E402
from hi2_amd.format import assemble, fwht_groups  # noqa: E402
from hi2_amd.moe import route  # noqa: E402
from hi2_amd.packed import PackedExperts, PackedLinear, moe_mlp, packed_linear  # noqa: E402


def pack(w: torch.Tensor, int2: float = 0.25):
    """``w [N, K]`` (device) packed with the first ``int2`` of its rows in INT2, blocks of 32,
    the others in INT4, blocks of 64, all columns rotated."""
    n, k = w.shape
    had = torch.ones(k // 16, dtype=torch.uint8)
    stored = fwht_groups(w.float(), had.to(w.device))
    cut = int(n * int2)
    pieces, nbits, block = [], torch.full((n,), 4), torch.full((n,), 64)
    nbits[:cut], block[:cut] = 2, 32
    flat = torch.ones(k, device=w.device)
    for rows, nb, b in ((torch.arange(cut), 2, 32), (torch.arange(cut, n), 4, 64)):
        if len(rows):
            e = encode_rows(stored[rows.to(w.device)], flat, nb, b)
            pieces.append((rows, e.codes, e.params, e.consts))
    return assemble(pieces, nbits, block, had, k)


def layer(tokens=256, experts=8, top_k=2, hidden=256, inter=128, train=0, dev="cuda"):
    """Returns (relative error of the packed layer's output, of its shared product, losses)."""
    g = torch.Generator(dev).manual_seed(0)

    def weights(n, k):
        return torch.randn(n, k, generator=g, device=dev) / k ** 0.5

    gate, up = ([weights(inter, hidden) for _ in range(experts)] for _ in range(2))
    down = [weights(hidden, inter) for _ in range(experts)]
    packed = [PackedExperts([pack(w) for w in p], dev) for p in (gate, up, down)]
    router, shared = weights(experts, hidden), weights(hidden, hidden)
    x = torch.randn(tokens, hidden, generator=g, device=dev).bfloat16()

    r = route((x.float() @ router.T), top_k)
    out = moe_mlp(x, r, *packed, residual=x)
    want = x.float()
    for e in range(experts):
        tok, j = (r.index == e).nonzero(as_tuple=True)
        v = x[tok].float()
        h = torch.nn.functional.silu(v @ gate[e].T) * (v @ up[e].T)
        want.index_add_(0, tok, r.weights[tok, j, None] * (h @ down[e].T))
    one = packed_linear(x, PackedLinear(pack(shared), dev))

    losses = []
    logits = torch.nn.Parameter(x.float() @ router.T)
    opt = torch.optim.SGD([logits], lr=200.0)
    for _ in range(train):
        opt.zero_grad()
        y = moe_mlp(x, route(logits, top_k), *packed, residual=x)
        loss = (y.float() - want).square().sum() / want.square().sum()
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))

    def off(a, b):
        return float((a.float() - b).norm() / b.norm())

    return off(out, want), off(one, x.float() @ shared.T), losses


if __name__ == "__main__":
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in (("tokens", 256), ("experts", 8), ("top-k", 2), ("hidden", 256),
                        ("inter", 128), ("train", 0)):
        p.add_argument(f"--{name}", type=int, default=value)
    moe, one, losses = layer(**{k.replace("-", "_"): v for k, v in vars(p.parse_args()).items()})
    print(f"packed layer against its unquantised weights: relative error {moe:.3f}, one product "
          f"{one:.3f}")
    if losses:
        print(f"loss over the router's steps: {losses[0]:.6f} -> {losses[-1]:.6f}")
