"""The host side of the packed products: sizes and checks that need no GPU."""

import ctypes

import pytest
import torch

from hi2_amd import _lib
from test_packed_abi import FAKE, packed, refused


def test_workspace_of_slots_that_index_no_rows():
    """Every index lies outside an empty batch: each slot becomes a row of NaN of its own, so
    the workspace holds the slots' rows, not the batch's."""
    size = _lib.lib().hi2x_packed_workspace_bytes
    for w in (packed(), packed(experts=4), packed(experts=4, per_expert=1)):
        ranges = int(w.experts > 1)
        some = size(ctypes.byref(w), 0, 2, 0, 40, 1, ranges)
        assert some >= 40 * 128 * 2 * 2 + 40 * 4
        assert size(ctypes.byref(w), 0, 2, 0, 0, 1, ranges) == 0


def test_tangents_are_seen_with_and_without_gradients():
    from torch.autograd import forward_ad

    x = torch.ones(3)
    _lib.refuse_tangents("this", x, None)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones(3))
        _lib.refuse_tangents("this", x, None)
        for ctx in (torch.no_grad(), torch.enable_grad()):
            with ctx, pytest.raises(RuntimeError, match="this has no forward-mode"):
                _lib.refuse_tangents("this", None, x, d)
    _lib.refuse_tangents("this", d)  # the level's end takes its tangents along


def test_workspace_of_the_weighted_sums_gradient():
    """One entry of 8 bytes for each row of y, where y has a gradient."""
    size = _lib.lib().hi2x_moe_combine_grad_workspace_bytes
    assert size(-1) == -1 and size(0) == 0 and size(100) >= 800

    def grad(dy, ws, n):
        return (FAKE, 0, FAKE, 0, 100, 16, FAKE, FAKE, 50, 2, FAKE, dy, ws, n, None)

    refused("hi2x_moe_combine_grad", "needed", *grad(FAKE, FAKE, 256))
    refused("hi2x_moe_combine_grad", "aligned", *grad(FAKE, FAKE + 8, 1024))
    refused("hi2x_moe_combine_grad", "bad shape", FAKE, 0, FAKE, 0, -1, 16, FAKE, FAKE, 50, 2,
            FAKE, FAKE, None, 0, None)
