"""What the packed products promise at the edges of their arguments, on the MI355X."""

import ctypes

import pytest
import torch

from test_gpu_packed import F, _experts

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
