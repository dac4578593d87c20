"""Options of groups that would change the step and are not there."""

import pytest
import torch

from hi2_amd.optim import AdamW

pytestmark = pytest.mark.gpu


def parameter():
    p = torch.nn.Parameter(torch.ones(10).cuda())
    p.grad = torch.ones_like(p)
    return p


VARIANTS = [("amsgrad", True), ("maximize", True), ("differentiable", True),
            ("decoupled_weight_decay", False)]


@pytest.mark.parametrize("name,value", VARIANTS)
def test_variants_are_refused(dev, name, value):
    with pytest.raises(ValueError, match=name):
        AdamW([dict(params=[parameter()]), {"params": [parameter()], name: value}])
    p = parameter()
    opt = AdamW([p])
    opt.param_groups[0][name] = value  # (between steps)
    with pytest.raises(ValueError, match=name):
        opt.step()
    assert bool((p == 1).all()) and not opt.moments()[0].any()
    opt.param_groups[0][name] = not value
    opt.step()
    state = opt.state_dict()
    state["param_groups"][0][name] = value
    other = AdamW([parameter()])
    with pytest.raises(ValueError, match=name):
        other.load_state_dict(state)
    assert not other.moments()[0].any()


def test_what_else_a_group_holds_stays(dev):
    p = parameter()
    opt = AdamW([{"params": [p], "name": "latents", "foreach": None, "fused": True, "amsgrad": False,
                  "maximize": False}], lr=0.5)
    torch.optim.lr_scheduler.OneCycleLR(opt, max_lr=1.0, total_steps=4)
    opt.step()
    assert opt.param_groups[0]["name"] == "latents" and "max_momentum" in opt.param_groups[0]
    other = AdamW([parameter()])
    other.load_state_dict(opt.state_dict())
    assert other.param_groups[0]["name"] == "latents"
