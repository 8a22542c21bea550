"""AdamW steps and dictionaries that are refused, whole: nothing is counted and nothing changes."""
import copy

import numpy as np
import pytest
import torch

from bit_reproducible_training_b200 import repro_optim
from test_gpu_optim import HYPER, bits, make
from test_gpu_optim_groups import alone, fill

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("state_bits", [32, 8])
def test_a_refused_step_is_not_counted(state_bits):
    sizes = [300, 7]
    ps, gs = make(sizes, 33)
    fill(ps, gs)
    opt = repro_optim.AdamW(ps, state_bits=state_bits, **HYPER)
    opt.step()
    group = opt.param_groups[0]
    for bad in (-1.0, float("nan")):
        group["lr"] = bad
        with pytest.raises(RuntimeError):
            opt.step()
        ps[1].grad = None                            # and where the parameters' counters part
        with pytest.raises(RuntimeError):
            opt.step()
        ps[1].grad = gs[1]
    group["lr"] = HYPER["lr"]
    assert [int(opt.state[p]["step"]) for p in ps] == [1, 1]
    opt.step()
    for i, p in enumerate(ps):
        assert np.array_equal(bits(p), bits(alone(sizes, 33, i, 2, state_bits=state_bits)))


def test_loading_refuses_what_would_not_be_obeyed():
    ps, gs = make([40, 50], 34)
    fill(ps, gs)
    theirs = torch.optim.AdamW([torch.nn.Parameter(p.detach().clone()) for p in ps], lr=0.5)
    for p, g in zip(theirs.param_groups[0]["params"], gs):
        p.grad = g.clone()
    theirs.step()
    opt = repro_optim.AdamW(ps, **HYPER)
    opt.step()
    before = copy.deepcopy(opt.state_dict())

    def same():
        now = opt.state_dict()
        assert now["param_groups"] == before["param_groups"]
        for i, s in before["state"].items():
            assert now["state"][i]["step"] == s["step"] and all(torch.equal(now["state"][i][k], s[k]) for k in ("exp_avg", "exp_avg_sq"))

    good = theirs.state_dict()
    for change in (dict(maximize=True), dict(amsgrad=True), dict(differentiable=True), dict(decoupled_weight_decay=False), dict(lr=-1.0), dict(betas=(0.9, 1.0)),
                   dict(eps=float("nan"))):
        bad = copy.deepcopy(good)
        bad["param_groups"][0].update(change)
        with pytest.raises(ValueError):
            opt.load_state_dict(bad)
        same()
    bad = copy.deepcopy(good)
    del bad["state"][1]["exp_avg_sq"]
    with pytest.raises((ValueError, KeyError)):
        opt.load_state_dict(bad)
    same()
    opt.load_state_dict(good)                        # torch's own dictionary: its moments, its step, and none of its switches
    group = opt.param_groups[0]
    assert group["lr"] == 0.5 and not {"maximize", "amsgrad", "foreach", "fused"} & set(group)
    now = opt.state_dict()["state"]
    assert now[0]["step"] == 1 and torch.equal(now[1]["exp_avg"], theirs.state[theirs.param_groups[0]["params"][1]]["exp_avg"])


def test_unequal_counts_are_refused_before_anything_changes():
    ps, gs = make([40, 50], 35)
    fill(ps, gs)
    opt = repro_optim.AdamW(ps, capturable=True, **HYPER)
    opt.step()
    before = copy.deepcopy(opt.state_dict())
    bad = copy.deepcopy(before)
    bad["state"][1]["step"] = 9
    bad["state"][0]["exp_avg"].fill_(7.0)
    bad["param_groups"][0]["lr"] = 0.25
    with pytest.raises(ValueError, match="same number of steps"):
        opt.load_state_dict(bad)
    now = opt.state_dict()
    assert now["param_groups"] == before["param_groups"] and torch.equal(now["state"][0]["exp_avg"], before["state"][0]["exp_avg"])
    assert now["state"][1]["step"] == 1
    fresh = repro_optim.AdamW(make([40, 50], 36)[0], capturable=True, **HYPER)
    with pytest.raises(ValueError, match="same number of steps"):
        fresh.load_state_dict(bad)
