"""AdamW beside a user's own changes to its groups."""
import numpy as np
import pytest
import torch

from bit_reproducible_training_b200 import repro_optim
from test_gpu_optim import HYPER, bits, host, make

pytestmark = pytest.mark.gpu


def fill(ps, gs):
    for p, g in zip(ps, gs):
        p.grad = g


def alone(sizes, seed, i, steps, **kw):
    """What parameter i comes to by itself."""
    ps, gs = make(sizes, seed)
    opt = repro_optim.AdamW([ps[i]], **{**HYPER, **kw})
    ps[i].grad = gs[i]
    for _ in range(steps):
        opt.step()
    return ps[i]


@pytest.mark.parametrize("state_bits", [32, 8])
def test_exchanged_and_reordered_parameters_keep_their_own_states(state_bits):
    sizes = [300, 300, 300]
    ps, gs = make(sizes, 30)
    fill(ps, gs)
    opt = repro_optim.AdamW(ps, state_bits=state_bits, **HYPER)
    opt.step()
    group = opt.param_groups[0]["params"]
    group.reverse()
    opt.step()
    for i, p in enumerate(ps):
        assert np.array_equal(bits(p), bits(alone(sizes, 30, i, 2, state_bits=state_bits))) and int(opt.state[p]["step"]) == 2
    fresh = torch.nn.Parameter(ps[1].detach().clone())
    start = host([fresh])[0]
    fresh.grad = gs[1]
    old = ps[1].detach().clone()
    group[1] = fresh                                 # another parameter of the same size: its first step
    opt.step()
    other = torch.nn.Parameter(torch.from_numpy(start).cuda())
    other.grad = gs[1]
    repro_optim.AdamW([other], state_bits=state_bits, **HYPER).step()
    assert np.array_equal(bits(fresh), bits(other)) and torch.equal(ps[1], old)
    assert np.array_equal(bits(ps[0]), bits(alone(sizes, 30, 0, 3, state_bits=state_bits)))
    assert int(opt.state[fresh]["step"]) == 1 and int(opt.state[ps[0]]["step"]) == 3


@pytest.mark.parametrize("capturable", [False, True])
def test_a_removed_group_and_one_that_grows(capturable):
    sizes = [200, 200, 200]
    ps, gs = make(sizes, 31)
    fill(ps, gs)
    opt = repro_optim.AdamW([dict(params=[ps[0]]), dict(params=[ps[1]])], capturable=capturable, **HYPER)
    opt.step()
    opt.step()
    del opt.param_groups[0]
    opt.step()
    assert np.array_equal(bits(ps[1]), bits(alone(sizes, 31, 1, 3))) and np.array_equal(bits(ps[0]), bits(alone(sizes, 31, 0, 2)))
    saved = opt.state_dict()
    assert len(saved["state"]) == 1 and saved["state"][0]["step"] == 3
    opt.add_param_group(dict(params=[ps[2]]))
    opt.step()
    assert np.array_equal(bits(ps[2]), bits(alone(sizes, 31, 2, 1))) and np.array_equal(bits(ps[1]), bits(alone(sizes, 31, 1, 4)))
    late = torch.nn.Parameter(torch.ones(8, device="cuda"))
    late.grad = torch.ones(8, device="cuda")
    opt.param_groups[0]["params"].append(late)
    if capturable:                                   # one counter for a group: refused, and the counts are the true ones
        with pytest.raises(ValueError, match="same number of steps"):
            opt.step()
        assert int(opt.state[ps[1]]["step"]) == 4
        opt.param_groups[0]["params"].pop()
        opt.step()
        assert np.array_equal(bits(ps[1]), bits(alone(sizes, 31, 1, 5)))
    else:
        opt.step()
        assert int(opt.state[late]["step"]) == 1 and np.array_equal(bits(ps[1]), bits(alone(sizes, 31, 1, 5)))


def test_a_captured_step_survives_changes_elsewhere():
    """Another group comes and goes: the captured step of this one goes on counting on the same words."""
    sizes = [500, 90]
    ps, gs = make(sizes, 32)
    fill(ps, gs)
    opt = repro_optim.AdamW([ps[0]], capturable=True, **HYPER)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    graph.replay()
    opt.add_param_group(dict(params=[ps[1]]))
    opt.step()
    graph.replay()
    torch.cuda.synchronize()
    assert np.array_equal(bits(ps[0]), bits(alone(sizes, 32, 0, 4))) and opt.state_dict()["state"][0]["step"] == 4
    assert np.array_equal(bits(ps[1]), bits(alone(sizes, 32, 1, 1)))
