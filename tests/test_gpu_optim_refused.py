"""AdamW steps and dictionaries that are refused, whole: nothing is counted and nothing changes."""
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
