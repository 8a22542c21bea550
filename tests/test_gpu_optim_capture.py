"""AdamW's memory and CUDA graphs: what a captured step holds stays valid, and a first step is not captured."""
import gc

import numpy as np
import pytest
import torch

from bit_reproducible_training_b200 import repro_optim
from test_gpu_optim import HYPER, bits, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("state_bits", [32, 8])
def test_a_captured_step_keeps_the_states_it_was_captured_with(state_bits):
    ps, gs = make([3000, 70], 50)
    qs, _ = make([3000, 70], 50)
    for p, q, g in zip(ps, qs, gs):
        p.grad, q.grad = g, g.clone()
    opt = repro_optim.AdamW(ps, state_bits=state_bits, capturable=True, **HYPER)
    twin = repro_optim.AdamW(qs, state_bits=state_bits, **HYPER)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    held = [t.data_ptr() for t in opt._tables[0]["kept"]] + [opt._tables[0]["device_step"].data_ptr()]
    names = opt._names()
    opt.adopt([tuple(torch.zeros_like(opt.state[p][k]) for k in names) for p in ps], step=0)
    gc.collect()
    torch.cuda.empty_cache()
    # nothing of the same sizes lands where the graph still writes
    fresh = [torch.zeros(n, dtype=d, device="cuda") for n in (3000, 70, 12, 1) for d in (torch.float32, torch.int8, torch.uint8, torch.int64) for _ in range(20)]
    assert not set(held) & {t.data_ptr() for t in fresh}
    graph.replay()
    torch.cuda.synchronize()
    assert not any(t.any() for t in fresh)
    twin.step()
    twin.step()
    for p, q in zip(ps, qs):
        assert np.array_equal(bits(p), bits(q))
    # the adopted states are the optimizer's: a step captured anew starts from them, with no eager one before it
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    graph.replay()
    torch.cuda.synchronize()
    assert opt.state_dict()["state"][0]["step"] == 1


@pytest.mark.parametrize("state_bits", [32, 8])
def test_a_first_step_is_not_captured(state_bits):
    """Its states and its counter would be made, and set to zero, inside the graph: at every replay."""
    ps, gs = make([256, 9], 51)
    for p, g in zip(ps, gs):
        p.grad = g
    opt = repro_optim.AdamW(ps, state_bits=state_bits, capturable=True, **HYPER)
    x = torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(RuntimeError, match="before it is captured"):
            opt.step()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(x, torch.ones(4, device="cuda")) and not opt.state
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    graph.replay()
    torch.cuda.synchronize()
    qs, _ = make([256, 9], 51)
    twin = repro_optim.AdamW(qs, state_bits=state_bits, **HYPER)
    for q, g in zip(qs, gs):
        q.grad = g
    twin.step()
    twin.step()
    for p, q in zip(ps, qs):
        assert np.array_equal(bits(p), bits(q))
