"""AdamW's memory and CUDA graphs: a first step is not captured."""
import numpy as np
import pytest
import torch

from bit_reproducible_training_b200 import repro_optim
from test_gpu_optim import HYPER, bits, make

pytestmark = pytest.mark.gpu


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
