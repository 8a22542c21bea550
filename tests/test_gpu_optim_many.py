"""AdamW over more tensors than one launch takes."""
import numpy as np
import pytest
import torch

from bit_reproducible_training_b200 import repro_optim
from optim_restated import adamw, decode, encode
from test_gpu_optim import HYPER, bits, host, make
from test_gpu_optim_groups import fill

pytestmark = pytest.mark.gpu


MANY = [("many", [64 + i % 5 for i in range(170)]), ("several launches", [33 + 7 * (i % 3) for i in range(1000)]), ("empty ones among them", [0, 9] * 460),
        ("long chunks", [2_600_000, 700_001, 3])]


@pytest.mark.parametrize("state_bits", [32, 8])
@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("name,sizes", MANY, ids=[m[0] for m in MANY])
def test_many_tensors_have_the_defined_bits(name, sizes, capturable, state_bits):
    """More than 160 tensors (the largest table), more than 448 (several launches), and chunks of more than 1024 values."""
    ps, gs = make(sizes, 40)
    opt = repro_optim.AdamW(ps, state_bits=state_bits, capturable=capturable, **HYPER)
    fill(ps, gs)
    flat, g = np.concatenate(host(ps)), np.concatenate(host(gs))
    cuts = np.cumsum([0] + sizes)
    m, v = np.zeros_like(flat), np.zeros_like(flat)
    for n in range(1, 4):
        flat, m, v = adamw(flat, g, m, v, HYPER["lr"], *HYPER["betas"], HYPER["eps"], HYPER["weight_decay"], n)
        if state_bits == 8:
            for a, b in zip(cuts[:-1], cuts[1:]):
                if b > a:
                    m[a:b], v[a:b] = decode(*encode(m[a:b], v[a:b]))
    opt.step()
    if capturable:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opt.step()
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
    else:
        opt.step()
        opt.step()
    assert np.array_equal(bits(np.concatenate(host(ps))), bits(flat))
    ms, vs = ([torch.empty(n, device="cuda") for n in sizes] for _ in range(2))
    opt.read_states(ms, vs)
    assert np.array_equal(bits(np.concatenate(host(ms))), bits(m)) and np.array_equal(bits(np.concatenate(host(vs))), bits(v))
    assert opt.state_dict()["state"][0]["step"] == 3
