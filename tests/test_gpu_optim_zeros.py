"""Second moments that are written: their zeros."""
import pytest
import torch

from bit_reproducible_training_b200 import repro_optim

pytestmark = pytest.mark.gpu


def test_a_negative_zero_is_a_zero_second_moment():
    p = torch.nn.Parameter(torch.ones(512, device="cuda"))
    opt = repro_optim.AdamW([p], state_bits=8)
    m, v = torch.ones(512, device="cuda"), torch.ones(512, device="cuda")
    v[3] = -0.0
    v[256:] = -0.0
    opt.write_states([m], [v])
    got_m, got_v = torch.empty(512, device="cuda"), torch.empty(512, device="cuda")
    opt.read_states([got_m], [got_v])
    assert torch.equal(got_m, m) and torch.equal(got_v, v)
