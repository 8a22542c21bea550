"""Activations and their derivatives over the whole range of finite pre-activations, whose squares and cubes leave it: beyond 100 every activation is
z or 0 and every derivative 1 or 0 to the last bit."""
import pytest
import torch

from bit_reproducible_training_b200 import layers
from bit_reproducible_training_b200 import repro_gemm as rg

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "gelu_tanh"])
def test_large_pre_activations(act):
    z = torch.tensor([1e2, 1e10, 1e12, 1.1e13, 1.3e13, 1e15, 1e19, 2e19, 1e30, 3.4e38], device="cuda")
    z = torch.cat([z, -z])[None]
    dz, db = rg.activation_backward(torch.full_like(z, 3.0), z, 1, z.numel(), act, True, True)
    want = torch.where(z > 0, 3.0, 0.0)
    assert torch.equal(dz, want) and torch.equal(db, want[0])
    one = torch.ones(1, 1, device="cuda")
    # one column at a time: the product of a single value with 1 is that value to 21 bits
    for v in z[0]:
        pre = rg.gemm(one, v.view(1, 1), 1, 1, 1)
        x = v.view(1, 1).clone().requires_grad_()
        y = layers.linear(x, one, activation=act)
        assert torch.equal(y.detach(), pre.clamp(min=0.0)), float(v)
        assert torch.equal(torch.autograd.grad(y, x)[0], torch.ones_like(pre) if v > 0 else torch.zeros_like(pre)), float(v)
