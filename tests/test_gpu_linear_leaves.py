"""layers.linear differentiated in any subset of its tensors: each gradient has the bits it has when all are asked for."""
import itertools

import pytest
import torch

from bit_reproducible_training_b200 import layers
from bit_reproducible_training_b200 import repro_gemm as rg

pytestmark = pytest.mark.gpu

NAMES = ("x", "weight", "bias", "residual")


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu", "gelu_tanh"])
def test_any_subset_of_leaves(act):
    m, n, k = 37, 24, 40
    g = torch.Generator(device="cuda").manual_seed(1)
    data = dict(x=torch.randn(m, k, device="cuda", generator=g), weight=torch.randn(n, k, device="cuda", generator=g),
                bias=torch.randn(n, device="cuda", generator=g), residual=torch.randn(m, n, device="cuda", generator=g))
    dy = torch.randn(m, n, device="cuda", generator=g)

    def grads(names):
        t = {k: v.clone().requires_grad_(k in names) for k, v in data.items()}
        y = layers.linear(t["x"], t["weight"], t["bias"], activation=act, residual=t["residual"])
        return dict(zip(names, torch.autograd.grad(y, [t[k] for k in names], dy)))

    want = grads(NAMES)
    assert torch.equal(want["residual"], dy)
    for size in (1, 2, 3):
        for names in itertools.combinations(NAMES, size):
            for name, got in grads(names).items():
                assert torch.equal(got, want[name]), (names, name)


def test_nothing_is_asked_for():
    z = torch.randn(4, 6, device="cuda")
    x, w = torch.randn(4, 5, device="cuda"), torch.randn(6, 5, device="cuda")
    assert rg.linear_backward(z, None, x, w, 4, 6, 5, "gelu", 3, False, False, False) == (None, None, None)
    with pytest.raises(ValueError):
        rg.linear_backward(z, None, x, w, 4, 6, 5, "gelu")
