"""Forward-mode derivatives are refused, by the layers that have none: a tangent must not vanish without a word."""
import pytest
import torch
from torch.autograd import forward_ad

from bit_reproducible_training_b200 import layers

X, W, T = torch.zeros(6, 8), torch.zeros(10, 8), torch.zeros(6, dtype=torch.int64)


def calls(x, w):
    yield lambda: layers.linear(x, w)
    yield lambda: layers.linear(X, W, residual=x[:, :1].expand(6, 10))
    yield lambda: layers.linear(X, W, torch.zeros(10) + w[0, 0])
    yield lambda: layers.block_norm(x, weight=torch.ones(8))
    yield lambda: layers.block_norm(X, X, weight=w[0])
    yield lambda: layers.linear_cross_entropy(x, w, T)
    yield lambda: layers.linear_cross_entropy(X, w, T)


@pytest.mark.parametrize("grad", [True, False])
def test_dual_tensors_are_refused(grad):
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        x, w = forward_ad.make_dual(X, torch.ones_like(X)), forward_ad.make_dual(W, torch.ones_like(W))
        for call in calls(x, w):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_other_tensors_pass_under_a_dual_level():
    """Nothing here is dual: the calls go on to their ordinary checks."""
    with forward_ad.dual_level():
        for call in (lambda: layers.linear(X, W), lambda: layers.block_norm(X, weight=torch.ones(8)), lambda: layers.linear_cross_entropy(X, W, T)):
            with pytest.raises(RuntimeError, match="no CPU path"):
                call()


def test_function_transforms_are_refused_too():
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda x: layers.linear(x, W), (X,), (X,))
