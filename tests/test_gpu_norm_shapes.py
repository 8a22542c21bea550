"""Gradients of block_norm have the shapes of the tensors they belong to, whatever dimensions of one those carry."""
import pytest
import torch

from bit_reproducible_training_b200 import layers

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(48,), (1, 48), (1, 1, 48)], ids=str)
def test_shapes_of_the_gradients(shape):
    g = torch.Generator(device="cuda").manual_seed(1)
    x, y, dr, dh = (torch.randn(2, 5, 48, device="cuda", generator=g) for _ in range(4))
    vectors = [torch.randn(48, device="cuda", generator=g) for _ in range(3)]

    def grads(of):
        w, b, pw = (v.clone().view(of).requires_grad_() for v in vectors)
        gate = vectors[0].clone().view(1, 48).requires_grad_()
        r, h = layers.block_norm(x, y, weight=w, bias=b, post_weight=pw, gate=gate, kind="layer")
        return torch.autograd.grad([r, h], [w, b, pw, gate], [dr, dh])

    for got, want, of in zip(grads(shape), grads((48,)), (shape, shape, shape, (1, 48))):
        assert got.shape == of and torch.equal(got.view(-1), want.view(-1))
