"""The linear cross entropy's rows where precision is hard to come by.

Confident rows.  x holds a row's logits and W begins with the identity, so the logits are exact: entries are multiples of 2^-11 below 2^9, an
S = 3 operand keeps multiples of 2^(e - 14) with 2^e <= 2^3.  Then dX row i is the gradient of the logits of the first words: the target's
entry is minus the sum of the other words' probabilities, which is tiny.  u = 2^-24: that sum has 32-value parts, joins and exponentials
(440 u, see test_gpu_loss.py), the division and the row's weight (4 u): relative to itself, whatever the logits are.  The loss is
max - target + log(sum): log1p of that sum where the target is the largest, 460 u relative.  The other words' entries are off by
(448 + 5 |lse| + 2 |z - lse| + 8) u relative, as there, and pass a product (2^-21 of the largest entry)."""
import pytest
import torch

from bit_reproducible_training_b200 import layers
from test_gpu_loss import H, U

pytestmark = pytest.mark.gpu


def confident(level, n=48, d=64, gap=15.5, seed=0):
    """Logits with the target at `level` and the others about `gap` below it, on the grid above."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.randint(0, d, (n,), device="cuda", generator=g)
    z = level - gap - torch.randint(0, 2 ** 11, (n, d), device="cuda", generator=g).float() / 2 ** 11
    z.scatter_(1, t[:, None], torch.full((n, 1), float(level), device="cuda"))
    return z, t


@pytest.mark.parametrize("vocab", [64, 70000])
@pytest.mark.parametrize("level,gap", [(20.0, 15.5), (60.0, 15.5), (300.0, 15.5), (-40.0, 15.5), (20.0, 4.0), (60.0, 40.0), (300.0, 0.0)])
def test_gradients_of_confident_rows(level, gap, vocab):
    z, t = confident(level, gap=gap)
    n, d = z.shape
    if vocab > d and level < 0:
        pytest.skip("the words without a row in W would be the likely ones")
    w = torch.zeros(vocab, d, device="cuda")
    w[:d] = torch.eye(d, device="cuda")
    x = z.clone().requires_grad_()
    loss = layers.linear_cross_entropy(x, w, t, reduction="none")
    dx = torch.autograd.grad(loss, x, torch.ones_like(loss))[0].double()
    z64 = z.double() @ w.double().t()
    top = z64.amax(1, keepdim=True)
    e = torch.exp(z64 - top)
    at = t[:, None]
    hit = e.gather(1, at)
    others = e.scatter(1, at, 0.0)
    rest, total = others.sum(1, keepdim=True), others.sum(1, keepdim=True) + hit
    # 0 < rest: a quotient below 2^-126 would be subnormal, which no level here reaches
    want_t = -(rest / total)[:, 0]
    assert ((dx.gather(1, at)[:, 0] - want_t).abs() <= 450 * U * want_t.abs()).all()
    p = others / total
    lse = (top + torch.log(total))
    bound = p * ((448 + 5 * lse.abs() + 2 * (z64 - lse).abs() + 8) * U) + H * p.amax(1, keepdim=True) + U * p
    off = (dx.scatter(1, at, 0.0) - p[:, :d]).abs() - bound[:, :d]
    assert float(off.max()) <= 0.0
    # so a row's entries add up to zero
    row = dx.sum(1) + p[:, d:].sum(1)
    assert (row.abs() <= 450 * U * want_t.abs() + bound.sum(1)).all()
    # the loss: log1p(rest / hit) for a target that is its row's largest
    want = torch.log1p(rest / hit)[:, 0]
    assert ((loss.detach().double() - want).abs() <= 460 * U * want).all()
