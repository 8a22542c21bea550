"""The linear cross entropy and the fused linear layer over more rows than an INT64 can sum the products of: dW takes them in ranges."""
import pytest
import torch

from bit_reproducible_training_b200 import layers
from bit_reproducible_training_b200 import repro_gemm as rg
from test_gpu_loss import U, case, expected, within

pytestmark = pytest.mark.gpu


def test_cross_entropy():
    n, d, v = 1_100_000, 8, 40
    x, w, t = case(n, d, v)
    loss = layers.linear_cross_entropy(x, w, t, reduction="sum")
    dx, dw = torch.autograd.grad(loss, [x, w])
    nll, e_nll, want_dx, e_dx, want_dw, e_dw = expected(x, w, t, (t >= 0).double())
    within(loss.detach(), nll.sum(), e_nll.sum() + 2 * U * nll.sum(), "loss")
    within(dx, want_dx, e_dx, "dX")
    within(dw, want_dw, e_dw, "dW")
    # each gradient alone, and the rows of the two halves on their own
    assert torch.equal(torch.autograd.grad(layers.linear_cross_entropy(x, w.detach(), t, reduction="sum"), x)[0], dx)
    assert torch.equal(torch.autograd.grad(layers.linear_cross_entropy(x.detach(), w, t, reduction="sum"), w)[0], dw)
    half = torch.autograd.grad(layers.linear_cross_entropy(x[:n // 2], w, t[:n // 2], reduction="sum"), w)[0].double() + \
        torch.autograd.grad(layers.linear_cross_entropy(x[n // 2:], w, t[n // 2:], reduction="sum"), w)[0].double()
    assert ((half - dw.double()).abs() <= 2 * e_dw).all()


@pytest.mark.parametrize("act", [None, "relu"])
@pytest.mark.parametrize("slices", [2, 3])
def test_linear(act, slices):
    """Small integers: every product is exact, every sum below 2^24, so the gradients are."""
    m, n, k = 1_100_000, 12, 20
    g = torch.Generator(device="cuda").manual_seed(3)
    x, w, dy = (torch.randint(-2, 3, s, device="cuda", generator=g).float() for s in ((m, k), (n, k), (m, n)))
    x, w = x.requires_grad_(), w.requires_grad_()
    b = torch.zeros(n, device="cuda", requires_grad=True)
    try:
        layers.set_slices(slices)
        y = layers.linear(x, w, b, activation=act)
        dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
        alone = torch.autograd.grad(layers.linear(x.detach(), w, b, activation=act), w, dy)[0]
    finally:
        layers.set_slices(3)
    z = x.detach().double() @ w.detach().double().t()
    dz = dy.double() * ((z > 0) if act else 1)
    assert torch.equal(y.detach().double(), z.clamp(min=0) if act else z)
    assert torch.equal(dx.double(), dz @ w.detach().double())
    assert torch.equal(dw.double(), dz.t() @ x.detach().double()) and torch.equal(alone, dw)
    assert torch.equal(db.double(), dz.sum(0))


@pytest.mark.parametrize("m", [2 ** 20, 2 ** 20 + 1, 1_056_751])
def test_as_many_rows_as_one_product_takes(m):
    """Up to there dW has the bits of the plain product."""
    n, k = 5, 9
    g = torch.Generator(device="cuda").manual_seed(m)
    x, w, dy = (torch.randn(s, device="cuda", generator=g) for s in ((m, k), (n, k), (m, n)))
    dx, dw, _ = rg.linear_backward(dy, None, x, w, m, n, k)
    assert torch.equal(dw, rg.gemm(dy, x, n, k, m, True, False)) and torch.equal(dx, rg.gemm(dy, w, m, k, n))
    assert rg.make_plan(n, k, 1_056_751)[0] == 0 and rg.make_plan(n, k, 1_056_752)[0] == 1
