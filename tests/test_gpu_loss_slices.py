"""The linear cross entropy's gradients at each slice count, with the rounding of its operands restated instead of bounded: a bound of 2^-7 of a
row's largest entry (S = 1) would pass almost anything."""
import pytest
import torch

from bit_reproducible_training_b200 import layers
from test_gpu_loss import IGNORE, U, within

pytestmark = pytest.mark.gpu


def quantized(p, e_p, slices):
    """Rows of p as an operand of `slices` digits holds them, p being known to e_p relative: values, how far an entry may be from them (a step
    where the border between two multiples of the row's scale lies within e_p), and the rows whose scale itself is certain."""
    top = p.abs().amax(1, keepdim=True)
    e = torch.ceil(torch.log2(top / 127))
    sure = (torch.ceil(torch.log2(top * (1 + 2 * e_p) / 127)) == e) & (torch.ceil(torch.log2(top * (1 - 2 * e_p) / 127)) == e)
    step = torch.exp2(e - 7 * (slices - 1))
    q = p / step
    near = ((q - torch.floor(q)) - 0.5).abs() <= q.abs() * e_p
    return torch.round(q) * step, near * step, sure[:, 0]


@pytest.mark.parametrize("slices", [1, 2, 3])
@pytest.mark.parametrize("n,d,v", [(70, 50, 400), (129, 130, 4097), (33, 100, 65), (1000, 40, 777), (301, 48, 20000), (1100, 24, 40000)])
def test_gradients_at_every_slice_count(n, d, v, slices):
    """x and W hold small integers times a power of two, which an operand of any slice count and scale holds exactly: then the products round
    nothing but P, by its rows for dX (one piece) and by its columns for dW, and that rounding is restated here."""
    g = torch.Generator(device="cuda").manual_seed(n + d + v)
    x = torch.randint(-2, 3, (n, d), device="cuda", generator=g).float().requires_grad_()
    w = (torch.randint(-2, 3, (v, d), device="cuda", generator=g).float() / 8).requires_grad_()
    t = torch.randint(0, v, (n,), device="cuda", generator=g)
    t[::7] = IGNORE
    try:
        layers.set_slices(slices)
        loss = layers.linear_cross_entropy(x, w, t, reduction="sum")
        dx, dw = torch.autograd.grad(loss, [x, w])
    finally:
        layers.set_slices(3)
    X, W = x.detach().double(), w.detach().double()
    keep = t >= 0
    at = torch.where(keep, t, torch.zeros_like(t))[:, None]
    z = X @ W.t()
    lse = torch.logsumexp(z, 1, keepdim=True)
    nll = torch.where(keep, (lse - z.gather(1, at))[:, 0], torch.zeros_like(lse[:, 0]))
    within(loss.detach(), nll.sum(), ((keep.sum() * 450 + 5 * lse.abs().sum()) * U + 2 * U * nll.sum()), "loss")
    p = torch.exp(z - lse) * keep[:, None]
    e_p = float((448 + 5 * lse.abs().max() + 2 * (z - lse).abs().max() + 8) * U)
    off = p.scatter(1, at, 0.0)
    c = (p.gather(1, at)[:, 0] - 1) * keep              # the targets' coefficients
    onehot = torch.zeros_like(p).scatter_(1, at, c[:, None])
    # dW: a column of P is a row of its operand; the sums are exact, then one rounding and one per row of a target
    q, may, sure = quantized(off.t(), e_p, slices)
    want = q @ X + onehot.t() @ X
    bound = may @ X.abs() + (e_p + (n + 4) * U) * (onehot.t().abs() @ X.abs()) + 4 * U * (q.abs() @ X.abs())
    assert sure.float().mean() > 0.95 and not may.all()
    within(dw[sure], want[sure], bound[sure], "dW")
    if v < 20000:                                       # one piece: a row's scale is that of all its words
        q, may, sure = quantized(torch.where(keep[:, None], off, torch.ones_like(off)), e_p, slices)
        q, may = q * keep[:, None], may * keep[:, None]
        want = q @ W + onehot @ W
        bound = may @ W.abs() + (e_p + 4 * U) * (onehot.abs() @ W.abs()) + 4 * U * (q.abs() @ W.abs())
        assert sure.float().mean() > 0.95
        within(dx[sure], want[sure], bound[sure], "dX")
    else:
        h = 2.0 ** (-7 * slices) * 1.0001
        within(dx, (off + onehot) @ W, h * off.amax(1)[:, None] * W.abs().sum(0)[None] + (e_p + 64 * U) * ((off + onehot.abs()) @ W.abs()), "dX")
