"""Infinities and NaN in the operators around the products: a row of x or dY, or a row or column of W, that holds one shows NaN in every output
that it takes part in, and all others keep their bits.  Rows that do not count in the cross entropy take no part in anything."""
import pytest
import torch

from bit_reproducible_training_b200 import layers
from bit_reproducible_training_b200 import repro_gemm as rg

pytestmark = pytest.mark.gpu

BAD = [float("nan"), float("inf"), -float("inf")]
# short and long rows, aligned and not, K ranges, rows beyond the registers of the split (K > 16384), narrow outputs
SHAPES = [(5, 3, 7), (70, 40, 64), (65, 70, 100), (130, 33, 128), (100, 96, 132), (40, 64, 515), (70, 65, 1024), (33, 24, 5000), (64, 64, 4096), (9, 20, 20000),
          (200, 130, 30), (600, 600, 140)]


def operands(m, n, k, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + m + 1000 * n + k)
    return [torch.randn(*s, device="cuda", generator=g) for s in ((m, k), (n, k), (n,), (m, n), (m, n))]


def check(got, clean, bad_rows=(), bad_cols=(), what=""):
    """NaN in those rows and columns, the clean bits elsewhere."""
    mask = torch.zeros_like(got, dtype=torch.bool)
    mask[list(bad_rows)] = True
    mask[:, list(bad_cols)] = True
    assert torch.isnan(got[mask]).all(), what
    assert torch.equal(got[~mask], clean[~mask]), what


@pytest.mark.parametrize("bad", BAD, ids=str)
@pytest.mark.parametrize("slices", [1, 2, 3])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product_with_an_epilogue(m, n, k, slices, bad):
    x, w, b, r, _ = operands(m, n, k)
    rows, cols = [1, m - 1], [0, n // 2]
    xb, wb = x.clone(), w.clone()
    xb[rows[0], 0], xb[rows[1], k - 1] = bad, bad
    wb[cols[0], k // 2], wb[cols[1], k - 1] = bad, bad
    for ta, tb in ((False, True), (False, False), (True, False), (True, True)):
        def run(a, c):
            a, c = (a.t().contiguous() if ta else a), (c if tb else c.t().contiguous())
            return rg.gemm_epilogue(a, c, m, n, k, ta, tb, slices, b, "silu", r, keep_pre=True)
        for a, c, bad_rows, bad_cols in ((xb, w, rows, ()), (x, wb, (), cols), (xb, wb, rows, cols)):
            # a clean row's and column's scale is its own, so its bits are those of the product without the bad ones
            for got, clean in zip(run(a, c), run(x, w)):
                check(got, clean, bad_rows, bad_cols, (ta, tb))


@pytest.mark.parametrize("bad", BAD, ids=str)
@pytest.mark.parametrize("slices", [1, 2, 3])
@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_backward_pass(m, n, k, act, slices, bad):
    x, w, _, z, dy = operands(m, n, k)
    row, col, kk = m // 2, n - 1, k // 3
    for asked in ((True, True, True), (True, False, False), (False, True, False), (True, False, True)):
        def run(dy, z, x, w):
            return rg.linear_backward(dy, z, x, w, m, n, k, act, slices, *asked)
        clean = run(dy, z, x, w)
        d = dy.clone()
        d[row, col] = bad
        dx, dw, db = run(d, z, x, w)
        if dx is not None:
            check(dx, clean[0], [row], (), asked)
        if dw is not None:
            check(dw, clean[1], [col], (), asked)
        if db is not None:
            assert not torch.isfinite(db[col]) and torch.equal(db[:col], clean[2][:col])
        xb = x.clone()
        xb[row, kk] = bad
        dx, dw, _ = run(dy, z, xb, w)
        if dw is not None:
            check(dw, clean[1], (), [kk], asked)
        wb = w.clone()
        wb[col, kk] = bad
        dx, dw, _ = run(dy, z, x, wb)
        if dx is not None:
            check(dx, clean[0], (), [kk], asked)
        if dw is not None:
            assert torch.equal(dw, clean[1])
        if act:
            zb = z.clone()
            zb[row, col] = float("nan")
            dx, dw, _ = run(dy, zb, x, w)
            if dx is not None:
                check(dx, clean[0], [row], (), asked)
            if dw is not None:
                check(dw, clean[1], [col], (), asked)


@pytest.mark.parametrize("bad", BAD, ids=str)
@pytest.mark.parametrize("slices", [1, 2, 3])
@pytest.mark.parametrize("m,n,k", [(200, 132, 32), (300, 516, 64), (129, 1028, 5), (25000, 8, 12), (30001, 20, 4)])
def test_narrow_gradients_and_long_sums(m, n, k, slices, bad):
    """One gradient at a time: dX of at most 64 columns splits dZ inside its product's kernel, dW of many rows finds the columns' maxima in a kernel
    of its own."""
    x, w, _, _, dy = operands(m, n, k)
    row, col, kk = m - 1, n // 2, k - 1
    d, xb, wb = dy.clone(), x.clone(), w.clone()
    d[row, col], xb[row, kk], wb[col, kk] = bad, bad, bad

    def run(dy, x, w, dx):
        return rg.linear_backward(dy, None, x, w, m, n, k, None, slices, dx, not dx)[0 if dx else 1]

    dx, dw = run(dy, x, w, True), run(dy, x, w, False)
    check(run(d, x, w, True), dx, [row])
    check(run(dy, x, wb, True), dx, (), [kk])
    check(run(d, x, w, False), dw, [col])
    check(run(dy, xb, w, False), dw, (), [kk])
    check(run(d, xb, wb, True), dx, [row], [kk])
    check(run(d, xb, wb, False), dw, [col], [kk])


LOSS = [(40, 24, 60), (130, 100, 1000), (70, 515, 333), (64, 64, 20000), (40, 16, 70000), (300, 33, 5001)]


def loss_case(n, d, v):
    g = torch.Generator(device="cuda").manual_seed(n + d + v)
    x, w = torch.randn(n, d, device="cuda", generator=g), torch.randn(v, d, device="cuda", generator=g) / d ** 0.5
    t = torch.randint(0, v, (n,), device="cuda", generator=g)
    t[[1, n - 2]] = -100
    return x, w, t


def gradients(x, w, t, want=("x", "w"), up=None):
    x, w = x.clone().requires_grad_("x" in want), w.clone().requires_grad_("w" in want)
    loss = layers.linear_cross_entropy(x, w, t, reduction="none")
    up = torch.ones_like(loss) if up is None else up
    got = dict(zip(want, torch.autograd.grad(loss, [dict(x=x, w=w)[k] for k in want], up)))
    return loss.detach(), got.get("x"), got.get("w")


@pytest.mark.parametrize("bad", BAD, ids=str)
@pytest.mark.parametrize("want", [("x", "w"), ("x",), ("w",)], ids=str)
@pytest.mark.parametrize("n,d,v", LOSS)
def test_cross_entropy(n, d, v, want, bad):
    x, w, t = loss_case(n, d, v)
    clean = gradients(x, w, t, want)
    # a row that counts: its loss, its gradient, and all of dW
    xb = x.clone()
    xb[5, d - 1] = bad
    loss, dx, dw = gradients(xb, w, t, want)
    check(loss[:, None], clean[0][:, None], [5])
    assert dx is None or (torch.isnan(dx[5]).all() and torch.isfinite(dx[torch.arange(n) != 5]).all())
    assert dw is None or torch.isnan(dw).all()
    for reduction in ("mean", "sum"):
        assert torch.isnan(layers.linear_cross_entropy(xb, w, t, reduction=reduction))
    # a word: every row that counts
    wb = w.clone()
    wb[v - 1, 0] = bad
    loss, dx, dw = gradients(x, wb, t, want)
    counts = (t >= 0).nonzero()[:, 0].tolist()
    check(loss[:, None], torch.zeros_like(loss)[:, None], counts)
    if dx is not None:
        check(dx, torch.zeros_like(dx), counts)
    assert dw is None or torch.isnan(dw).all()
    # a gradient of the loss
    up = torch.ones(n, device="cuda")
    up[7] = bad
    loss, dx, dw = gradients(x, w, t, want, up)
    assert torch.equal(loss, clean[0])
    assert dx is None or not torch.isfinite(dx[7]).any()
    assert dx is None or torch.isfinite(dx[torch.arange(n) != 7]).all()
    assert dw is None or not torch.isfinite(dw).any()


@pytest.mark.parametrize("bad", BAD, ids=str)
@pytest.mark.parametrize("want", [("x", "w"), ("x",), ("w",)], ids=str)
@pytest.mark.parametrize("n,d,v", LOSS)
def test_rows_that_do_not_count(n, d, v, want, bad):
    """Padding may hold anything: with its values that are not finite at zero, the same bits."""
    x, w, t = loss_case(n, d, v)
    xb, x0 = x.clone(), x.clone()
    xb[1, ::3], x0[1, ::3] = bad, 0.0
    xb[n - 2, d - 1], x0[n - 2, d - 1] = bad, 0.0
    for got, clean in zip(gradients(xb, w, t, want), gradients(x0, w, t, want)):
        assert (got is None) == (clean is None)
        assert got is None or torch.equal(got, clean)
    for reduction in ("mean", "sum"):
        assert torch.equal(layers.linear_cross_entropy(xb, w, t, reduction=reduction), layers.linear_cross_entropy(x0, w, t, reduction=reduction))


def test_a_captured_step_meets_them_too():
    m, n, k = 70, 40, 100
    x, w, b, z, dy = operands(m, n, k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = rg.gemm_epilogue(x, w, m, n, k, False, True, bias=b)
        dx, dw, db = rg.linear_backward(dy, z, x, w, m, n, k, "gelu", 3, True, True, True)
    graph.replay()
    torch.cuda.synchronize()
    clean = [t.clone() for t in (y, dx, dw)]
    x[3, 4], dy[5, 6] = float("nan"), float("inf")
    graph.replay()
    torch.cuda.synchronize()
    check(y, clean[0], [3])
    check(dx, clean[1], [5])
    check(dw, clean[2], [6], [4])
    x[3, 4], dy[5, 6] = 1.0, 1.0
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.isfinite(t).all() for t in (y, dx, dw, db))
