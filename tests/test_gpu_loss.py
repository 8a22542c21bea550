"""The linear cross entropy and its gradients against the definition in 64 bits.

Bounds.  u = 2^-24.  An S = 3 product rounds each operand to a multiple of its row's scale: by at most h = 2^-21 of the row's largest
magnitude (half a step of 2^e / 2^14 with 2^e < 2 max / 127).  A product of length L of rows with largest magnitudes a, b and
magnitude sums A1, B1 is therefore off by at most h (a B1 + b A1) + L h^2 a b, and by u of the result for its own rounding.
  logits:   e_z = h (x_max |w|_1 + w_max |x|_1) + D h^2 x_max w_max + u |z|, the largest over the words
  lse:      e_z, and 32-value sums, joins and exp / log: each part's sum is off by (32 + 8) u relative, each of at most 40 joins
            by 10 u, the logarithm by 4 u of itself and one addition: e_l = e_z + (440 + 8) u + 5 u |lse|
  p:        relative (e_z + e_l) + (|z - lse| + 6) u
  dX:       P W by the product bound over each piece with P's own error, plus the running sum's rounding per piece
  dW:       the same with the rows of P^T; the target's rows are added one after the other."""
import pytest
import torch

from bit_reproducible_training_b200 import layers, repro_loss

pytestmark = pytest.mark.gpu

U, H = 2.0 ** -24, 2.0 ** -21 * 1.0001
IGNORE = -100


def case(n, d, v, ignored=0.2, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + n + 1000 * d + v)
    x = torch.randn(n, d, device="cuda", generator=g).requires_grad_()
    w = (torch.randn(v, d, device="cuda", generator=g) * (scale / d ** 0.5)).requires_grad_()
    t = torch.randint(0, v, (n,), device="cuda", generator=g)
    t[torch.rand(n, device="cuda", generator=g) < ignored] = IGNORE
    return x, w, t


def expected(x, w, t, g):
    """Losses, gradients for row weights g (0 where ignored) and their bounds, in 64 bits."""
    x, w, g = x.detach().double(), w.detach().double(), g.double()
    n, d = x.shape
    keep = (t >= 0) & (t < w.shape[0])
    at = torch.where(keep, t, torch.zeros_like(t))
    z = x @ w.t()
    lse = torch.logsumexp(z, 1)
    nll = torch.where(keep, lse - z.gather(1, at[:, None])[:, 0], torch.zeros_like(lse))
    xm, wm = x.abs().amax(1), w.abs().amax(1)
    e_z = (H * (xm[:, None] * w.abs().sum(1)[None] + x.abs().sum(1)[:, None] * wm[None]) + d * H * H * xm[:, None] * wm[None]).amax(1) + U * z.abs().amax(1)
    e_l = e_z + 448 * U + 5 * U * lse.abs()
    e_nll = torch.where(keep, 2 * e_z + 448 * U + 5 * U * lse.abs() + U * nll.abs(), torch.zeros_like(nll))
    p = torch.exp(z - lse[:, None]) * g[:, None]
    e_p = p.abs() * (e_z[:, None] + e_l[:, None] + ((z - lse[:, None]).abs() + 8) * U)
    onehot = torch.zeros_like(p)
    onehot.scatter_(1, at[:, None], torch.where(keep, g, torch.zeros_like(g))[:, None])
    q = p - onehot
    # off-target entries go through the products; the target's coefficient has p's error and three roundings
    off = torch.where(onehot != 0, torch.zeros_like(p), p)
    e_off = torch.where(onehot != 0, torch.zeros_like(p), e_p)
    e_t = torch.where(onehot != 0, e_p + 4 * U * (p.abs() + onehot.abs()), torch.zeros_like(p))
    pieces = 64
    dx = q @ w
    e_dx = (e_off + e_t) @ w.abs() + H * (off.abs().amax(1)[:, None] * w.abs().sum(0)[None] + off.abs().sum(1)[:, None] * w.abs().amax(0)[None]) \
        + w.shape[0] * H * H * off.abs().amax(1)[:, None] * w.abs().amax(0)[None] + (pieces + 2) * U * (q.abs() @ w.abs())
    dw = q.t() @ x
    e_dw = (e_off + e_t).t() @ x.abs() + H * (off.abs().amax(0)[:, None] * x.abs().sum(0)[None] + off.abs().sum(0)[:, None] * x.abs().amax(0)[None]) \
        + n * H * H * off.abs().amax(0)[:, None] * x.abs().amax(0)[None] + (keep.sum() + 10) * U * (q.abs().t() @ x.abs())
    return nll, e_nll, dx, e_dx, dw, e_dw


def within(got, want, bound, what):
    assert torch.isfinite(got).all(), what
    over = float(((got.double() - want).abs() - bound).max())
    assert over <= 0.0, "%s is %.3g over its bound" % (what, over)


SHAPES = [(1, 1, 1), (1, 8, 50), (5, 3, 7), (31, 16, 64), (33, 100, 65), (128, 64, 1000), (129, 130, 4097), (300, 48, 20000), (64, 768, 33000), (1000, 40, 777),
          (2500, 96, 3001)]


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("n,d,v", SHAPES)
def test_loss_and_gradients(n, d, v, reduction):
    x, w, t = case(n, d, v)
    loss = layers.linear_cross_entropy(x, w, t, reduction=reduction)
    keep = (t >= 0).double()
    count = max(1.0, float(keep.sum()))
    g = torch.Generator(device="cuda").manual_seed(9)
    up = torch.randn(n, device="cuda", generator=g) if reduction == "none" else torch.tensor(1.7, device="cuda")
    row = up.double() * keep if reduction == "none" else keep * 1.7 / (count if reduction == "mean" else 1.0)
    nll, e_nll, dx, e_dx, dw, e_dw = expected(x, w, t, row)
    if reduction == "none":
        within(loss.detach(), nll, e_nll, "losses")
    else:
        many = count if reduction == "mean" else 1.0
        within(loss.detach(), nll.sum() / many, (e_nll.sum() + 2 * U * nll.abs().sum()) / many, "loss")
    got = torch.autograd.grad(loss, [x, w], up)
    extra = 0 if reduction == "none" else 2 * U            # 1.7 and the reciprocal count are rounded
    within(got[0], dx, e_dx + extra * dx.abs() + 3 * U * e_dx, "dX")
    within(got[1], dw, e_dw + extra * dw.abs() + 3 * U * e_dw, "dW")


@pytest.mark.parametrize("want", ["x", "w"])
def test_one_gradient_at_a_time(want):
    x, w, t = case(200, 64, 900)
    both = torch.autograd.grad(layers.linear_cross_entropy(x, w, t), [x, w])
    if want == "x":
        got, ref = torch.autograd.grad(layers.linear_cross_entropy(x, w.detach(), t), x)[0], both[0]
    else:
        got, ref = torch.autograd.grad(layers.linear_cross_entropy(x.detach(), w, t), w)[0], both[1]
    assert torch.equal(got, ref)


def test_gradients_against_differences():
    x, w, t = case(40, 24, 60)
    loss = layers.linear_cross_entropy(x, w, t)
    dx, dw = torch.autograd.grad(loss, [x, w])
    g = torch.Generator(device="cuda").manual_seed(2)
    a, b = (torch.randn(s.shape, device="cuda", generator=g, dtype=torch.float64) for s in (x, w))

    def f(s):
        return torch.nn.functional.cross_entropy((x.detach().double() + s * a) @ (w.detach().double() + s * b).t(), t)

    step = 1e-5
    slope = float((f(step) - f(-step)) / (2 * step))
    keep = (t >= 0).double()
    _, _, _, e_dx, _, e_dw = expected(x, w, t, keep / keep.sum())
    mine = float((dx.double() * a).sum() + (dw.double() * b).sum())
    bound = float((e_dx * a.abs()).sum() + (e_dw * b.abs()).sum()) + 3 * U * (float((dx * a).abs().sum()) + float((dw * b).abs().sum()))
    assert abs(slope - mine) <= bound + 1e-7 * abs(slope) + 1e-9


def test_every_row_ignored_and_no_rows():
    x, w, t = case(50, 32, 100)
    t.fill_(IGNORE)
    for reduction in ("mean", "sum"):
        loss = layers.linear_cross_entropy(x, w, t, reduction=reduction)
        dx, dw = torch.autograd.grad(loss, [x, w])
        assert float(loss) == 0.0 and not dx.any() and not dw.any()
    e = torch.zeros(0, 32, device="cuda", requires_grad=True)
    loss = layers.linear_cross_entropy(e, w, t[:0], reduction="mean")
    dx, dw = torch.autograd.grad(loss, [e, w])
    assert float(loss) == 0.0 and dx.shape == (0, 32) and not dw.any()
    assert layers.linear_cross_entropy(e, w, t[:0], reduction="none").shape == (0,)


def test_an_ignored_word_of_the_vocabulary():
    """ignore_index may be a word (padding): its rows do not count although the word is in every row's sum."""
    x, w, t = case(60, 16, 40, ignored=0.0)
    t[::3] = 5
    moved = torch.where(t == 5, torch.full_like(t, IGNORE), t)
    a, b = layers.linear_cross_entropy(x, w, t, ignore_index=5), layers.linear_cross_entropy(x, w, moved)
    assert torch.equal(a, b)
    for p, q in zip(torch.autograd.grad(a, [x, w]), torch.autograd.grad(b, [x, w])):
        assert torch.equal(p, q)


def test_targets_outside_the_vocabulary():
    x, w, t = case(30, 16, 40, ignored=0.0)
    bad = t.clone()
    bad[3], bad[7], bad[9], bad[11] = 40, -1, 2 ** 40, -2 ** 40
    losses = layers.linear_cross_entropy(x, w, bad, reduction="none")
    wrong = torch.zeros(30, dtype=torch.bool, device="cuda")
    wrong[[3, 7, 9, 11]] = True
    assert torch.isnan(losses[wrong]).all() and torch.isfinite(losses[~wrong]).all()
    assert torch.isnan(layers.linear_cross_entropy(x, w, bad))
    good = torch.where(wrong, torch.full_like(t, IGNORE), t)
    up = torch.ones(30, device="cuda")
    for p, q in zip(torch.autograd.grad(losses, [x, w], up), torch.autograd.grad(layers.linear_cross_entropy(x, w, good, reduction="none"), [x, w], up)):
        assert torch.equal(p, q)


@pytest.mark.parametrize("same", [True, False])
def test_frequent_targets(same):
    """Every row has the same target, or one of three: long runs of additions to one row of dW."""
    n, d, v = 3000, 200, 500
    x, w, t = case(n, d, v, ignored=0.1)
    t = torch.where(t < 0, t, torch.full_like(t, 7) if same else t % 3)
    got = torch.autograd.grad(layers.linear_cross_entropy(x, w, t, reduction="sum"), [x, w])
    _, _, dx, e_dx, dw, e_dw = expected(x, w, t, (t >= 0).double())
    within(got[0], dx, e_dx, "dX")
    within(got[1], dw, e_dw, "dW")


def test_peaked_rows():
    """Confident rows: the target's probability near 1 (its entry p - 1 is tiny) and near 0."""
    n, d, v = 64, 32, 300
    x, w, t = case(n, d, v, ignored=0.0, scale=12.0)
    with torch.no_grad():
        top = (x @ w.t()).argmax(1)
    t = torch.where(torch.arange(n, device="cuda") % 2 == 0, top, t)
    got = torch.autograd.grad(layers.linear_cross_entropy(x, w, t, reduction="sum"), [x, w])
    nll, e_nll, dx, e_dx, dw, e_dw = expected(x, w, t, torch.ones(n, device="cuda"))
    within(layers.linear_cross_entropy(x, w, t, reduction="none").detach(), nll, e_nll, "losses")
    within(got[0], dx, e_dx, "dX")
    within(got[1], dw, e_dw, "dW")


def test_shapes_strides_and_module():
    m = layers.LinearCrossEntropy(24, 90).cuda()
    x = torch.randn(24, 4, 10, device="cuda").permute(1, 2, 0).requires_grad_()
    t = torch.randint(0, 90, (10, 4), device="cuda").t()
    loss = m(x, t)
    loss.backward()
    flat = layers.linear_cross_entropy(x.detach().reshape(40, 24), m.weight.detach(), t.reshape(40))
    assert torch.equal(loss.detach(), flat) and m.weight.grad.shape == (90, 24) and x.grad.shape == x.shape
    wide = torch.empty(40 * 24 + 1, device="cuda")
    wide[1:] = x.detach().reshape(-1)
    assert torch.equal(layers.linear_cross_entropy(wide[1:].view(40, 24), m.weight.detach(), t.reshape(40)), flat)


def test_other_slice_counts():
    try:
        x, w, t = case(70, 50, 400)
        for s, tol in ((1, 0.2), (2, 2e-3)):
            layers.set_slices(s)
            loss = layers.linear_cross_entropy(x, w, t)
            dx, dw = torch.autograd.grad(loss, [x, w])
            want = torch.nn.functional.cross_entropy(x.detach().double() @ w.detach().double().t(), t)
            # an operand is off by 2^-7 (S = 1) or 2^-14 (S = 2) of its row's largest magnitude: see `expected`
            xm, wm = x.detach().abs().amax(1), w.detach().abs().amax(1)
            h = 2.0 ** -(7 * s)
            e = float((h * (xm[:, None] * w.detach().abs().sum(1)[None] + x.detach().abs().sum(1)[:, None] * wm[None])).max()) * (1 + h)
            assert abs(float(loss) - float(want)) <= 2 * e + 1e-4 and torch.isfinite(dx).all() and torch.isfinite(dw).all()
    finally:
        layers.set_slices(3)


def test_status_is_read_after_the_calls(monkeypatch):
    monkeypatch.setenv("RGB200_CHECK_STATUS", "1")
    x, w, t = case(100, 32, 20000)
    torch.autograd.grad(layers.linear_cross_entropy(x, w, t), [x, w])


def test_runs_repeat_on_streams_and_in_graphs_at_once():
    x, w, t = case(600, 96, 5000)
    x, w = x.detach(), w.detach()
    up = torch.tensor(1.0, device="cuda")

    def once():
        loss, stats = repro_loss.linear_cross_entropy(x, w, t)
        return (loss,) + repro_loss.linear_cross_entropy_backward(up, x, w, t, stats)

    want = once()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = once()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(once())
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for got in [other] + outs:
        for a, b in zip(got, want):
            assert torch.equal(a, b)
