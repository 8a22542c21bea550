"""The product with bias, activation and residual in its epilogue, and its gradients.

The product itself is pinned elsewhere (oracle, golden hashes), so the epilogue is checked against the library's own plain
product: c = gemm(...) has the same bits, and behind it come at most three FP32 operations and the activation.  Bounds, with
u = 2^-24: z = c + bias is rounded as torch rounds it, so equal bits.  Activations: exp and erf are within 2 ulp = 4 u of their
values.  silu: exp's argument is exact, 1 + exp adds u, the quotient u: 6 u of |y|, taken as 8.  gelu_tanh: the argument of exp
has four roundings and two rounded constants on positive terms of one sign, 6 u |t|, which moves y by at most |y| 6 u |t|;
with exp, sum and quotient 8 u more.  gelu: erf 4 u and its rounded argument (2 u |x| times erf's slope <= 2 / sqrt(pi), at most
0.97 u in all) and the sum, u, all of them relative to 1, times |z| / 2, and two products: (8 |z| / 2 + 3 |y|) u."""
import numpy as np
import pytest
import torch

import oracle
from bit_reproducible_training_b200 import fixtures as fx
from bit_reproducible_training_b200 import layers
from bit_reproducible_training_b200 import repro_gemm as rg

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
# Where exp(t) leaves the float range (t > 88.7) a sigmoid comes out as 0 and not as e^-t < 2^-127; that difference is multiplied by z in
# the activations and by the inner slope s in their derivatives.
TINY = 2.0 ** -127
ACTS = [None, "relu", "silu", "gelu", "gelu_tanh"]
# one tile and less, ragged tiles, several K blocks, one K block (K <= 128), narrow outputs, K ranges (few tiles, long K)
SHAPES = [(1, 1, 1), (1, 64, 64), (5, 3, 7), (128, 64, 128), (129, 65, 129), (200, 100, 515), (77, 1001, 300), (256, 40, 1024), (33, 768, 768), (16, 24, 8192),
          (130, 96, 5000), (64, 131, 4096)]


def value(z, act):
    """(act(z), its derivative) in 64 bits.  gelu_tanh as z sigmoid(2 t), which equals z/2 (1 + tanh t) without the cancellation
    that leaves even 64 bits without a correct digit below z = -6."""
    z = z.double().requires_grad_()
    F = torch.nn.functional
    y = {None: lambda t: t * 1.0, "relu": F.relu, "silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda t: t * torch.sigmoid(2 * (2 / np.pi) ** 0.5 * (t + 0.044715 * t ** 3))}[act](z)
    return y.detach(), torch.autograd.grad(y.sum(), z)[0]


def act_bound(z, y, act):
    z, y = z.double().abs(), y.abs()
    t = 1.5957691216057308 * z + 0.0713548162726009 * z ** 3
    return {None: 0 * y, "relu": 0 * y, "silu": 8 * U * y, "gelu": U * (4 * z + 3 * y), "gelu_tanh": U * y * (6 * t + 8)}[act] + TINY * (1 + z)


def slope_bound(z, act):
    """dsilu = p (1 + z (1 - p)): p within 6 u, at most eight more roundings of terms no larger than 1 + |z| p (1 - p) + p: 16 u (p + |z| p
    (1 - p)) plus 6 u p |z| p from 1 - p's error.  dgelu: Phi within 4 u absolute, the density's term |z| pdf within (6 + z^2) u (its exponent is
    rounded once).  dgelu_tanh: p moves by p (1 - p) 6 u |t|, then as silu with the inner slope s."""
    z = z.double()
    a = z.abs()
    if act in (None, "relu"):
        return 0 * a
    if act == "gelu":
        pdf = torch.exp(-0.5 * z * z) * 0.3989422804014327
        return U * (5 + a * pdf * (8 + z * z)) + 1e-38
    if act == "silu":
        p = torch.sigmoid(z)
        return U * (16 * (p + a * p * (1 - p)) + 6 * a * p * p) + TINY * (1 + a)
    t = 1.5957691216057308 * z + 0.0713548162726009 * z ** 3
    s = (1.5957691216057308 * z + 3 * 0.0713548162726009 * z ** 3).abs()
    p = torch.sigmoid(t)
    move = p * (1 - p) * 6 * t.abs() + 6 * p
    return U * (move * (1 + s) + 12 * p * (1 - p) * s + 2 * p) + TINY * (1 + s)


def operands(m, n, k, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + m + 1000 * n + k)

    def normal(*s, std=1.0):
        return torch.randn(*s, device="cuda", generator=g) * std

    return normal(m, k), normal(n, k, std=2.0 / k ** 0.5), normal(n), normal(m, n), normal(m, n)


@pytest.mark.parametrize("slices", [1, 2, 3])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_epilogue(m, n, k, act, slices):
    x, w, b, r, _ = operands(m, n, k)
    c = rg.gemm(x, w, m, n, k, False, True, slices)
    for bias in (None, b):
        z_want = c if bias is None else c + bias
        y64, _ = value(z_want, act)
        y, z = rg.gemm_epilogue(x, w, m, n, k, False, True, slices, bias, act, None, keep_pre=True)
        assert torch.equal(z, z_want)
        assert ((y.double() - y64).abs() <= act_bound(z_want, y64, act)).all()
        if act in (None, "relu"):
            assert torch.equal(y, y64.float())
        with_r = rg.gemm_epilogue(x, w, m, n, k, False, True, slices, bias, act, r)
        assert torch.equal(with_r, y + r)
        assert torch.equal(rg.gemm_epilogue(x, w, m, n, k, False, True, slices, bias, act), y)


@pytest.mark.parametrize("ta,tb", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("m,n,k", [(70, 72, 260), (64, 64, 4096)])
def test_other_storage_orders(m, n, k, ta, tb):
    x, w, b, r, _ = operands(m, n, k)
    A, B = (x.t().contiguous() if ta else x), (w if tb else w.t().contiguous())
    c = rg.gemm(A, B, m, n, k, ta, tb)
    assert torch.equal(rg.gemm_epilogue(A, B, m, n, k, ta, tb, bias=b, activation="relu", residual=r), torch.relu(c + b) + r)


def test_product_under_the_epilogue_is_the_oracles():
    m, n, k = 150, 90, 700
    g = fx.Rng(3)
    A, B = g.wide(m * k, -10, 10), g.normal(n * k)
    want = oracle.gemm(A, B, m, n, k, tb=True, S=3)
    got, pre = rg.gemm_epilogue(torch.from_numpy(A).cuda(), torch.from_numpy(B).cuda(), m, n, k, False, True, activation="relu", keep_pre=True)
    assert np.array_equal(pre.cpu().numpy().view(np.uint32), want.reshape(m, n).view(np.uint32))
    assert torch.equal(got, torch.relu(pre))


def test_in_place_residual_and_unaligned_rows():
    m, n, k = 140, 128, 300
    x, w, b, r, _ = operands(m, n, k)
    want = rg.gemm_epilogue(x, w, m, n, k, False, True, bias=b, activation="silu", residual=r)
    acc = r.clone()
    assert rg.gemm_epilogue(x, w, m, n, k, False, True, bias=b, activation="silu", residual=acc, out=acc) is acc
    assert torch.equal(acc, want)
    flat = torch.empty(m * n + 1, device="cuda")
    shifted = flat[1:].view(m, n)
    shifted.copy_(r)
    assert torch.equal(rg.gemm_epilogue(x, w, m, n, k, False, True, bias=b, activation="silu", residual=shifted, out=shifted), want)


def test_values_behind_the_output_stay():
    m, n, k = 100, 70, 256
    x, w, b, r, _ = operands(m, n, k)
    buf = torch.full((m * n + 512,), 7.0, device="cuda")
    rg.gemm_epilogue(x, w, m, n, k, False, True, bias=b, activation="gelu", out=buf[:m * n].view(m, n))
    assert (buf[m * n:] == 7.0).all()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n", [(1, 1), (3, 5), (31, 64), (33, 130), (100, 1001), (1000, 128), (257, 2304), (5000, 12)])
def test_activation_backward(m, n, act):
    _, _, _, z, dy = operands(m, n, 1)
    z = z * 3
    slope = value(z, act)[1]
    dz, db = rg.activation_backward(dy, z, m, n, act, True, True)
    want = dy.double() * slope
    assert ((dz.double() - want).abs() <= dy.double().abs() * slope_bound(z, act) + U * want.abs()).all()
    # a column's sum: at most m additions deep, each off by u of a partial sum
    assert ((db.double() - dz.double().sum(0)).abs() <= (m + 1) * U * dz.double().abs().sum(0)).all()
    only = rg.activation_backward(dy, z, m, n, act, False, True)
    assert only[0] is None and torch.equal(only[1], db)
    assert torch.equal(rg.activation_backward(dy, z, m, n, act)[0], dz)
    flat = torch.empty(m * n + 1, device="cuda")
    flat[1:] = dy.view(-1)
    moved = rg.activation_backward(flat[1:], z, m, n, act, True, True)
    assert torch.equal(moved[0], dz) and torch.equal(moved[1], db)


def test_extreme_pre_activations():
    z = torch.tensor([[0.0, -0.0, 1e-40, -1e-40, 30.0, -30.0, 90.0, -90.0, 300.0, -300.0, 1e6, -1e6, 1e10, -1e10]], device="cuda")
    one = torch.ones_like(z)
    for act in ACTS[1:]:
        y, slope = value(z, act)
        dz, _ = rg.activation_backward(one, z, 1, z.numel(), act)
        assert torch.isfinite(dz).all() and ((dz.double() - slope).abs() <= 1e-6 * (1 + slope.abs())).all(), act
        # the product of z with the identity's first row: z itself as a sum of one term
        got = torch.cat([rg.gemm_epilogue(torch.ones(1, 1, device="cuda"), v.view(1, 1), 1, 1, 1, False, True, activation=act, residual=None) for v in z[0]], 1)
        exact = rg.gemm(torch.ones(1, 1, device="cuda"), z.view(-1, 1), 1, z.numel(), 1, False, True)
        y = value(exact, act)[0]
        assert torch.isfinite(got).all() and ((got.double() - y).abs() <= act_bound(exact, y, act)).all(), act


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias,residual", [(True, False), (False, True), (True, True)])
def test_layer_gradients(act, bias, residual):
    """dX and dW are plain products of dZ, so they must have those bits; db and dZ are bounded above."""
    m, n, k = 96, 80, 200
    x, w, b, r, dy = operands(m, n, k)
    x, w = x.requires_grad_(), w.requires_grad_()
    b = b.requires_grad_() if bias else None
    r = r.requires_grad_() if residual else None
    y = layers.linear(x.view(4, 24, k), w, b, activation=act, residual=None if r is None else r.view(4, 24, n))
    assert y.shape == (4, 24, n)
    leaves = [t for t in (x, w, b, r) if t is not None]
    grads = dict(zip([id(t) for t in leaves], torch.autograd.grad(y, leaves, dy.view(4, 24, n))))
    z = rg.gemm(x.detach(), w.detach(), m, n, k, False, True)
    z = z if b is None else z + b.detach()
    dz, db = rg.activation_backward(dy, z, m, n, act, True, True)
    assert torch.equal(grads[id(x)], rg.gemm(dz, w.detach(), m, k, n))
    assert torch.equal(grads[id(w)], rg.gemm(dz, x.detach(), n, k, m, True, False))
    if bias:
        assert torch.equal(grads[id(b)], db)
    if residual:
        assert torch.equal(grads[id(r)], dy)


@pytest.mark.parametrize("slices", [1, 2, 3])
@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (3, 5, 7), (64, 64, 64), (100, 33, 48), (127, 130, 65), (128, 128, 200), (129, 260, 70), (300, 1001, 33), (1000, 64, 1500),
                                   (40, 3000, 50), (5000, 40, 60)])
def test_whole_backward_pass(m, n, k, act, slices):
    """dX and dW have the bits of the plain products on dZ, whichever of the three gradients are asked for."""
    x, w, _, z, dy = operands(m, n, k)
    dz, db = rg.activation_backward(dy, z, m, n, act, True, True)
    want = rg.gemm(dz, w, m, k, n, False, False, slices), rg.gemm(dz, x, n, k, m, True, False, slices), db
    for asked in ((True, True, True), (True, True, False), (True, False, True), (False, True, False), (False, False, True)):
        got = rg.linear_backward(dy, z, x, w, m, n, k, act, slices, *asked)
        for g, t, a in zip(got, want, asked):
            assert (g is None) != a and (not a or torch.equal(g, t)), asked
    flat = torch.empty(m * n + 1, device="cuda")
    flat[1:] = dy.view(-1)
    for g, t in zip(rg.linear_backward(flat[1:], z, x, w, m, n, k, act, slices, True, True, True), want):
        assert torch.equal(g, t)


def test_backward_of_wide_range_gradients():
    """Rows and columns of very different magnitudes, zeros, subnormals: the exponents of the one-pass split are the plain ones."""
    m, n, k = 150, 200, 40
    g = fx.Rng(7)
    dy = torch.from_numpy(g.wide(m * n, -100, 60)).cuda().view(m, n)
    dy[3] = 0
    dy[:, 5] = 0
    dy[7] *= 1e-30
    dy[:, 11] = 1e-42
    x, w, _, _, _ = operands(m, n, k)
    dx, dw, _ = rg.linear_backward(dy, None, x, w, m, n, k)
    assert torch.equal(dx, rg.gemm(dy, w, m, k, n)) and torch.equal(dw, rg.gemm(dy, x, n, k, m, True, False))


def test_gradients_against_differences():
    """The derivative along a direction by the 64-bit formula's central difference.  dX and dW are S = 3 products: each operand is off
    by at most 2^-21 of its row's largest magnitude, so a product of length L is off by at most L 2^-20 of the two largest magnitudes."""
    m, n, k = 40, 48, 56
    x, w, b, r, dy = operands(m, n, k)
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    y = layers.linear(x, w, b, activation="gelu_tanh", residual=r)
    grads = torch.autograd.grad(y, leaves, dy)
    way = [torch.randn_like(t, dtype=torch.float64) for t in leaves]

    def f(s):
        X, W, B, R = (t.detach().double() + s * d for t, d in zip(leaves, way))
        return ((torch.nn.functional.gelu(X @ W.t() + B, approximate="tanh") + R) * dy.double()).sum()

    step = 1e-5
    slope = float((f(step) - f(-step)) / (2 * step))
    mine = sum(float((g.double() * d).sum()) for g, d in zip(grads, way))
    dz = rg.activation_backward(dy, x.detach() @ w.detach().t() + b.detach(), m, n, "gelu_tanh")[0].abs()
    off_x = n * 2.0 ** -20 * float(dz.max() * w.detach().abs().max())
    off_w = m * 2.0 ** -20 * float(dz.max() * x.detach().abs().max())
    # Z is off by k 2^-20 of the largest magnitudes, which moves dZ by that times dY and the second derivative (below 1.2)
    off_z = 1.2 * k * 2.0 ** -20 * float(x.detach().abs().max() * w.detach().abs().max() * dy.abs().max()) + 40 * U * float(dy.abs().max())
    bound = float(way[0].abs().sum()) * (off_x + off_z * float(w.detach().abs().sum(0).max())) + \
        float(way[1].abs().sum()) * (off_w + off_z * float(x.detach().abs().sum(0).max())) + float(way[2].abs().sum()) * m * (off_z + U * float(dz.sum(0).max()))
    assert abs(slope - mine) <= bound + 1e-7 * abs(slope)


def test_module_and_empty_batches():
    layer = layers.FusedLinear(24, 40, activation="gelu").cuda()
    x = torch.randn(3, 7, 24, device="cuda")
    y = layer(x, residual=torch.ones(3, 7, 40, device="cuda"))
    y.sum().backward()
    assert layer.bias.grad is not None and layer.weight.grad is not None
    e = torch.zeros(0, 24, device="cuda", requires_grad=True)
    out = layer(e)
    assert out.shape == (0, 40)
    assert torch.equal(torch.autograd.grad(out.sum(), layer.weight)[0], torch.zeros_like(layer.weight))


def test_refusals():
    x, w, b, r, _ = operands(8, 16, 24)
    for bad in (dict(activation="tanh"), dict(residual=r[:4]), dict(bias=b[:3])):
        with pytest.raises(ValueError):
            layers.linear(x, w, **bad)
    with pytest.raises(ValueError):
        layers.linear(x, w.t(), b)
    with pytest.raises(TypeError):
        layers.linear(x, w, b.double())
    with pytest.raises(ValueError):
        rg.activation_backward(r, None, 8, 16, "gelu")
    with pytest.raises(ValueError):
        rg.gemm_epilogue(x, w, 8, 16, 24, False, True, out=torch.empty(8, 15, device="cuda"))


def test_status_is_read_after_the_calls(monkeypatch):
    monkeypatch.setenv("RGB200_CHECK_STATUS", "1")
    x, w, b, r, dy = operands(50, 60, 70)
    rg.gemm_epilogue(x, w, 50, 60, 70, False, True, bias=b)
    rg.linear_backward(dy, r, x, w, 50, 60, 70, "silu", want_db=True)


def test_two_graphs_at_once_and_other_streams():
    m, n, k = 300, 200, 400
    x, w, b, r, dy = operands(m, n, k)

    def once():
        y, z = rg.gemm_epilogue(x, w, m, n, k, False, True, bias=b, activation="gelu", residual=r, keep_pre=True)
        dz, db = rg.activation_backward(dy, z, m, n, "gelu", True, True)
        return (y, z, dz, db) + rg.linear_backward(dy, z, x, w, m, n, k, "gelu", 3, True, True, True)

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
    for _ in range(5):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for got in [other] + outs:
        for a, b_ in zip(got, want):
            assert torch.equal(a, b_)
