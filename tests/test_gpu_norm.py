"""block_norm and its gradients against the formula in 64 bits; the bounds are derived in norm_restated.py."""
import pytest
import torch

import norm_restated as ref
from bit_reproducible_training_b200 import layers, repro_norm

pytestmark = pytest.mark.gpu

MODES = ["plain", "residual", "gate", "post", "post_gate", "post_groups", "groups"]
SHAPES = [(1, 1), (5, 3), (3, 32), (2, 33), (7, 100), (4, 255), (9, 256), (6, 257), (11, 768), (4, 1001), (3, 1024), (2, 2047), (3, 2304), (2, 4096),
          (2, 5000), (1, 8191), (2, 8192), (300, 64), (1000, 20)]


def case(rows, dim, mode, kind, seed=0, bias=True):
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 10007 + dim)

    def n(*s, std=1.0, mean=0.0):
        return (torch.randn(*s, device="cuda", generator=g) * std + mean).requires_grad_()

    t = dict(x=n(rows, dim, mean=0.3), y=None, weight=n(dim, std=0.2, mean=1.0), bias=n(dim, std=0.3) if bias else None, post_weight=None, gate=None)
    if mode != "plain":
        t["y"] = n(rows, dim, std=0.5, mean=0.1)
    if "post" in mode:
        t["post_weight"] = n(dim, std=0.2, mean=1.0)
    if "gate" in mode:
        t["gate"] = n(dim, std=0.5)
    if "groups" in mode:
        t["gate"] = n(rows if rows < 4 else max(k for k in (1, 2, 3, 4, 5, 7, 100) if rows % k == 0), dim, std=0.5)
    seeds = (torch.randn(rows, dim, device="cuda", generator=g), torch.randn(rows, dim, device="cuda", generator=g))
    return t, seeds, dict(kind=kind, eps=1e-5, residual_scale=0.75)


def call(t, how):
    return layers.block_norm(t["x"], t["y"], weight=t["weight"], bias=t["bias"], post_weight=t["post_weight"], gate=t["gate"], **how)


def up(t):
    return None if t is None else t.detach().double()


def restated(t, how):
    return ref.forward(up(t["x"]), up(t["y"]), up(t["weight"]), up(t["bias"]), up(t["post_weight"]), up(t["gate"]), how["residual_scale"], how["kind"], how["eps"])


def within(got, want, bound, what):
    off = (got.double() - want).abs() - bound
    assert torch.isfinite(got).all() and float(off.max()) <= 0.0, "%s: %.3g over its bound" % (what, float(off.max()))


def check(t, seeds, how, use_dr=True):
    r, h = call(t, how)
    s = restated(t, how)
    within(h.detach(), s["h"], s["e_h"], "h")
    if t["y"] is not None:
        within(r.detach(), s["r"], s["e_r"], "r")
    names = [k for k, v in t.items() if v is not None]
    ends, grads = ([r, h], list(seeds)) if t["y"] is not None and use_dr else ([h], [seeds[1]])
    got = dict(zip(names, torch.autograd.grad(ends, [t[k] for k in names], grads)))
    want = ref.backward(s, up(seeds[1]), up(seeds[0]) if len(ends) == 2 else None, up(t["weight"]), up(t["bias"]), up(t["post_weight"]), up(t["gate"]),
                        how["residual_scale"], how["kind"])
    assert set(want) == set(got)
    for k in names:
        within(got[k], *want[k], "gradient of " + k)
    return got, want


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("rows,dim", SHAPES)
def test_values_and_gradients(rows, dim, mode, kind):
    if kind == "layer" and dim == 1:
        pytest.skip("a row of one value has no deviation")
    check(*case(rows, dim, mode, kind))


@pytest.mark.parametrize("mode", ["plain", "residual", "post_gate"])
def test_without_bias_and_without_a_residual_gradient(mode):
    t, seeds, how = case(10, 96, mode, "rms", bias=False)
    check(t, seeds, how, use_dr=False)


def test_only_the_residual_stream_is_used():
    t, seeds, how = case(6, 40, "post_gate", "layer")
    r, _ = call(t, how)
    names = ["x", "y", "post_weight", "gate", "weight"]
    got = torch.autograd.grad(r, [t[k] for k in names], seeds[0])
    want = ref.backward(restated(t, how), torch.zeros_like(up(seeds[0])), up(seeds[0]), up(t["weight"]), up(t["bias"]), up(t["post_weight"]), up(t["gate"]),
                        how["residual_scale"], how["kind"])
    for k, v in zip(names, got):
        within(v, *want[k], k)


@pytest.mark.parametrize("mode,kind", [("post_groups", "layer"), ("post_gate", "rms"), ("plain", "layer")])
def test_gradients_against_differences(mode, kind):
    """The 64-bit formula's central difference along a direction, whose own error at this step is below 1e-7 of the sums of
    magnitudes, against the kernels' gradients, whose bounds add up along the direction."""
    t, seeds, how = case(12, 48, mode, kind)
    got, want = check(t, seeds, how)
    names = list(got)
    g = torch.Generator(device="cuda").manual_seed(1)
    way = {k: torch.randn(t[k].shape, device="cuda", generator=g, dtype=torch.float64) for k in names}

    def f(step):
        moved = {k: (None if v is None else up(v) + step * way[k]) for k, v in t.items()}
        s = restated_of(moved, how)
        total = (s["h"] * up(seeds[1])).sum()
        return total + (s["r"] * up(seeds[0])).sum() if t["y"] is not None else total

    def restated_of(m, how):
        return ref.forward(m["x"], m["y"], m["weight"], m["bias"], m["post_weight"], m["gate"], how["residual_scale"], how["kind"], how["eps"])

    step = 1e-5
    slope = float((f(step) - f(-step)) / (2 * step))
    mine = sum(float((got[k].double() * way[k]).sum()) for k in names)
    size = sum(float((want[k][0] * way[k]).abs().sum()) for k in names)
    bound = sum(float((want[k][1] * way[k].abs()).sum()) for k in names)
    assert abs(slope - mine) <= bound + 1e-7 * size


@pytest.mark.parametrize("dim", [64, 1000, 1001])
def test_unaligned_and_strided_tensors_give_the_same_bits(dim):
    t, seeds, how = case(8, dim, "post_gate", "layer")
    r, h = call(t, how)
    base = torch.autograd.grad([r, h], [t["x"], t["y"], t["gate"]], list(seeds))
    moved = {}
    for k, v in t.items():
        flat = torch.empty(v.numel() + 1, device="cuda")
        flat[1:] = v.detach().view(-1)
        moved[k] = flat[1:].view(v.shape).requires_grad_()
    r2, h2 = call(moved, how)
    again = torch.autograd.grad([r2, h2], [moved["x"], moved["y"], moved["gate"]], [s.t().contiguous().t() for s in seeds])
    for a, b in zip((r, h) + base, (r2, h2) + again):
        assert torch.equal(a, b)


def test_values_that_are_not_finite_stay_in_their_rows():
    t, seeds, how = case(6, 300, "post_gate", "layer")
    clean = call(t, how)[1].detach()
    x = t["x"].detach().clone()
    x[2, 7] = float("nan")
    y = t["y"].detach().clone()
    y[4, 5] = float("inf")
    r, h = layers.block_norm(x, y, weight=t["weight"], bias=t["bias"], post_weight=t["post_weight"], gate=t["gate"], **how)
    for row in range(6):
        assert torch.isnan(h[row]).any() if row in (2, 4) else torch.equal(h[row], clean[row])


def test_rows_of_zeros_and_no_rows():
    w = torch.ones(40, device="cuda", requires_grad=True)
    x = torch.zeros(3, 40, device="cuda", requires_grad=True)
    r, h = layers.block_norm(x, None, weight=w)
    assert torch.equal(h, torch.zeros_like(h))
    dx, dw = torch.autograd.grad(h, [x, w], torch.ones_like(h))
    assert torch.equal(dw, torch.zeros_like(dw)) and torch.isfinite(dx).all()
    e = torch.zeros(0, 40, device="cuda", requires_grad=True)
    y = torch.zeros(0, 40, device="cuda", requires_grad=True)
    gate = torch.ones(40, device="cuda", requires_grad=True)
    r, h = layers.block_norm(e, y, weight=w, post_weight=w.detach().clone().requires_grad_(), gate=gate)
    assert h.shape == (0, 40)
    dw, dg = torch.autograd.grad([r, h], [w, gate], [torch.zeros_like(r), torch.zeros_like(h)])
    assert torch.equal(dw, torch.zeros_like(dw)) and torch.equal(dg, torch.zeros_like(dg))
    gates = torch.ones(3, 40, device="cuda", requires_grad=True)
    r, h = layers.block_norm(e, y, weight=w, post_weight=gate, gate=gates)
    for d in torch.autograd.grad([r, h], [w, gate, gates], [torch.zeros_like(r), torch.zeros_like(h)]):
        assert torch.equal(d, torch.zeros_like(d))


def test_leading_dimensions_and_module():
    m = layers.BlockNorm(96, kind="layer", bias=True, post=True, gate=True, residual_scale=0.5).cuda()
    x, y = torch.randn(2, 5, 96, device="cuda", requires_grad=True), torch.randn(2, 5, 96, device="cuda", requires_grad=True)
    r, h = m(x, y)
    r2, h2 = layers.block_norm(x.view(10, 96), y.view(10, 96), weight=m.weight, bias=m.bias, post_weight=m.post_weight, gate=m.gate, residual_scale=0.5, kind="layer")
    assert r.shape == x.shape and torch.equal(r.view(10, 96), r2) and torch.equal(h.view(10, 96), h2)
    (r.sum() + h.sum()).backward()
    assert all(p.grad is not None for p in m.parameters())
    same, first = m(x)
    assert same is x and first.shape == x.shape
    free = layers.BlockNorm(96, post=True).cuda()
    gates = torch.randn(2, 96, device="cuda")
    assert torch.equal(free(x, y, gate=gates)[1][1], layers.block_norm(x[1], y[1], weight=free.weight, post_weight=free.post_weight, gate=gates[1])[1])
    with pytest.raises(ValueError):
        m(x, y, gate=gates)


def test_runs_repeat_and_do_not_depend_on_the_stream():
    t, seeds, how = case(1000, 520, "post_groups", "layer")
    names = [k for k, v in t.items() if v is not None]

    def once():
        r, h = call(t, how)
        return [r, h] + list(torch.autograd.grad([r, h], [t[k] for k in names], list(seeds)))

    first = once()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        second = once()
    third = once()
    torch.cuda.synchronize()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_captured_calls_at_once():
    """Two graphs captured from the same calls, replayed on two streams at the same time."""
    t, seeds, how = case(512, 768, "post_gate", "rms")
    how = dict(how)
    args = {k: (None if v is None else v.detach()) for k, v in t.items()}

    def once():
        kw = dict(weight=args["weight"], bias=args["bias"], post_weight=args["post_weight"], gate=args["gate"], **how)
        r, h, stats = repro_norm.block_norm(args["x"], args["y"], keep_stats=True, **kw)
        g = repro_norm.block_norm_backward(seeds[1], seeds[0], r, args["y"], stats, **kw)
        return [r, h, g.x, g.y, g.weight, g.bias, g.post_weight, g.gate]

    want = once()
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
    for out in outs:
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_sums_depend_on_sizes_alone():
    """A row's results do not depend on the rows around it."""
    t, seeds, how = case(64, 768, "post_gate", "layer")
    r, h = call(t, how)
    part = {k: (v if k not in ("x", "y") else v[16:24].detach().requires_grad_()) for k, v in t.items()}
    r2, h2 = call(part, how)
    assert torch.equal(r[16:24], r2) and torch.equal(h[16:24], h2)
