"""AdamW over many tensors against its restatement in numpy float32 (equal bits) and the formula in 64 bits."""
import copy

import numpy as np
import pytest
import torch

from bit_reproducible_training_b200 import repro_optim
from optim_restated import adamw, decode, encode

pytestmark = pytest.mark.gpu

HYPER = dict(lr=3e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
SIZES = [[1], [3, 1, 255, 256, 257], [0, 5, 0, 4096, 0], [100003], [1024] * 60, [7, 2049, 8192, 1]]


def bits(t):
    a = t.detach().cpu().numpy() if isinstance(t, torch.Tensor) else t
    return a.reshape(-1).view(np.uint32)


def make(sizes, seed, offset=0):
    """Parameters and gradients, each starting `offset` values past an aligned address."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    ps, gs = [], []
    for n in sizes:
        ps.append(torch.nn.Parameter(torch.randn(n + offset, device="cuda", generator=g)[offset:]))
        gs.append((torch.randn(n + offset, device="cuda", generator=g) * 1e-2)[offset:])
    return ps, gs


def host(ts):
    return [t.detach().cpu().numpy().copy() for t in ts]


@pytest.mark.parametrize("offset", [0, 1, 2])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "%dx%d" % (len(s), max(s)))
def test_fp32_states_have_the_defined_bits(sizes, offset):
    ps, gs = make(sizes, 1, offset)
    opt = repro_optim.AdamW(ps, **HYPER)
    want, m, v = host(ps), [np.zeros(n, np.float32) for n in sizes], [np.zeros(n, np.float32) for n in sizes]
    for n in range(1, 4):
        for i, (p, g) in enumerate(zip(ps, gs)):
            p.grad = g * float(n)
            want[i], m[i], v[i] = adamw(want[i], host([p.grad])[0], m[i], v[i], HYPER["lr"], *HYPER["betas"], HYPER["eps"], HYPER["weight_decay"], n)
        opt.step()
    for i, p in enumerate(ps):
        assert np.array_equal(bits(p), bits(want[i]))
        assert np.array_equal(bits(opt.state[p]["exp_avg"]), bits(m[i])) and np.array_equal(bits(opt.state[p]["exp_avg_sq"]), bits(v[i]))


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: "%dx%d" % (len(s), max(s)))
def test_8_bit_states_have_the_defined_bits(sizes, offset):
    ps, gs = make(sizes, 2, offset)
    opt = repro_optim.AdamW(ps, state_bits=8, **HYPER)
    want = host(ps)
    codes = [encode(np.zeros(n, np.float32), np.zeros(n, np.float32)) for n in sizes]
    for n in range(1, 4):
        for i, (p, g) in enumerate(zip(ps, gs)):
            p.grad = g * float(n)
            m, v = decode(*codes[i])
            want[i], m, v = adamw(want[i], host([p.grad])[0], m, v, HYPER["lr"], *HYPER["betas"], HYPER["eps"], HYPER["weight_decay"], n)
            codes[i] = encode(m, v)
        opt.step()
    ms, vs = [torch.full((n,), 7.0, device="cuda") for n in sizes], [torch.full((n,), 7.0, device="cuda") for n in sizes]
    opt.read_states(ms, vs)
    for i, p in enumerate(ps):
        s = opt.state[p]
        assert np.array_equal(bits(p), bits(want[i]))
        for name, w in zip(("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale"), codes[i]):
            assert np.array_equal(s[name].cpu().numpy(), w), name
        m, v = decode(*codes[i])
        assert np.array_equal(bits(ms[i]), bits(m)) and np.array_equal(bits(vs[i]), bits(v))


def test_many_magnitudes_take_the_defined_codes():
    """Values over the whole float range, subnormals included: every code must be the restatement's."""
    rng = np.random.default_rng(5)
    n = 256 * 400
    m = (rng.standard_normal(n) * 10.0 ** rng.uniform(-44, 37, n)).astype(np.float32)
    m[:256] = 0.0
    m[256:512] = np.float32(1e-45)
    m[512:768] = (rng.standard_normal(256) * 1e-3).astype(np.float32)
    v = np.abs(m[::-1]).copy()
    # magnitudes around the borders between two codes, where a quotient off by one bit would pick the other code
    k = np.arange(256 * 100)
    edge = ((k % 127 + 0.5) / 127) ** 2
    m[1024:1024 + len(k)] = (edge * (1 + (k % 9 - 4) * 2.0 ** -24)).astype(np.float32)
    m[1024:1024 + len(k):256] = 1.0
    edge = ((k % 255 + 0.5) / 255) ** 4
    v[1024:1024 + len(k)] = (edge * (1 + (k % 9 - 4) * 2.0 ** -24)).astype(np.float32)
    v[1024:1024 + len(k):256] = 1.0
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    opt = repro_optim.AdamW([p], state_bits=8)
    opt.write_states([torch.from_numpy(m).cuda()], [torch.from_numpy(v).cuda()])
    s = opt.state[p]
    for name, w in zip(("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale"), encode(m, v)):
        assert np.array_equal(s[name].cpu().numpy(), w), name


def test_step_against_64_bits():
    """Each rounding is off by at most half a step u = 2^-24 of its result.  m': two rounded constants, two products, one sum;
    v': four roundings of positive terms at most on each, so 4u + 1u relative; the divisor: 2.5u + 1u (root) + 2u (product
    and its constant) + 1u (sum); the update: that, the quotient, the product and its constant; p: decay constant, product, sum."""
    u = 2.0 ** -24
    ps, gs = make([5000], 3)
    p0, g = host(ps)[0].astype(np.float64), host(gs)[0].astype(np.float64)
    rng = np.random.default_rng(0)
    m0 = (rng.standard_normal(5000) * 1e-2).astype(np.float32)
    v0 = ((rng.standard_normal(5000) * 1e-2) ** 2).astype(np.float32)
    opt = repro_optim.AdamW(ps, **HYPER)
    opt.adopt([(torch.from_numpy(m0).cuda(), torch.from_numpy(v0).cuda())], step=6)
    ps[0].grad = gs[0]
    opt.step()
    b1, b2 = HYPER["betas"]
    m, v = m0 * b1 + g * (1 - b1), v0 * b2 + g * g * (1 - b2)
    err_m = u * (2 * np.abs(m0 * b1) + 2 * np.abs(g * (1 - b1)) + np.abs(m)) * 1.001
    d = np.sqrt(v / (1 - b2 ** 7)) + HYPER["eps"]
    upd = HYPER["lr"] / (1 - b1 ** 7) * m / d
    err_u = np.abs(upd) * 9.5 * u * 1.001 + HYPER["lr"] / (1 - b1 ** 7) * err_m / d
    p1 = p0 * (1 - HYPER["lr"] * HYPER["weight_decay"])
    assert (np.abs(opt.state[ps[0]]["exp_avg"].cpu().numpy() - m) <= err_m).all()
    assert (np.abs(opt.state[ps[0]]["exp_avg_sq"].cpu().numpy() - v) <= 5.01 * u * v).all()
    assert (np.abs(host(ps)[0] - (p1 - upd)) <= err_u + 2.01 * u * np.abs(p1) + u * np.abs(p1 - upd) * 1.001).all()


@pytest.mark.parametrize("state_bits", [32, 8])
def test_values_that_are_not_finite_stay_visible(state_bits):
    ps, gs = make([1000, 300], 4)
    opt = repro_optim.AdamW(ps, state_bits=state_bits, **HYPER)
    gs[0][300] = float("nan")
    gs[0][900] = float("inf")
    for p, g in zip(ps, gs):
        p.grad = g
    opt.step()
    assert torch.isnan(ps[0][300]) and torch.isnan(ps[0][900])
    assert torch.isfinite(ps[0][:256]).all() and torch.isfinite(ps[1]).all()
    opt.step()
    ms, vs = [torch.empty(1000, device="cuda"), torch.empty(300, device="cuda")], [torch.empty(1000, device="cuda"), torch.empty(300, device="cuda")]
    opt.read_states(ms, vs)
    assert torch.isnan(ms[0][300]) and torch.isfinite(ms[0][:256]).all() and torch.isfinite(ms[1]).all()
    if state_bits == 8:
        assert torch.isnan(ms[0][256:512]).all() and torch.isfinite(ms[0][512:768]).all()


@pytest.mark.parametrize("state_bits", [32, 8])
def test_parameters_without_gradients_wait(state_bits):
    ps, gs = make([600, 700], 6)
    opt = repro_optim.AdamW(ps, state_bits=state_bits, **HYPER)
    before = host(ps)
    ps[0].grad = gs[0]
    opt.step()
    assert np.array_equal(bits(ps[1]), bits(before[1])) and not np.array_equal(bits(ps[0]), bits(before[0]))
    ps[1].grad = gs[1]
    opt.step()                     # the second parameter does its first step, the first its second
    lone, lg = make([600, 700], 6)
    other = repro_optim.AdamW([lone[1]], state_bits=state_bits, **HYPER)
    lone[1].grad = lg[1]
    other.step()
    assert np.array_equal(bits(ps[1]), bits(lone[1]))
    assert opt.state[ps[0]]["step"] == 2 and opt.state[ps[1]]["step"] == 1


@pytest.mark.parametrize("state_bits", [32, 8])
def test_captured_steps_count_on(state_bits):
    ps, gs = make([1000, 77], 7)
    qs, _ = make([1000, 77], 7)
    for p, q, g in zip(ps, qs, gs):
        p.grad, q.grad = g, g.clone()
    eager = repro_optim.AdamW(qs, state_bits=state_bits, **HYPER)
    opt = repro_optim.AdamW(ps, state_bits=state_bits, capturable=True, **HYPER)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(3):
        graph.replay()
    for _ in range(4):
        eager.step()
    torch.cuda.synchronize()
    for p, q in zip(ps, qs):
        assert np.array_equal(bits(p), bits(q))
    assert opt.state_dict()["state"][0]["step"] == 4
    # a loaded state reaches the captured step: the tensors and the counter are the same ones
    opt.load_state_dict(copy.deepcopy(eager.state_dict()))
    graph.replay()
    eager.step()
    torch.cuda.synchronize()
    for p, q in zip(ps, qs):
        assert np.array_equal(bits(p), bits(q))


def test_capture_without_a_device_counter_is_refused():
    ps, gs = make([64], 8)
    ps[0].grad = gs[0]
    opt = repro_optim.AdamW(ps, **HYPER)
    opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    x = torch.zeros(4, device="cuda")
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(RuntimeError, match="capturable"):
            opt.step()
    graph.replay()
    torch.cuda.synchronize()
    cap = repro_optim.AdamW(make([4, 4], 9)[0], capturable=True)
    cap.param_groups[0]["params"][0].grad = torch.zeros(4, device="cuda")
    with pytest.raises(RuntimeError, match="gradient"):
        cap.step()


@pytest.mark.parametrize("first,second", [(32, 32), (8, 8), (32, 8), (8, 32)])
def test_checkpoints_load_into_either_width(first, second):
    ps, gs = make([500, 1000], 10)
    a = repro_optim.AdamW(ps, state_bits=first, **HYPER)
    for p, g in zip(ps, gs):
        p.grad = g
    a.step()
    a.step()
    saved = copy.deepcopy(a.state_dict())
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    b = repro_optim.AdamW(qs, lr=1.0, state_bits=second)
    b.load_state_dict(saved)
    for p, q in zip(ps, qs):
        q.grad = p.grad.clone()
    assert b.param_groups[0]["lr"] == HYPER["lr"] and b.state[qs[0]]["step"] == 2
    a.step()
    b.step()
    if first == second or second == 32:        # the same values are held: the same step
        for p, q in zip(ps, qs):
            assert np.array_equal(bits(p), bits(q))


def test_gradients_of_another_kind_are_refused():
    ps, gs = make([64], 11)
    opt = repro_optim.AdamW(ps, **HYPER)
    before = host(ps)[0]
    for bad in (gs[0].to_sparse(),):
        ps[0].grad = bad
        with pytest.raises(TypeError):
            opt.step()
    assert np.array_equal(bits(ps[0]), bits(before))
    w = torch.nn.Parameter(torch.randn(8, 6, device="cuda"))
    opt = repro_optim.AdamW([w], **HYPER)
    w.grad = torch.randn(6, 8, device="cuda").t()              # a strided gradient is laid out anew
    want = adamw(w.detach().cpu().numpy().reshape(-1), w.grad.cpu().numpy().reshape(-1).copy(), np.zeros(48, np.float32), np.zeros(48, np.float32),
                 HYPER["lr"], *HYPER["betas"], HYPER["eps"], HYPER["weight_decay"], 1)[0]
    opt.step()
    assert np.array_equal(bits(w), bits(want))
    with pytest.raises(ValueError):
        repro_optim.AdamW([w, w])
    with pytest.raises(ValueError):
        opt.read_states([torch.empty(47, device="cuda")], [torch.empty(48, device="cuda")])
    with pytest.raises(ValueError):
        opt.adopt([], step=0)


def test_a_saved_graph_notices_the_step():
    w = torch.nn.Parameter(torch.randn(4, 4, device="cuda"))
    x = torch.randn(4, 4, device="cuda", requires_grad=True)
    loss = (x @ w).sum()
    w.grad = torch.ones_like(w)
    repro_optim.AdamW([w], **HYPER).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_step_on_another_stream():
    ps, gs = make([200000], 12)
    qs, _ = make([200000], 12)
    ps[0].grad = qs[0].grad = gs[0]
    a, b = repro_optim.AdamW(ps, **HYPER), repro_optim.AdamW(qs, **HYPER)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        a.step()
    b.step()
    torch.cuda.synchronize()
    assert np.array_equal(bits(ps[0]), bits(qs[0]))


def test_hooks_and_schedulers_work():
    ps, gs = make([64], 13)
    ps[0].grad = gs[0]
    opt = repro_optim.AdamW(ps, **HYPER)
    seen = []
    opt.register_step_pre_hook(lambda o, a, k: seen.append("before"))
    opt.register_step_post_hook(lambda o, a, k: seen.append("after"))
    sched = torch.optim.lr_scheduler.StepLR(opt, 1, gamma=0.5)
    assert opt.step(lambda: 5.0) == 5.0
    sched.step()
    assert seen == ["before", "after"] and opt.param_groups[0]["lr"] == HYPER["lr"] * 0.5 and opt.state[ps[0]]["step"] == 1


def test_a_parameter_that_changed_its_size_is_refused():
    ps, gs = make([64, 8], 14)
    for p, g in zip(ps, gs):
        p.grad = g
    opt = repro_optim.AdamW(ps, **HYPER)
    opt.step()
    ps[0].data = torch.zeros(32, device="cuda")
    with pytest.raises(ValueError):
        opt.step()


@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("state_bits", [32, 8])
def test_a_copied_optimizer_has_states_of_its_own(state_bits, capturable):
    ps, gs = make([300, 40], 15)
    for p, g in zip(ps, gs):
        p.grad = g
    opt = repro_optim.AdamW(ps, state_bits=state_bits, capturable=capturable, **HYPER)
    opt.step()
    twin = copy.deepcopy(opt)
    qs = twin.param_groups[0]["params"]
    for p, q in zip(ps, qs):
        assert q is not p
        q.grad = p.grad.clone()
    kept = [t.clone() for t in opt.state[ps[0]].values() if isinstance(t, torch.Tensor)]
    twin.step()
    assert all(torch.equal(a, b) for a, b in zip(kept, (t for t in opt.state[ps[0]].values() if isinstance(t, torch.Tensor))))
    opt.step()
    for p, q in zip(ps, qs):
        assert np.array_equal(bits(p), bits(q))


def test_replaced_state_tensors_do_not_leave_the_kernel_without_memory():
    ps, gs = make([300], 16)
    ps[0].grad = gs[0]
    opt = repro_optim.AdamW(ps, **HYPER)
    opt.step()
    held = opt._tables[0]["kept"][0]
    opt.state[ps[0]]["exp_avg"] = torch.zeros(300, device="cuda")
    before = held.clone()
    opt.step()
    assert not torch.equal(held, before)             # the step's own tensor was updated; adopt() is the way to replace it


def test_parameters_part_and_meet_again():
    """Missing gradients part the parameters' counters; a loaded state joins them again; a table made from states that differ works too."""
    ps, gs = make([300, 40, 5], 17)
    opt = repro_optim.AdamW(ps, **HYPER)
    for have in ((0, 1, 2), (0, 2), (1,), (), (0, 1, 2)):
        for i, p in enumerate(ps):
            p.grad = gs[i] if i in have else None
        opt.step()
    assert [int(opt.state[p]["step"]) for p in ps] == [3, 3, 3]
    saved = copy.deepcopy(opt.state_dict())
    saved["state"][1]["step"] = 7
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    twin = repro_optim.AdamW(qs, **HYPER)
    twin.load_state_dict(saved)
    for q, g in zip(qs, gs):
        q.grad = g
    twin.step()
    assert [int(twin.state[q]["step"]) for q in qs] == [4, 8, 4]
    want = adamw(host([ps[1]])[0], host([gs[1]])[0], *(saved["state"][1][k].cpu().numpy() for k in ("exp_avg", "exp_avg_sq")), HYPER["lr"], *HYPER["betas"],
                 HYPER["eps"], HYPER["weight_decay"], 8)[0]
    assert np.array_equal(bits(qs[1]), bits(want))
    saved["state"][1]["step"] = 3
    twin.load_state_dict(saved)
    twin.step()
    assert [int(twin.state[q]["step"]) for q in qs] == [4, 4, 4] and twin.state[qs[0]]["step"] is twin.state[qs[2]]["step"]
    # the same sequence of steps on each parameter alone
    for i, p in enumerate(ps):
        lone = torch.nn.Parameter(make([300, 40, 5], 17)[0][i].detach().clone())
        alone = repro_optim.AdamW([lone], **HYPER)
        lone.grad = gs[i]
        for _ in range(3):
            alone.step()
        assert np.array_equal(bits(p), bits(lone))


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float64])
def test_swapped_gradient_data_is_refused(kind):
    ps, gs = make([64, 8], 18)
    for p, g in zip(ps, gs):
        p.grad = g
    opt = repro_optim.AdamW(ps, **HYPER)
    opt.step()
    before = host(ps)
    ps[0].grad.data = ps[0].grad.data.to(kind)
    with pytest.raises(TypeError):
        opt.step()
    ps[0].grad = None
    ps[0].grad = gs[0].float()
    ps[1].grad.data = ps[1].grad.data.cpu()
    with pytest.raises(TypeError):
        opt.step()
    assert all(np.array_equal(bits(a), bits(b)) for a, b in zip(ps, before)) and int(opt.state[ps[0]]["step"]) == 1
