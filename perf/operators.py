"""The operators around the reproducible products of a language-model training step, as cases that can be timed.

Four operators, each with its plain form in elementary torch operations and, where ``own`` is true, the call a user
of this library makes:

linear  Y = act(X W^T + b) + R, and as a training step also dX, dW, db from dY
        (``layers.linear``; the residual's gradient is dY itself)
norm    r = s X + g * (w' * N(Y)), h = w * N(r) + b: the norm behind a block, its gate, the residual stream and the
        norm in front of the next block; as a training step also every gradient (``layers.block_norm``)
xent    the cross entropy of X W^T against targets without the [tokens, vocabulary] logits, with dX and dW
        (``layers.linear_cross_entropy``)
adamw   one AdamW step over a model's tensors, states in 32 bits or as 8-bit codes with a scale for each 256 values
        (``repro_optim.AdamW``); 8-bit states come back as the values they stand for

All tensors are float32, like everything else in this library.
"""
import math

import torch

own = False

BLOCK = 256         # values that share a scale in 8-bit optimizer states


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # attention output projection of a few tokens: bias and residual behind a small product, bound by latency
        dict(name="linear_fwd_small", op="linear", step=False, m=32, k=768, n=768, act="none", bias=True, residual=True),
        # a ragged evaluation batch through a layer of odd widths
        dict(name="linear_fwd_ragged", op="linear", step=False, m=777, k=515, n=1001, act="silu", bias=True, residual=True),
        # the widening half of an MLP in training: 8192 tokens, 1024 -> 4096, forward and all gradients
        dict(name="linear_step_mlp", op="linear", step=True, m=8192, k=1024, n=4096, act="gelu_tanh", bias=True, residual=False),
        # the norm in front of the first block for a handful of tokens
        dict(name="norm_fwd_small", op="norm", step=False, rows=32, dim=768, kind="rms", block=False, post=False, gate="none", groups=1, bias=False, scale=1.0),
        # layer norms with a gate for each of seven sequences (adaptive modulation), odd width
        dict(name="norm_step_ragged", op="norm", step=True, rows=1995, dim=1001, kind="layer", block=True, post=True, gate="groups", groups=7, bias=True, scale=1.0),
        # norms on both sides of a wide block, a learned gate for each channel, scaled residual stream
        dict(name="norm_step_wide", op="norm", step=True, rows=8192, dim=4096, kind="rms", block=True, post=True, gate="channel", groups=1, bias=False, scale=0.5),
        # a small character-level model's loss
        dict(name="xent_small", op="xent", tokens=128, dim=256, vocab=1000, ignored=0.0, reduction="mean"),
        # prompts masked out of the loss, odd vocabulary, summed loss (gradient accumulation)
        dict(name="xent_ragged", op="xent", tokens=1000, dim=512, vocab=32003, ignored=0.25, reduction="sum"),
        # the lm_head of the suite's model (768 wide, 50257 words) on a training batch of 8192 tokens
        dict(name="xent_large", op="xent", tokens=8192, dim=768, vocab=50257, ignored=0.02, reduction="mean"),
        # a toy model: a few dozen small tensors, bound by launches
        dict(name="adamw32_small", op="adamw", bits=32, layers=4, width=64, hidden=176, vocab=257),
        # all tensors of a 12-layer, 768-wide model with a 50257-word embedding (124 M values)
        dict(name="adamw32_model", op="adamw", bits=32, layers=12, width=768, hidden=2048, vocab=50257),
        # the same model with states in 8 bits
        dict(name="adamw8_model", op="adamw", bits=8, layers=12, width=768, hidden=2048, vocab=50257),
    ]


def _log(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["linear", "norm", "xent", "adamw"])
    if op == "linear":
        while True:
            m, k, n = _log(rng, 1, 8192), _log(rng, 16, 4096), _log(rng, 16, 4096)
            if m * k * n <= 8192 * 1024 * 4096:
                break
        return dict(op=op, step=rng.random() < 0.6, m=m, k=k, n=n, act=rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]),
                    bias=rng.random() < 0.8, residual=rng.random() < 0.5)
    if op == "norm":
        while True:
            rows, dim = _log(rng, 1, 16384), _log(rng, 32, 8192)
            if rows * dim <= 8192 * 4096:
                break
        block = rng.random() < 0.8
        post = block and rng.random() < 0.6
        gate = rng.choice(["none", "channel", "groups"]) if block else "none"
        groups = rng.choice([g for g in (1, 2, 3, 4, 7, 8, 16) if rows % g == 0]) if gate == "groups" else 1
        kind = rng.choice(["rms", "layer"])
        return dict(op=op, step=rng.random() < 0.6, rows=rows, dim=dim, kind=kind, block=block, post=post, gate=gate, groups=groups,
                    bias=kind == "layer", scale=rng.choice([1.0, 0.5, 0.7071]))
    if op == "xent":
        while True:
            tokens, dim, vocab = _log(rng, 4, 8192), _log(rng, 32, 1024), _log(rng, 50, 65536)
            if tokens * dim * vocab <= 8192 * 768 * 50257:
                break
        return dict(op=op, tokens=tokens, dim=dim, vocab=vocab, ignored=rng.choice([0.0, 0.05, 0.5]), reduction=rng.choice(["mean", "sum"]))
    layers, width = rng.randint(1, 12), _log(rng, 32, 768)
    return dict(op=op, bits=rng.choice([32, 8]), layers=layers, width=width, hidden=width * 8 // 3, vocab=_log(rng, 100, 50257))


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _shapes(case):
    d, f = case["width"], case["hidden"]
    per_layer = [(d,), (d, d), (d, d), (d, d), (d, d), (d,), (f, d), (f, d), (d, f)]
    return [(case["vocab"], d)] + per_layer * case["layers"] + [(d,)]


def _adamw_layout(case):
    """Each tensor at a multiple of BLOCK values of one flat buffer: (offset, count, shape) of each, and the buffer's length."""
    at, got = 0, []
    for s in _shapes(case):
        n = math.prod(s)
        got.append((at, n, s))
        at += -(-n // BLOCK) * BLOCK
    return got, at


def _encode(m, v):
    """8-bit codes of first and second moments, flat buffers of whole blocks: square-law for m, fourth-power for v."""
    m, v = m.view(-1, BLOCK), v.view(-1, BLOCK)
    sm, sv = m.abs().amax(1, keepdim=True), v.amax(1, keepdim=True)
    rm = torch.sqrt(m.abs() / torch.where(sm > 0, sm, torch.ones_like(sm)))
    rv = torch.sqrt(torch.sqrt(v / torch.where(sv > 0, sv, torch.ones_like(sv))))
    qm = torch.round(rm * 127.0) * torch.sign(m)
    qv = torch.maximum(torch.round(rv * 255.0), (v > 0).float())
    return qm.to(torch.int8).view(-1), sm.view(-1), qv.to(torch.uint8).view(-1), sv.view(-1)


def _decode(qm, sm, qv, sv):
    tm = qm.view(-1, BLOCK).float() * (1.0 / 127.0)
    tv = qv.view(-1, BLOCK).float() * (1.0 / 255.0)
    tv = tv * tv
    return ((tm * tm.abs()) * sm[:, None]).view(-1), ((tv * tv) * sv[:, None]).view(-1)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, device="cuda", generator=g).mul_(std).add_(mean)

    op, s = case["op"], {"case": case}
    if op == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        s.update(x=normal(m, k).requires_grad_(), w=normal(n, k, std=0.02).requires_grad_(),
                 b=normal(n, std=0.02).requires_grad_() if case["bias"] else None,
                 r=normal(m, n) if case["residual"] else None, dy=normal(m, n, std=1e-3) if case["step"] else None)
    elif op == "norm":
        rows, dim = case["rows"], case["dim"]
        s.update(x=normal(rows, dim).requires_grad_(), y=normal(rows, dim, std=0.5).requires_grad_() if case["block"] else None,
                 w=normal(dim, std=0.1, mean=1.0).requires_grad_(),
                 b=normal(dim, std=0.1).requires_grad_() if case["bias"] else None,
                 pw=normal(dim, std=0.1, mean=1.0).requires_grad_() if case["post"] else None, gate=None)
        if case["gate"] != "none":
            shape = (dim,) if case["gate"] == "channel" else (case["groups"], dim)
            s["gate"] = normal(*shape, std=0.2, mean=0.5).requires_grad_()
        if case["step"]:
            s.update(dr=normal(rows, dim, std=1e-3) if case["block"] else None, dh=normal(rows, dim, std=1e-3))
    elif op == "xent":
        n, d, v = case["tokens"], case["dim"], case["vocab"]
        # words by rank: the frequent ones come many times in a batch, as in text
        u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
        t = (torch.exp(u * math.log(v + 1)) - 1).long().clamp_(0, v - 1)
        t[torch.rand(n, device="cuda", generator=g) < case["ignored"]] = -100
        s.update(x=normal(n, d).requires_grad_(), w=normal(v, d, std=0.02 * math.sqrt(768 / d)).requires_grad_(), t=t)
    else:
        lay, total = _adamw_layout(case)
        used = torch.zeros(total, device="cuda", dtype=torch.bool)
        for at, n, _ in lay:
            used[at:at + n] = True
        flat = {"p": normal(total, std=0.02), "g": normal(total, std=1e-3), "m": normal(total, std=3e-4), "v": normal(total, std=1e-3).square_()}
        for f in flat.values():
            f.mul_(used)
        s.update(flat=flat, count=10, hyper=dict(lr=3e-4, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1))
        if case["bits"] == 8:
            s["codes"] = _encode(flat.pop("m"), flat.pop("v"))
            s["values"] = (torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda"))
        if own:
            s["opt"] = _optimizer(s, lay)
    return s


def _views(flat, lay, per=1):
    return [flat[at // per:at // per + -(-n // per)].view(shape if per == 1 else (-1,)) for at, n, shape in lay]


def _optimizer(s, lay):
    """The handle a training program keeps: the optimizer over its parameters, resumed from the states at hand."""
    from bit_reproducible_training_b200 import repro_optim
    params = [torch.nn.Parameter(p) for p in _views(s["flat"]["p"], lay)]
    for p, grad in zip(params, _views(s["flat"]["g"], lay)):
        p.grad = grad
    if s["case"]["bits"] == 8:
        qm, sm, qv, sv = s["codes"]
        states = list(zip(_views(qm, lay), _views(qv, lay), _views(sm, lay, BLOCK), _views(sv, lay, BLOCK)))
        s["out"] = [_views(v, lay) for v in s["values"]]
    else:
        states = list(zip(_views(s["flat"]["m"], lay), _views(s["flat"]["v"], lay)))
    opt = repro_optim.AdamW(params, state_bits=s["case"]["bits"], **s["hyper"])
    opt.adopt(states, step=s["count"])
    return opt


# ---------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------
C0, C1 = math.sqrt(2.0 / math.pi), 0.044715


def _act(z, kind):
    if kind == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if kind == "silu":
        return z / (1.0 + torch.exp(-z))
    if kind == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if kind == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(C0 * (z + C1 * z * z * z)))
    return z


def _act_slope(z, kind):
    if kind == "relu":
        return (z > 0).float()
    if kind == "silu":
        p = 1.0 / (1.0 + torch.exp(-z))
        return p * (1.0 + z * (1.0 - p))
    if kind == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    t = torch.tanh(C0 * (z + C1 * z * z * z))
    return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * C0 * (1.0 + 3.0 * C1 * z * z)


def _plain_linear(s):
    c = s["case"]
    z = s["x"] @ s["w"].t()
    if s["b"] is not None:
        z = z + s["b"]
    y = _act(z, c["act"])
    if s["r"] is not None:
        y = y + s["r"]
    if not c["step"]:
        return {"y": y}
    dz = s["dy"] if c["act"] == "none" else s["dy"] * _act_slope(z, c["act"])
    out = {"y": y, "dx": dz @ s["w"], "dw": dz.t() @ s["x"]}
    if s["b"] is not None:
        out["db"] = dz.sum(0)
    return out


def _center(x, kind, eps):
    """(x - mean) / std, and 1 / std."""
    if kind == "layer":
        x = x - x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((x * x).mean(1, keepdim=True) + eps)
    return x * rstd, rstd


def _center_back(d, xhat, rstd, kind):
    d = d - xhat * (d * xhat).mean(1, keepdim=True) - (d.mean(1, keepdim=True) if kind == "layer" else 0.0)
    return d * rstd


EPS = 1e-5


def _plain_norm(s):
    c = s["case"]
    kind, x, y, gate = c["kind"], s["x"], s["y"], s["gate"]
    rows, dim = x.shape
    if y is not None:
        u, yhat, ystd = y, None, None
        if s["pw"] is not None:
            yhat, ystd = _center(y, kind, EPS)
            u = yhat * s["pw"]
        rows_gate = None
        if gate is not None:
            rows_gate = gate if gate.dim() == 1 else gate[:, None, :].expand(gate.shape[0], rows // gate.shape[0], dim).reshape(rows, dim)
        r = c["scale"] * x + (u if gate is None else rows_gate * u)
    else:
        r = x
    rhat, rstd = _center(r, kind, EPS)
    h = rhat * s["w"]
    if s["b"] is not None:
        h = h + s["b"]
    out = {"h": h}
    if y is not None:
        out["r"] = r
    if not c["step"]:
        return out
    dh = s["dh"]
    out["dw"] = (dh * rhat).sum(0)
    if s["b"] is not None:
        out["db"] = dh.sum(0)
    dr = _center_back(dh * s["w"], rhat, rstd, kind)
    if y is None:
        out["dx"] = dr
        return out
    dr = dr + s["dr"]
    out["dx"] = dr * c["scale"]
    if gate is not None:
        t = dr * u
        out["dgate"] = t.sum(0) if gate.dim() == 1 else t.view(gate.shape[0], -1, dim).sum(1)
        du = dr * rows_gate
    else:
        du = dr
    if s["pw"] is not None:
        out["dpw"] = (du * yhat).sum(0)
        du = _center_back(du * s["pw"], yhat, ystd, kind)
    out["dy"] = du
    return out


def _plain_xent(s):
    c, x, w, t = s["case"], s["x"], s["w"], s["t"]
    keep = t >= 0
    at = torch.where(keep, t, torch.zeros_like(t))[:, None]
    z = x @ w.t()
    top = z.amax(1, keepdim=True)
    p = torch.exp(z - top)
    total = p.sum(1, keepdim=True)
    nll = torch.where(keep, (torch.log(total) + top - z.gather(1, at))[:, 0], torch.zeros_like(top[:, 0]))
    scale = keep.float()
    loss = nll.sum()
    if c["reduction"] == "mean":
        count = scale.sum().clamp(min=1.0)
        loss, scale = loss / count, scale / count
    p = p / total
    p.scatter_add_(1, at, torch.full_like(top, -1.0))
    p = p * scale[:, None]
    return {"loss": loss, "dx": p @ w, "dw": p.t() @ x}


def _plain_adamw(s):
    h, f = s["hyper"], s["flat"]
    (b1, b2), lr = h["betas"], h["lr"]
    s["count"] += 1
    p, g = f["p"], f["g"]
    m, v = _decode(*s["codes"]) if "codes" in s else (f["m"], f["v"])
    p.mul_(1.0 - lr * h["weight_decay"])
    m.mul_(b1).add_(g * (1.0 - b1))
    v.mul_(b2).add_((g * g) * (1.0 - b2))
    denom = torch.sqrt(v).mul_(1.0 / math.sqrt(1.0 - b2 ** s["count"])).add_(h["eps"])
    p.sub_((m / denom).mul_(lr / (1.0 - b1 ** s["count"])))
    if "codes" not in s:
        return {"p": p, "m": m, "v": v}
    s["codes"] = _encode(m, v)
    m, v = _decode(*s["codes"])
    return {"p": p, "m": m, "v": v}


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def run(s):
    if own:
        return _own(s)
    with torch.no_grad():
        return {"linear": _plain_linear, "norm": _plain_norm, "xent": _plain_xent, "adamw": _plain_adamw}[s["case"]["op"]](s)


def _own(s):
    from bit_reproducible_training_b200 import layers
    c = s["case"]
    if c["op"] == "linear":
        act = None if c["act"] == "none" else c["act"]
        if not c["step"]:
            with torch.no_grad():
                return {"y": layers.linear(s["x"], s["w"], s["b"], activation=act, residual=s["r"])}
        y = layers.linear(s["x"], s["w"], s["b"], activation=act, residual=s["r"])
        names = ["x", "w"] + (["b"] if s["b"] is not None else [])
        grads = torch.autograd.grad(y, [s[k] for k in names], s["dy"])
        return {"y": y, **{"d" + k: v for k, v in zip(names, grads)}}
    if c["op"] == "norm":
        kw = dict(weight=s["w"], bias=s["b"], post_weight=s["pw"], gate=s["gate"], residual_scale=c["scale"], kind=c["kind"], eps=EPS)
        if not c["step"]:
            with torch.no_grad():
                r, h = layers.block_norm(s["x"], s["y"], **kw)
            return {"h": h} if s["y"] is None else {"h": h, "r": r}
        r, h = layers.block_norm(s["x"], s["y"], **kw)
        names = [k for k in ("x", "y", "w", "b", "pw", "gate") if s[k] is not None]
        if s["y"] is None:
            grads = torch.autograd.grad(h, [s[k] for k in names], s["dh"])
            return {"h": h, **{"d" + k: v for k, v in zip(names, grads)}}
        grads = torch.autograd.grad([r, h], [s[k] for k in names], [s["dr"], s["dh"]])
        return {"h": h, "r": r, **{"d" + k: v for k, v in zip(names, grads)}}
    if c["op"] == "xent":
        loss = layers.linear_cross_entropy(s["x"], s["w"], s["t"], reduction=c["reduction"])
        dx, dw = torch.autograd.grad(loss, [s["x"], s["w"]])
        return {"loss": loss, "dx": dx, "dw": dw}
    s["opt"].step()
    if c["bits"] == 32:
        return {k: s["flat"][k] for k in ("p", "m", "v")}
    s["opt"].read_states(*s["out"])
    return {"p": s["flat"]["p"], "m": s["values"][0], "v": s["values"][1]}


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        moved = m * k + n * k + m * n + n * case["bias"] + m * n * case["residual"]
        if case["step"]:
            moved += m * n + m * k + n * k + n * case["bias"]
        return {"bytes": 4 * moved, "flops": 2 * m * n * k * (3 if case["step"] else 1)}
    if op == "norm":
        n, d = case["rows"] * case["dim"], case["dim"]
        vectors = d * (1 + case["bias"] + case["post"]) + (d * case["groups"] if case["gate"] != "none" else 0)
        tensors = 4 if case["block"] else 2
        return {"bytes": 4 * (tensors * n + vectors) * (2 if case["step"] else 1), "flops": 10 * n * (3 if case["step"] else 1)}
    if op == "xent":
        n, d, v = case["tokens"], case["dim"], case["vocab"]
        return {"bytes": 4 * 2 * (n * d + v * d) + 8 * n, "flops": 3 * 2 * n * v * d}
    n = sum(math.prod(s) for s in _shapes(case))
    if case["bits"] == 32:
        return {"bytes": 28 * n, "flops": 14 * n}
    # parameters and gradients, codes read and written, scales, and the values that the codes stand for
    return {"bytes": (12 + 4 + 8) * n + 4 * 4 * (n // BLOCK), "flops": 24 * n}


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    F = torch.nn.functional

    def up(name):
        t = s.get(name)
        return None if t is None else t.detach().double().requires_grad_(t.requires_grad)

    if case["op"] == "linear":
        x, w, b, r = up("x"), up("w"), up("b"), up("r")
        z = F.linear(x, w, b)
        y = {"none": lambda t: t, "relu": F.relu, "silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh")}[case["act"]](z)
        y = y if r is None else y + r
        if not case["step"]:
            return {"y": y.detach()}
        names = [("dx", x), ("dw", w)] + ([("db", b)] if b is not None else [])
        grads = torch.autograd.grad(y, [t for _, t in names], s["dy"].double())
        return {"y": y.detach(), **{n: v for (n, _), v in zip(names, grads)}}
    if case["op"] == "norm":
        leaves = {k: up(k) for k in ("x", "y", "w", "b", "pw", "gate")}
        dim = (case["dim"],)

        def norm(t, weight, bias=None):
            if case["kind"] == "layer":
                return F.layer_norm(t, dim, weight, bias, EPS)
            t = t / torch.sqrt(torch.mean(t.pow(2), -1, keepdim=True) + EPS) * weight
            return t if bias is None else t + bias

        r = leaves["x"]
        if case["block"]:
            u = leaves["y"] if leaves["pw"] is None else norm(leaves["y"], leaves["pw"])
            if leaves["gate"] is not None:
                u = (u.view(case["groups"], -1, case["dim"]) * leaves["gate"].view(case["groups"], 1, case["dim"])).view(u.shape)
            r = case["scale"] * leaves["x"] + u
        h = norm(r, leaves["w"], leaves["b"])
        out = {"h": h.detach(), **({"r": r.detach()} if case["block"] else {})}
        if case["step"]:
            names = [k for k, t in leaves.items() if t is not None]
            ends, seeds = ([r, h], [s["dr"].double(), s["dh"].double()]) if case["block"] else ([h], [s["dh"].double()])
            out.update({"d" + k: v for k, v in zip(names, torch.autograd.grad(ends, [leaves[k] for k in names], seeds))})
        return out
    if case["op"] == "xent":
        x, w = up("x"), up("w")
        loss = F.cross_entropy(F.linear(x, w), s["t"], ignore_index=-100, reduction="sum")
        if case["reduction"] == "mean":
            loss = loss / max(1, int((s["t"] != -100).sum()))
        dx, dw = torch.autograd.grad(loss, [x, w])
        return {"loss": loss.detach(), "dx": dx, "dw": dw}
    f, h, n = s["flat"], s["hyper"], s["count"] + 1
    (b1, b2), g = h["betas"], f["g"].double()
    m, v = (t.double() for t in (_decode(*s["codes"]) if "codes" in s else (f["m"], f["v"])))
    m, v = torch.lerp(g, m, b1), torch.lerp(g.square(), v, b2)
    step = (m / (1 - b1 ** n)) / ((v / (1 - b2 ** n)).sqrt() + h["eps"])
    p = f["p"].double()
    p = p - h["lr"] * (step + h["weight_decay"] * p)
    # codes have no 64-bit value: a value beside a border between two codes may take either
    return {"p": p, "m": None, "v": None} if "codes" in s else {"p": p, "m": m, "v": v}
