"""block_norm and its gradients in float64, with bounds on what float32 kernels may be off by.

u = 2^-24 is the largest relative error of one rounding.  A row's sum adds 8 values a thread, five butterfly steps and up
to 32 warps: at most K = 45 additions deep, so it is off by at most K u times the sum of the magnitudes.  The root
mean square: K + 3 roundings under the root, the root, the reciprocal and the product: (K + 3) / 2 + 3 < 27 u relative.  For the
layer kind the mean is off by (K + 1) u times the mean magnitude A, which moves every centred value by that much and the
deviation by as much relative to it: with a = A / deviation, 46 a u both ways."""
import torch

U = 2.0 ** -24
K = 45


def center(t, kind, eps):
    mean = t.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(t[:, :1])
    rstd = (((t - mean) ** 2).mean(1, keepdim=True) + eps).rsqrt()
    hat = (t - mean) * rstd
    a = t.abs().mean(1, keepdim=True) * rstd * (1.0 if kind == "layer" else 0.0)
    return hat, rstd, U * (hat.abs() * (30 + 46 * a) + 46 * a), a


def rms(t):
    return (t * t).mean(1, keepdim=True).sqrt()


def forward(x, y, w, b, pw, gate, scale, kind, eps):
    """Values (r, h) and the bounds of their errors, plus what the backward pass needs."""
    s = {"r": x, "e_r": torch.zeros_like(x), "x": x, "y": y}
    if y is not None:
        g = torch.ones_like(x) if gate is None else (gate if gate.dim() == 2 else gate[None]).repeat_interleave(
            x.shape[0] // (1 if gate.dim() == 1 else gate.shape[0]), 0) if x.shape[0] else torch.ones_like(x)
        u, e_u = y, torch.zeros_like(y)
        if pw is not None:
            s["yhat"], s["ystd"], e_hat, s["ya"] = center(y, kind, eps)
            u, e_u = s["yhat"] * pw, pw.abs() * e_hat
        s["g"], s["u"] = g, u
        s["r"] = scale * x + g * u
        s["e_r"] = g.abs() * e_u + 3 * U * (g * u).abs() + 2 * U * (scale * x).abs() + U * s["r"].abs()
    s["rhat"], s["rstd"], e_hat, s["ra"] = center(s["r"], kind, eps)
    moved = s["rstd"] * (s["e_r"] + s["e_r"].mean(1, keepdim=True) + s["rhat"].abs() * rms(s["e_r"]))
    s["e_rhat"] = e_hat + moved
    s["h"] = s["rhat"] * w + (0 if b is None else b)
    s["e_h"] = w.abs() * s["e_rhat"] + 3 * U * (s["rhat"] * w).abs() + U * s["h"].abs()
    return s


def _through(q, e_q, hat, rstd, kind, a, e_hat):
    """N' applied to q (off by e_q): value and bound."""
    layer = 1.0 if kind == "layer" else 0.0
    out = rstd * (q - hat * (q * hat).mean(1, keepdim=True) - layer * q.mean(1, keepdim=True))
    size = rstd * (q.abs() + hat.abs() * (q * hat).abs().mean(1, keepdim=True) + layer * q.abs().mean(1, keepdim=True))
    moved = rstd * (e_q + hat.abs() * (e_q * hat.abs()).mean(1, keepdim=True) + layer * e_q.mean(1, keepdim=True)
                    + e_hat * (q * hat).abs().mean(1, keepdim=True) + hat.abs() * (q.abs() * e_hat).mean(1, keepdim=True))
    return out, moved + U * (K + 40 + 46 * a) * size


def backward(s, dh, dr, w, b, pw, gate, scale, kind):
    """{name: (gradient, bound)}.  Column sums add at most as many rows as there are, one rounding each."""
    rows = dh.shape[0]

    def column(term, e_term):
        return term.sum(0), e_term.sum(0) + (rows + 2) * U * term.abs().sum(0)

    out = {"weight": column(dh * s["rhat"], dh.abs() * s["e_rhat"] + U * (dh * s["rhat"]).abs())}
    if b is not None:
        out["bias"] = column(dh, torch.zeros_like(dh))
    q = w * dh
    d, e_d = _through(q, U * q.abs(), s["rhat"], s["rstd"], kind, s["ra"], s["e_rhat"])
    if s["y"] is None:
        out["x"] = (d, e_d)
        return out
    if dr is not None:
        d, e_d = d + dr, e_d + U * (d + dr).abs()
    out["x"] = (scale * d, abs(scale) * e_d + 2 * U * (scale * d).abs())
    hat = s["y"] if pw is None else s["yhat"]
    e_hat = torch.zeros_like(d) if pw is None else U * (hat.abs() * (30 + 46 * s["ya"]) + 46 * s["ya"])
    term, e_term = d * hat, e_d * hat.abs() + d.abs() * e_hat + U * (d * hat).abs()
    if gate is not None:
        groups = 1 if gate.dim() == 1 else gate.shape[0]
        v = (term * (1 if pw is None else pw)).view(groups, -1, d.shape[1])
        e = (e_term * (1 if pw is None else pw.abs())).view(groups, -1, d.shape[1]).sum(1) + (rows + 2) * U * v.abs().sum(1)
        out["gate"] = (v.sum(1).view(gate.shape), e.view(gate.shape))
    if pw is not None:
        out["post_weight"] = column(s["g"] * term, s["g"].abs() * e_term + 2 * U * (s["g"] * term).abs())
    t = d * s["g"] * (1 if pw is None else pw)
    e_t = e_d * (s["g"] * (1 if pw is None else pw)).abs() + 2 * U * t.abs()
    out["y"] = (t, e_t) if pw is None else _through(t, e_t, s["yhat"], s["ystd"], kind, s["ya"], e_hat)
    return out
