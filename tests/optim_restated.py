"""The AdamW step and the 8-bit codes restated in numpy float32, operation by operation, as include/rgb200_train.h defines them
(numpy rounds each float32 operation once, like the kernels)."""
import numpy as np

F = np.float32
BLOCK = 256


def adamw(p, g, m, v, lr, b1, b2, eps, wd, n):
    p1 = p * F(1.0 - lr * wd)
    m = m * F(b1) + g * F(1.0 - b1)
    v = v * F(b2) + (g * g) * F(1.0 - b2)
    d = np.sqrt(v) * F(1.0 / np.sqrt(1.0 - b2 ** n)) + F(eps)
    return p1 - (m / d) * F(lr / (1.0 - b1 ** n)), m, v


def _blocked(x):
    pad = -len(x) % BLOCK
    return np.concatenate([x, np.zeros(pad, F)]).reshape(-1, BLOCK)


def encode(m, v):
    n = len(m)
    m, v = _blocked(m), _blocked(v)
    out = []
    for x, second in ((m, False), (v, True)):
        scale = np.abs(x).max(1)
        bad = ~np.isfinite(x).all(1)
        d = np.where(bad | (scale == 0), F(1), scale)[:, None]
        x = np.where(bad[:, None], F(0), x)
        if second:
            q = np.rint(np.sqrt(np.sqrt(x / d)) * F(255))
            q = np.where((q == 0) & (x > 0), 1, q).astype(np.uint8)
        else:
            q = (np.rint(np.sqrt(np.abs(x) / d) * F(127)) * np.sign(x)).astype(np.int8)
        out += [q.reshape(-1)[:n], np.where(bad, F(np.nan), scale).astype(F)]
    return tuple(out)


def decode(qm, sm, qv, sv):
    n = len(qm)
    t = qm.astype(F) * F(1.0 / 127.0)
    u = qv.astype(F) * F(1.0 / 255.0)
    u = u * u
    return (t * np.abs(t)) * np.repeat(sm, BLOCK)[:n], (u * u) * np.repeat(sv, BLOCK)[:n]
