"""The norm behind a block, its gate, the residual stream and the norm in front of the next block, on the C ABI.

    u = post_weight * N(y)        (u = y without a post weight)
    r = residual_scale * x + gate * u
    h = weight * N(r) + bias      (h = weight * N(x) + bias without y)

One pass over the rows forward, one backward; ``layers.block_norm`` and ``layers.BlockNorm`` are the differentiable forms.
CUDA float32 tensors only; sums are taken in an order that depends on the sizes alone.
"""
import ctypes as C
from dataclasses import dataclass

import torch

from . import _lib
from .repro_gemm import ReproGemmError, _addr, _check, _extent, _on, _raw_stream, _scratch, cudaSuccess

KINDS = {"rms": 0, "layer": 1}
MAX_DIM = 8192
MAX_GROUPS = 1 << 30


@dataclass
class NormGrads:
    """What block_norm_backward returns; None where no gradient was asked for."""
    x: torch.Tensor = None
    y: torch.Tensor = None
    weight: torch.Tensor = None
    bias: torch.Tensor = None
    post_weight: torch.Tensor = None
    gate: torch.Tensor = None


def _same_device(tensors):
    where = tensors[0].device
    for t in tensors:
        if t is not None and t.device != where:
            raise ValueError("all tensors must be on one device")


def _sizes(x, y, weight, bias, post_weight, gate, kind, eps):
    if kind not in KINDS:
        raise ValueError("kind must be 'rms' or 'layer'")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_DIM:
        raise ValueError("the last dimension must have 1 to %d values" % MAX_DIM)
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    dim = x.shape[-1]
    rows = x.numel() // dim
    if y is None and (post_weight is not None or gate is not None):
        raise ValueError("post_weight and gate need y")
    if y is not None and y.shape != x.shape:
        raise ValueError("y must have the shape of x")
    _extent(rows)
    groups = 1
    if gate is not None:
        if gate.dim() not in (1, 2) or gate.shape[-1] != dim:
            raise ValueError("gate must be [dim] or [groups, dim]")
        groups = 1 if gate.dim() == 1 else gate.shape[0]
        if groups < 1 or rows % groups != 0:
            raise ValueError("the rows must divide into the gate's groups")
        if groups > MAX_GROUPS:
            raise ValueError("a gate may have 2^30 rows at most")
    _same_device((x, y, weight, bias, post_weight, gate))
    return rows, dim, groups


def block_norm(x, y=None, *, weight, bias=None, post_weight=None, gate=None, residual_scale=1.0, kind="rms", eps=1e-5, keep_stats=False):
    """(r, h, stats) with r = x when y is None, and stats None unless kept for block_norm_backward.

    x, y: [..., dim]; weight, bias, post_weight: [dim]; gate: [dim] or [groups, dim], each row of the gate for rows / groups
    consecutive rows of x (a batch of equally long sequences: groups = batch)."""
    rows, dim, groups = _sizes(x, y, weight, bias, post_weight, gate, kind, eps)
    shape = x.shape
    x = _check(x, rows * dim, "x")
    y = None if y is None else _check(y, rows * dim, "y")
    weight = _check(weight, dim, "weight")
    bias = None if bias is None else _check(bias, dim, "bias")
    post_weight = None if post_weight is None else _check(post_weight, dim, "post_weight")
    gate = None if gate is None else _check(gate, groups * dim, "gate")
    h = torch.empty(shape, dtype=torch.float32, device=x.device)
    r = x if y is None else torch.empty(shape, dtype=torch.float32, device=x.device)
    stats = torch.empty((4, rows), dtype=torch.float32, device=x.device) if keep_stats else None
    n = _lib.BlockNorm(rows, dim, groups, KINDS[kind], residual_scale, eps, _addr(x), _addr(y), _addr(weight), _addr(bias), _addr(post_weight),
                       _addr(gate), None if y is None else _addr(r), _addr(h), _addr(stats))
    with _on(x.device):
        rc = _lib.lib().rgb200_block_norm_forward(C.byref(n), _raw_stream(x.device))
    if rc != cudaSuccess:
        raise ReproGemmError(rc, "block_norm_forward")
    return r, h, stats


def block_norm_backward(dh, dr, r, y, stats, *, weight, bias=None, post_weight=None, gate=None, residual_scale=1.0, kind="rms", eps=1e-5,
                        wanted=("x", "y", "weight", "bias", "post_weight", "gate")):
    """Gradients of block_norm from dh and dr (the gradient that reaches r, without y x itself, from the residual stream; may be None).
    r, y, stats: what the forward call returned and took.  `wanted` names the gradients to form."""
    rows, dim, groups = _sizes(r, y, weight, bias, post_weight, gate, kind, eps)
    _same_device((r, dh, dr, stats))
    shape = r.shape
    like = {name: t.shape for name, t in (("weight", weight), ("bias", bias), ("post_weight", post_weight), ("gate", gate)) if t is not None}
    r, dh, stats, weight = _check(r, rows * dim, "r"), _check(dh, rows * dim, "dh"), _check(stats, 4 * rows, "stats"), _check(weight, dim, "weight")
    dr = None if dr is None else _check(dr, rows * dim, "dr")
    y = None if y is None else _check(y, rows * dim, "y")
    post_weight = None if post_weight is None else _check(post_weight, dim, "post_weight")
    gate = None if gate is None else _check(gate, groups * dim, "gate")

    like["x"] = shape
    if y is not None:
        like["y"] = shape

    def out(name):
        return torch.empty(like[name], dtype=torch.float32, device=r.device) if name in wanted and name in like else None

    g = NormGrads(out("x"), out("y"), out("weight"), out("bias"), out("post_weight"), out("gate"))
    L = _lib.lib()
    with _on(r.device):
        ws = _scratch(L.rgb200_block_norm_backward_workspace(rows, dim, groups), r.device)
        n = _lib.BlockNorm(rows, dim, groups, KINDS[kind], residual_scale, eps, _addr(r), _addr(y), _addr(weight), None, _addr(post_weight), _addr(gate),
                           _addr(r), None, _addr(stats), _addr(dr), _addr(dh), _addr(g.x), _addr(g.y), _addr(g.weight), _addr(g.bias),
                           _addr(g.post_weight), _addr(g.gate))
        rc = L.rgb200_block_norm_backward(C.byref(n), _addr(ws), ws.numel(), _raw_stream(r.device))
    if rc != cudaSuccess:
        raise ReproGemmError(rc, "block_norm_backward")
    return g
