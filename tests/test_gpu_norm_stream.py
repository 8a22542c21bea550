"""block_norm_backward where the residual stream passes by a norm without a block's output: r is x itself, and the gradient that reaches it
from elsewhere (dr) belongs to dx.  Bounds as in norm_restated.py: the addition of dr is one more rounding."""
import pytest
import torch

import norm_restated as ref
from bit_reproducible_training_b200 import repro_norm

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1), (5, 3), (3, 33), (7, 100), (9, 256), (11, 768), (4, 1001), (3, 2304), (2, 4096), (2, 5000), (2, 8192), (700, 64), (0, 40)]


def tensors(rows, dim, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 10007 + dim)
    x, dh, dr = (torch.randn(rows, dim, device="cuda", generator=g) for _ in range(3))
    return x + 0.3, dh, dr, torch.randn(dim, device="cuda", generator=g) * 0.2 + 1.0, torch.randn(dim, device="cuda", generator=g)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,dim", SHAPES)
def test_the_streams_gradient_without_a_block(rows, dim, kind):
    if kind == "layer" and dim == 1:
        pytest.skip("a row of one value has no deviation")
    x, dh, dr, w, b = tensors(rows, dim)
    # the scale belongs to r = scale x + ..., which is not formed without y
    how = dict(weight=w, bias=b, kind=kind, eps=1e-5, residual_scale=0.75)
    r, h, stats = repro_norm.block_norm(x, keep_stats=True, **how)
    got = repro_norm.block_norm_backward(dh, dr, r, None, stats, **how)
    bare = repro_norm.block_norm_backward(dh, None, r, None, stats, **how)
    # the column sums do not know dr, and a stream without a gradient changes nothing
    assert torch.equal(got.weight, bare.weight) and torch.equal(got.bias, bare.bias)
    zero = repro_norm.block_norm_backward(dh, torch.zeros_like(dr), r, None, stats, **how)
    assert torch.equal(zero.x, bare.x) and torch.equal(zero.weight, bare.weight)
    if rows == 0:
        return
    s = ref.forward(x.double(), None, w.double(), b.double(), None, None, 0.75, kind, 1e-5)
    want, bound = ref.backward(s, dh.double(), None, w.double(), b.double(), None, None, 0.75, kind)["x"]
    want = want + dr.double()
    over = (got.x.double() - want).abs() - (bound + ref.U * want.abs())
    assert torch.isfinite(got.x).all() and float(over.max()) <= 0.0


def test_only_dx_is_asked_for_and_unaligned():
    x, dh, dr, w, b = tensors(9, 132)
    how = dict(weight=w, bias=b, kind="layer")
    r, h, stats = repro_norm.block_norm(x, keep_stats=True, **how)
    want = repro_norm.block_norm_backward(dh, dr, r, None, stats, **how).x
    got = repro_norm.block_norm_backward(dh, dr, r, None, stats, wanted=("x",), **how)
    assert torch.equal(got.x, want) and got.weight is None and got.bias is None
    flat = torch.empty(dr.numel() + 1, device="cuda")
    flat[1:] = dr.view(-1)
    assert torch.equal(repro_norm.block_norm_backward(dh, flat[1:].view_as(dr), r, None, stats, **how).x, want)
