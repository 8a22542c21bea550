"""block_norm on the CPU: refusals of the C ABI and of the Python functions, made before any device is touched."""
import ctypes as C
import os

import pytest
import torch

from bit_reproducible_training_b200 import _lib, layers, repro_norm

needs_lib = pytest.mark.skipif(not os.path.exists(_lib._build.LIB), reason="librgb200.so is not built")
HERE = 1 << 20            # an address that is never followed: every call here is refused


def norm(**kw):
    n = _lib.BlockNorm(4, 8, 1, 0, 1.0, 1e-5)
    for name in ("x", "weight", "h", "stats", "dh"):
        setattr(n, name, HERE)
    for k, v in kw.items():
        setattr(n, k, v)
    return n


BAD = [dict(rows=-1), dict(dim=0), dict(dim=8193), dict(groups=0), dict(groups=3, y=HERE, gate=HERE, r=HERE), dict(groups=2), dict(kind=2), dict(eps=-1e-6),
       dict(eps=float("nan")), dict(scale=float("nan")), dict(x=None), dict(weight=None), dict(post_weight=HERE), dict(gate=HERE), dict(y=HERE, r=None)]


@needs_lib
@pytest.mark.parametrize("bad", BAD, ids=str)
def test_forward_and_backward_refuse(bad):
    L = _lib.lib()
    n = norm(**bad)
    assert L.rgb200_block_norm_forward(C.byref(n), None) == 1
    assert L.rgb200_block_norm_backward(C.byref(n), HERE, 1 << 30, None) == 1


@needs_lib
def test_backward_checks_its_outputs_and_workspace():
    L = _lib.lib()
    need = L.rgb200_block_norm_backward_workspace(4, 8, 1)
    assert need >= 256 and L.rgb200_block_norm_backward_workspace(4, 9000, 1) == 0 and L.rgb200_block_norm_backward_workspace(4, 8, 3) == 0
    for bad, ws, size in ((dict(), None, need), (dict(), HERE, need - 1), (dict(), HERE + 4, need), (dict(dh=None), HERE, need), (dict(stats=None), HERE, need),
                          (dict(dy=HERE), HERE, need), (dict(dpost_weight=HERE), HERE, need), (dict(dgate=HERE), HERE, need)):
        n = norm(**bad)
        assert L.rgb200_block_norm_backward(C.byref(n), ws, size, None) == 1, (bad, ws, size)
    assert L.rgb200_block_norm_forward(None, None) == 1
    n = norm(h=None)
    assert L.rgb200_block_norm_forward(C.byref(n), None) == 1


def test_python_refusals():
    x, w = torch.zeros(6, 8), torch.ones(8)
    for bad in (dict(kind="batch"), dict(eps=-1.0), dict(gate=w), dict(post_weight=w), dict(y=torch.zeros(6, 4)), dict(y=x, gate=torch.ones(4, 8)),
                dict(y=x, gate=torch.ones(7)), dict(y=x, gate=torch.ones(1, 1, 8))):
        with pytest.raises(ValueError):
            repro_norm.block_norm(x, bad.pop("y", None), weight=w, **bad)
    with pytest.raises(ValueError):
        repro_norm.block_norm(torch.zeros(2, 9000), weight=torch.ones(9000))
    with pytest.raises(RuntimeError, match="no CPU path"):
        repro_norm.block_norm(x, weight=w)
    with pytest.raises(TypeError):
        repro_norm.block_norm(x.double(), weight=w)
    with pytest.raises(ValueError):
        layers.BlockNorm(8, kind="batch")
