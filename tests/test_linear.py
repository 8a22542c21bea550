"""The fused linear layer on the CPU: refusals of the C ABI and of the Python functions, made before any device is touched."""
import ctypes as C
import os

import pytest
import torch

from bit_reproducible_training_b200 import _lib, layers
from bit_reproducible_training_b200 import repro_gemm as rg

needs_lib = pytest.mark.skipif(not os.path.exists(_lib._build.LIB), reason="librgb200.so is not built")
HERE = 1 << 20            # an address that is never followed: every call here is refused


def epilogue(A=HERE, B=HERE, Cout=HERE, act=0, cfg=True, e=True):
    c, ep = _lib.Config(1, 16, 16, 32, 0, 3, 0, 1), _lib.Epilogue(None, None, None, act)
    return _lib.lib().rgb200_gemm_epilogue_fp32_ws(A, B, Cout, 4, 8, 16, C.byref(c) if cfg else None, C.byref(ep) if e else None, HERE, 1 << 30, None)


@needs_lib
@pytest.mark.parametrize("bad", [dict(A=None), dict(B=None), dict(Cout=None), dict(act=-1), dict(act=5), dict(cfg=False), dict(e=False)], ids=str)
def test_epilogue_refuses(bad):
    assert epilogue(**bad) == 1


@needs_lib
def test_activation_backward_refuses():
    f = _lib.lib().rgb200_activation_backward
    need = _lib.lib().rgb200_activation_backward_workspace(4, 8)
    good = dict(dY=HERE, Z=HERE, dZ=HERE, db=HERE, M=4, N=8, act=2, ws=HERE, size=need)
    for bad in (dict(dY=None), dict(Z=None), dict(dZ=None, db=None), dict(M=-1), dict(N=0), dict(act=5), dict(act=-1), dict(ws=None), dict(size=need - 1)):
        assert f(*{**good, **bad}.values(), None) == 1, bad
    assert _lib.lib().rgb200_activation_backward_workspace(4, 0) == 0


@needs_lib
def test_linear_backward_refuses():
    L = _lib.lib()
    need = L.rgb200_linear_backward_workspace(4, 8, 16, 2, 3)
    assert need > 0 and L.rgb200_linear_backward_workspace(0, 8, 16, 2, 3) == 0 and L.rgb200_linear_backward_workspace(4, 8, 16, 9, 3) == 0
    good = dict(dY=HERE, Z=HERE, X=HERE, W=HERE, dX=HERE, dW=HERE, db=HERE, M=4, N=8, K=16, act=2, S=3, ws=HERE, size=need)
    for bad in (dict(dY=None), dict(Z=None), dict(X=None), dict(W=None), dict(dX=None, dW=None, db=None), dict(M=0), dict(N=0), dict(K=0), dict(act=5), dict(S=0),
                dict(S=4), dict(ws=None), dict(ws=HERE + 64), dict(size=need - 1)):
        assert L.rgb200_linear_backward(*{**good, **bad}.values(), None) == 1, bad


def test_python_refusals():
    x, w, b = torch.zeros(6, 8), torch.zeros(10, 8), torch.zeros(10)
    for bad in (dict(activation="tanh"), dict(bias=b[:9]), dict(residual=torch.zeros(5, 10))):
        with pytest.raises(ValueError):
            layers.linear(x, w, **bad)
    with pytest.raises(ValueError):
        layers.linear(x, w.t())
    with pytest.raises(RuntimeError, match="no CPU path"):
        layers.linear(x, w, b)
    with pytest.raises(TypeError):
        layers.linear(x.double(), w, b)
    with pytest.raises(ValueError):
        layers.FusedLinear(8, 10, activation="swish")
    with pytest.raises(ValueError):
        rg.linear_backward(torch.zeros(6, 10), None, x, w, 6, 10, 8, "elu")
