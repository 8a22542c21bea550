"""The linear cross entropy on the CPU: refusals of the C ABI and of the Python functions, made before any device is touched, and the
workspace's size."""
import os

import pytest
import torch

from bit_reproducible_training_b200 import _lib, layers, repro_loss

needs_lib = pytest.mark.skipif(not os.path.exists(_lib._build.LIB), reason="librgb200.so is not built")
HERE = 1 << 20            # an address that is never followed: every call here is refused


def forward(**kw):
    a = dict(X=HERE, W=HERE, target=HERE, ignore=-100, reduction=1, N=4, V=10, D=8, S=3, loss=HERE, nll=HERE, lse=HERE, tl=HERE, inv=HERE, ws=HERE, size=1 << 40)
    a.update(kw)
    return _lib.lib().rgb200_linear_xent_forward(*a.values(), None)


def backward(**kw):
    a = dict(X=HERE, W=HERE, target=HERE, ignore=-100, reduction=1, N=4, V=10, D=8, S=3, lse=HERE, tl=HERE, inv=HERE, dloss=HERE, dX=HERE, dW=HERE, ws=HERE, size=1 << 40)
    a.update(kw)
    return _lib.lib().rgb200_linear_xent_backward(*a.values(), None)


@needs_lib
@pytest.mark.parametrize("bad", [dict(X=None), dict(W=None), dict(target=None), dict(N=0), dict(V=0), dict(V=(1 << 30) + 1), dict(N=(1 << 30) + 1), dict(D=0), dict(S=0), dict(S=4), dict(D=200000), dict(reduction=3),
                                 dict(reduction=-1), dict(ws=None), dict(ws=HERE + 16), dict(size=100), dict(lse=None), dict(tl=None), dict(inv=None)], ids=str)
def test_both_calls_refuse(bad):
    assert forward(**bad) == 1 and backward(**bad) == 1


@needs_lib
def test_each_call_refuses_its_own():
    assert forward(nll=None) == 1 and forward(loss=None) == 1
    assert backward(dloss=None) == 1 and backward(dX=None, dW=None) == 1


@needs_lib
def test_workspace_stays_below_the_logits():
    L = _lib.lib()
    for n, v, d in ((8192, 50257, 768), (32768, 50257, 768), (1024, 200000, 512)):
        f, b = L.rgb200_linear_xent_workspace(n, v, d, 3, 0), L.rgb200_linear_xent_workspace(n, v, d, 3, 1)
        # statistics and digit planes forward; backward one piece of P in FP32 and its planes for two products
        assert 0 < f < n * v and 0 < b < 4 * n * v
    assert L.rgb200_linear_xent_workspace(0, 10, 8, 3, 0) == 0 and L.rgb200_linear_xent_workspace(4, 10, 8, 5, 1) == 0


def test_python_refusals():
    x, w, t = torch.zeros(6, 8), torch.zeros(10, 8), torch.zeros(6, dtype=torch.int64)
    for call in (repro_loss.linear_cross_entropy, layers.linear_cross_entropy):
        with pytest.raises(ValueError):
            call(x, w, t, reduction="max")
        with pytest.raises(ValueError):
            call(x, w.t(), t)
        with pytest.raises(ValueError):
            call(x, w, t[:5])
        with pytest.raises(TypeError):
            call(x, w, t.int())
        with pytest.raises(RuntimeError, match="no CPU path"):
            call(x, w, t)
    with pytest.raises(ValueError):
        layers.LinearCrossEntropy(8, 10, reduction="max")
