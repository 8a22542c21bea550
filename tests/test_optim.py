"""AdamW over many tensors, on the CPU: argument checks of the C ABI (made before any device is touched), refusals of the
Python class, and the 8-bit codes' properties in the numpy restatement that the GPU tests compare with."""
import ctypes as C
import os

import numpy as np
import pytest
import torch

from bit_reproducible_training_b200 import _lib, repro_optim
from optim_restated import decode, encode

needs_lib = pytest.mark.skipif(not os.path.exists(_lib._build.LIB), reason="librgb200.so is not built")


def call(rows, count=None, fn="rgb200_adamw_step", **kw):
    h = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, step=1, device_step=None, state_bits=32)
    h.update(kw)
    hyper = _lib.AdamwHyper(*[h[n] for n, _ in _lib.AdamwHyper._fields_])
    args = [rows.ctypes.data if rows is not None else None, len(rows) if count is None else count]
    if fn == "rgb200_adamw_step":
        args.append(C.byref(hyper))
    return getattr(_lib.lib(), fn)(*args, None)


def rows(**kw):
    r = np.zeros(1, repro_optim._ROW)
    for n in ("param", "grad", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"):
        r[n] = 1 << 20                                   # never followed: every call here is refused
    r["count"] = 8
    for k, v in kw.items():
        r[k] = v
    return r


@needs_lib
@pytest.mark.parametrize("hyper", [dict(lr=-1.0), dict(lr=float("nan")), dict(beta1=1.0), dict(beta1=-0.1), dict(beta2=1.0),
                                   dict(beta2=float("nan")), dict(eps=-1e-9), dict(weight_decay=-0.1), dict(step=0), dict(state_bits=16)])
def test_hyper_parameters_are_checked(hyper):
    assert call(rows(), **hyper) == 1


@needs_lib
@pytest.mark.parametrize("field", ["param", "grad", "exp_avg", "exp_avg_sq"])
def test_null_tensors_are_refused(field):
    assert call(rows(**{field: 0})) == 1
    assert call(rows(count=-1)) == 1


@needs_lib
def test_scales_are_needed_with_codes_only():
    for field in ("exp_avg_scale", "exp_avg_sq_scale"):
        assert call(rows(**{field: 0}), state_bits=8) == 1
        for fn in ("rgb200_adamw_states_read", "rgb200_adamw_states_write"):
            assert call(rows(**{field: 0}), fn=fn) == 1
    assert call(None, count=1) == 1 and call(rows(), count=-1) == 1


def test_python_class_refuses_what_it_cannot_do():
    p = torch.nn.Parameter(torch.zeros(4))
    with pytest.raises(RuntimeError, match="no CPU path"):
        repro_optim.AdamW([p])
    with pytest.raises(ValueError):
        repro_optim.AdamW([p], state_bits=4)
    with pytest.raises(ValueError):
        repro_optim.AdamW([p], lr=-1.0)
    with pytest.raises(ValueError):
        repro_optim.AdamW([p], betas=(0.9, 1.0))
    with pytest.raises(TypeError):
        repro_optim.AdamW([torch.nn.Parameter(torch.zeros(4, dtype=torch.bfloat16))])


@pytest.mark.parametrize("n", [1, 255, 256, 257, 1000])
def test_codes_survive_a_second_coding(n):
    rng = np.random.default_rng(n)
    m = (rng.standard_normal(n) * 10.0 ** rng.uniform(-12, 2, n)).astype(np.float32)
    v = (m * m).astype(np.float32)
    codes = encode(m, v)
    again = encode(*decode(*codes))
    for a, b in zip(codes, again):
        assert np.array_equal(a, b)


def test_codes_are_the_nearest_ones_in_the_companded_domain():
    rng = np.random.default_rng(3)
    m = rng.standard_normal(2560).astype(np.float32)
    v = (rng.standard_normal(2560) ** 2).astype(np.float32)
    qm, sm, qv, sv = encode(m, v)
    x = np.sqrt(np.abs(m.astype(np.float64)) / np.repeat(sm, 256)) * np.sign(m) * 127
    y = (v / np.repeat(sv, 256).astype(np.float64)) ** 0.25 * 255
    # half a step, and the roundings of the quotient, the square roots and the product (at most four half-ulps of 255)
    slack = 4 * 255 * 2.0 ** -24
    assert np.abs(x - qm).max() <= 0.5 + slack
    assert np.abs(y - qv)[v > 0].max() <= 0.5 + slack
    assert ((qv > 0) | (v == 0)).all()
