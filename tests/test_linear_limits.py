"""Sizes next to 2^31 in the backward pass of an activation: the indexes and the ranges' arithmetic must stay within 32 bits."""
import os

import pytest
import torch

from bit_reproducible_training_b200 import _lib
from bit_reproducible_training_b200 import repro_gemm as rg

HERE = 1 << 20            # an address that is never followed: every call here is refused


@pytest.mark.skipif(not os.path.exists(_lib._build.LIB), reason="librgb200.so is not built")
def test_the_c_calls():
    L = _lib.lib()
    for rows in (2 ** 31 - 4096, 2 ** 31 - 900, 2 ** 31 - 32, 2 ** 31 - 1):
        assert L.rgb200_activation_backward_workspace(rows, 1) == 0 and L.rgb200_linear_backward_workspace(rows, 1, 1, 0, 1) == 0
        for dz, db in ((HERE, None), (None, HERE), (HERE, HERE)):
            assert L.rgb200_activation_backward(HERE, HERE, dz, db, rows, 1, 2, HERE, 1 << 60, None) == 1, rows
            assert L.rgb200_activation_backward(HERE, HERE, dz, db, 1, rows, 2, HERE, 1 << 60, None) == 1, rows
    # 888 ranges of a column for one strip of columns
    assert L.rgb200_activation_backward_workspace(2 ** 31 - 4097, 1) == 888 * 4 and L.rgb200_activation_backward_workspace(10 ** 6, 128) == 888 * 128 * 4


def test_the_python_function():
    t = torch.zeros(1)
    for rows in (2 ** 31 - 4096, 2 ** 31 - 1):
        with pytest.raises(ValueError, match="2\\^31"):
            rg.activation_backward(t.expand(rows), t.expand(rows), rows, 1, "silu")
        with pytest.raises(ValueError, match="2\\^31"):
            rg.activation_backward(t.expand(rows), t.expand(rows), 1, rows, "silu")
