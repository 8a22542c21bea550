"""The workspace of block_norm_backward over the whole range of row counts: as many bytes as there are row ranges, whose count stays small."""
import ctypes as C
import os

import pytest
import torch

from bit_reproducible_training_b200 import _lib, repro_norm

pytestmark = pytest.mark.skipif(not os.path.exists(_lib._build.LIB), reason="librgb200.so is not built")


@pytest.mark.parametrize("dim,threads", [(1, 32), (300, 64), (1000, 128), (4096, 512), (8192, 1024)])
def test_workspace_of_any_row_count(dim, threads):
    need = _lib.lib().rgb200_block_norm_backward_workspace
    assert need(0, dim, 1) == 256
    most = 148 * max(1, 512 // threads)
    for rows in (1, 7, 8, 9, 4095, 10 ** 6, 2 ** 30, 2 ** 31 - 10 ** 6, 2 ** 31 - 9, 2 ** 31 - 8, 2 ** 31 - 1):
        ranges = min(most, -(-rows // 8))
        length = -(-rows // ranges)
        assert need(rows, dim, 1) == max(256, -(-rows // length) * 3 * dim * 4), rows


def test_a_gate_of_too_many_rows():
    """Above 2^30 the strides of the sums over the gate's rows would leave 32 bits."""
    L, rows = _lib.lib(), 2 ** 30 + 64
    here = 1 << 20            # never followed
    n = _lib.BlockNorm(rows, 1, rows, 0, 1.0, 1e-5)
    for name in ("x", "y", "weight", "gate", "r", "h", "stats", "dh"):
        setattr(n, name, here)
    assert L.rgb200_block_norm_backward_workspace(rows, 1, rows) == 0 and L.rgb200_block_norm_backward_workspace(2 ** 30, 1, 2 ** 30) == 3 * 4 * 2 ** 30
    assert L.rgb200_block_norm_forward(C.byref(n), None) == 1 and L.rgb200_block_norm_backward(C.byref(n), here, 1 << 50, None) == 1
    x = torch.zeros(1).expand(rows, 1)
    with pytest.raises(ValueError, match="2\\^30"):
        repro_norm.block_norm(x, x, weight=torch.ones(1), gate=x)
