"""The workspace of block_norm_backward over the whole range of row counts: as many bytes as there are row ranges, whose count stays small."""
import os

import pytest

from bit_reproducible_training_b200 import _lib

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
