"""block_norm_backward at the largest row count there is, 2^31 - 1, where a row index that runs ahead of the last row leaves 32 bits."""
import pytest
import torch

from bit_reproducible_training_b200 import repro_norm

pytestmark = pytest.mark.gpu

ROWS = 2 ** 31 - 1


def test_the_last_rows_of_the_longest_tensor():
    if torch.cuda.mem_get_info()[0] < 75 * 2 ** 30:
        pytest.skip("needs 75 GB")
    # rows of one value, and statistics that make the gradient d (1 - r^2) = 0.75 d exactly
    stats = torch.zeros(4, ROWS, device="cuda")
    stats[1] = 1.0
    r, dh = torch.full((ROWS, 1), 0.5, device="cuda"), torch.ones(ROWS, 1, device="cuda")
    dh[-3:, 0] = torch.tensor([2.0, 3.0, 4.0])
    try:
        got = repro_norm.block_norm_backward(dh, None, r, None, stats, weight=torch.ones(1, device="cuda"), wanted=("x",)).x
        assert torch.equal(got[-3:, 0].cpu(), torch.tensor([1.5, 2.25, 3.0]))
        for at in range(0, ROWS - 3, 2 ** 28):
            assert bool((got[at:min(at + 2 ** 28, ROWS - 3)] == 0.75).all())
    finally:
        del stats, r, dh
        got = None
        torch.cuda.empty_cache()
