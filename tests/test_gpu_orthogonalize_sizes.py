"""Orthogonal updates at sizes where a kernel goes several ways: each matrix of a batch against the same steps in 64 bits, at the
bounds of include/prefree_moe.h (test_gpu_orthogonalize_bounds.py says what they rest on)."""
import pytest
import torch

from moe_util import ROUND
from test_gpu_orthogonalize import momentum, reference, run
from test_gpu_orthogonalize_bounds import off

pytestmark = pytest.mark.gpu


def check(batch, rows, columns, bound):
    for flip in (False, True):
        g = momentum(batch, rows, columns, batch + rows)
        got, held = run(g.transpose(1, 2).contiguous() if flip else g, "f32", "f16")
        assert off(got, reference(held)) <= bound + ROUND["f16"]


# More than eight blocks of 32 columns a share: waves take several, the next one's pieces on their way while one is stored.  128
# matrices have two shares, of 61 and 33 blocks; 300 have one, of 22, 200 one of 9, of which the last is cut, and 4 have 64 of 9.
@pytest.mark.parametrize("batch,rows,columns", [(128, 37, 3871), (128, 64, 2100), (300, 33, 700), (200, 64, 260), (4, 50, 16500)])
def test_several_blocks_a_wave(batch, rows, columns):
    check(batch, rows, columns, 2.0 ** -11)


# Tiles of 256 x 256 with a last round in quarters: 16 x 2048 x 2048 has 576 tiles of A and B, the last 64 with diagonal ones; 17 x
# 1500 x 1800 also 816 of X', 48 in quarters, of which the last rows' and columns' are cut or not there.
@pytest.mark.parametrize("batch,rows,columns", [(16, 2048, 2048), (17, 1500, 1800)])
def test_a_last_round_in_quarters(batch, rows, columns):
    check(batch, rows, columns, 2.0 ** -8)


# X' of 129 to 192 rows in tiles of 64 x 128, more than compute units
@pytest.mark.parametrize("batch,rows,columns", [(96, 139, 2765), (40, 180, 1400), (24, 192, 2048)])
def test_three_tiles_of_64_rows(batch, rows, columns):
    check(batch, rows, columns, 2.0 ** -8)


def test_one_matrix_of_many_is_not_a_number():
    """In quarters and in several blocks a wave, too, the others do not see it."""
    for batch, rows, columns in ((16, 2048, 2048), (200, 64, 260), (40, 139, 1400)):
        g = momentum(batch, rows, columns, 3)
        want, _ = run(g)
        g[batch - 2, rows - 1, columns - 1] = float("inf")
        got, _ = run(g)
        assert got[batch - 2].isnan().all()
        others = torch.arange(batch, device=g.device) != batch - 2
        assert torch.equal(got[others], want[others])
