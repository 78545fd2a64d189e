"""SpMV with more work items than one launch has (2^32), on the GPU."""
import pytest
import torch

import prefree_amd as pf
from gpu_util import DEV

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,tile", [((1 << 27) + 9, 32), ((1 << 28) + 300, 16)])
def test_row_groups_past_a_launch(m, tile):
    """`tile` lanes a row: one launch ends at 2^32 / tile rows."""
    n, every = 1000, 64
    rp = (torch.arange(m + 1, dtype=torch.int32, device=DEV) + (every - 1)) // every   # one entry in every 64th row
    nnz = int(rp[-1])
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    col = torch.randint(0, n, (nnz,), generator=g, device=DEV, dtype=torch.int32)
    val, x = torch.randn(nnz, generator=g, device=DEV), torch.randn(n, generator=g, device=DEV)
    y = torch.full((m,), float("nan"), device=DEV)
    stream = torch.cuda.current_stream()
    with pf.Plan(rp, col, m, n, nnz, "f32", "flat", tile, stream=stream) as p:
        p.execute(rp, col, val, x, y, stream=stream)
        torch.cuda.synchronize()
        p.check(stream=stream)
    assert torch.equal(y[::every], val * x[col.long()])   # a row's one product, rounded once
    y[::every] = 0
    assert (y == 0).all()
    torch.cuda.empty_cache()
