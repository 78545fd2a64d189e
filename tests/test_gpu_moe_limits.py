"""Expert-layer operators (include/prefree_moe.h) at the ends of what they take, on the GPU: workspaces of exactly the size
that is asked for, and grids of more work items than one launch has."""
import numpy as np
import pytest
import torch

import prefree_amd as pf
from moe_util import DEV, NAN, route_reference

pytestmark = pytest.mark.gpu

GUARD = 1 << 16   # bytes behind a workspace, more than the sums of any size here


def routed(z, top_k, dtype, normalise=True):
    """What pf_moe_route writes with a workspace of exactly its size, whose neighbours behind it have to stay."""
    tokens, experts = z.shape
    size = pf.moe_route_workspace(tokens, experts)
    flat = torch.full((size + GUARD,), 0x5a, dtype=torch.uint8, device=DEV)
    out = {name: torch.full((tokens * top_k,), 77, dtype=torch.int32, device=DEV) for name in ("choice", "order", "slot")}
    out["weight"] = torch.full((tokens * top_k,), NAN, device=DEV)
    out["offsets"] = torch.full((experts + 1,), 77, dtype=torch.int32, device=DEV)
    pf.moe_route(z, tokens, experts, top_k, out["choice"], out["weight"], out["offsets"], out["order"], out["slot"], flat,
                 dtype=dtype, normalise=normalise, workspace_bytes=size)
    assert (flat[size:] == 0x5a).all(), "written behind the workspace"
    return out


@pytest.mark.parametrize("experts", [1, 2, 3, 5, 64])
@pytest.mark.parametrize("tokens", [65, 4097, 65536, 65537, 70001])
def test_route_stays_inside_its_workspace(tokens, experts):
    g = torch.Generator(device=DEV)
    g.manual_seed(tokens + experts)
    z = torch.randn(tokens, experts, generator=g, device=DEV)
    z[3::7] = -float("inf")
    top_k = min(2, experts)
    got = routed(z, top_k, "f32")
    ref = dict(zip(("choice", "weight", "offsets", "order", "slot"), route_reference(z.double().cpu().numpy(), top_k, True)))
    for name in ("choice", "offsets", "order", "slot"):
        assert np.array_equal(got[name].cpu().numpy(), ref[name].reshape(-1)), name
