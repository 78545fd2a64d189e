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


# ---- more work items than one launch has (2^32) -------------------------------------------------------------------

@pytest.fixture(autouse=True)
def give_back_memory():
    yield
    torch.cuda.empty_cache()


def test_route_past_a_launch():
    """1024 work items take 64 tokens: one launch ends at 2^28 tokens."""
    tokens, experts = (1 << 28) + 65, 2
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    z = torch.empty(tokens, experts, dtype=torch.float16, device=DEV).normal_(generator=g)
    z[3::16] = -float("inf")
    got = routed(z, 1, "f16")
    best = (z[:, 1] > z[:, 0]).int()
    best[z[:, 0] == -float("inf")] = -1          # in rows of which both are
    assert torch.equal(got["choice"], best)
    assert torch.equal(got["weight"], (best >= 0).float())
    del z
    which = [torch.nonzero(best == e)[:, 0].int() for e in range(experts)]
    counts = [w.numel() for w in which]
    used = sum(counts)
    assert got["offsets"].tolist() == [0, counts[0], used]
    assert torch.equal(got["order"][:used], torch.cat(which)) and (got["order"][used:] == -1).all()
    slot = torch.full((tokens,), -1, dtype=torch.int32, device=DEV)
    slot[got["order"][:used].long()] = torch.arange(used, dtype=torch.int32, device=DEV)
    assert torch.equal(got["slot"], slot)


def test_route_backward_past_a_launch():
    """A wave a token: one launch ends at 2^26 tokens."""
    tokens, experts = (1 << 26) + 5, 2
    g = torch.Generator(device=DEV)
    g.manual_seed(2)
    z = torch.randn(tokens, experts, generator=g, device=DEV)
    choice = (z[:, 1] > z[:, 0]).int()
    weight = torch.sigmoid((z[:, 1] - z[:, 0]).abs())          # of the larger, over both
    dweight = torch.randn(tokens, generator=g, device=DEV)
    dz = torch.full_like(z, NAN)
    pf.moe_route_backward(z, tokens, experts, 1, choice, weight, dweight, dz, normalise=False)
    # d weight / d z = w (1 - w) for the chosen and the opposite for the other.  A dozen fp32 roundings of numbers of up to
    # |dweight|, and of an exponential of up to 20: (12 + 20) 2^-23.
    want = weight.double() * (1 - weight.double()) * dweight.double()
    want = torch.where(choice == 1, want, -want)
    room = 32 * 2.0 ** -23 * dweight.double().abs() + 2.0 ** -126
    for column, sign in ((1, 1), (0, -1)):
        assert ((dz[:, column].double() - sign * want).abs() <= room).all()


def test_combine_past_a_launch():
    """A wave a token of up to 512 columns: one launch ends at 2^26 tokens."""
    tokens = (1 << 26) + 5
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    y = torch.empty(tokens, 1, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    weight = torch.randn(tokens, generator=g, device=DEV)
    slot = torch.arange(tokens - 1, -1, -1, dtype=torch.int32, device=DEV)
    slot[::1000] = -1
    out = torch.full((tokens, 1), 7.0, dtype=torch.bfloat16, device=DEV)
    pf.moe_combine(y, slot, weight, tokens, 1, 1, out)
    want = torch.where(slot >= 0, weight * y.flip(0)[:, 0].float(), 0.0).bfloat16()   # one product, rounded to fp32 and to bf16
    assert torch.equal(out[:, 0], want)


def test_combine_backward_past_a_launch():
    """A workgroup a token: one launch ends at 2^24 tokens."""
    tokens, width = (1 << 24) + 9, 3
    g = torch.Generator(device=DEV)
    g.manual_seed(4)
    y, dout = (torch.empty(tokens, width, dtype=torch.float16, device=DEV).normal_(generator=g) for _ in range(2))
    weight = torch.randn(tokens, generator=g, device=DEV)
    slot = torch.arange(tokens - 1, -1, -1, dtype=torch.int32, device=DEV)
    dy, dweight = torch.full_like(y, 7.0), torch.full((tokens,), NAN, device=DEV)
    pf.moe_combine_backward(dout, y, slot, weight, tokens, 1, width, dy, dweight, dtype="f16")
    assert torch.equal(dy, (weight[:, None] * dout.float()).half().flip(0))
    terms = dout.double() * y.flip(0).double()
    assert ((dweight.double() - terms.sum(1)).abs() <= (width + 2) * 2.0 ** -23 * terms.abs().sum(1)).all()


# With k = 1 a product of 16-bit numbers has one term, which fp32 holds exactly: it is rounded once, as torch rounds it.

def outer(x, w, out, rows):
    """Whether out [experts * rows, n] is x [experts * rows] times w [experts, n] of its expert."""
    for e in range(w.shape[0]):
        at = slice(e * rows, (e + 1) * rows)
        if not torch.equal(out[at], x[at, None] * w[e][None]):
            return False
    return True


@pytest.mark.parametrize("rows,n", [(2, (1 << 18) + 5), (5, (1 << 21) + 9)])
def test_mm_past_a_launch(rows, n):
    """16 x 16 tiles (two rows an expert) and 128 x 128 tiles (five) of 256 work items: one launch ends at 2^24 tiles."""
    experts, dtype = 1024, torch.bfloat16
    assert experts * -(-n // (16 if rows == 2 else 128)) > 1 << 24
    g = torch.Generator(device=DEV)
    g.manual_seed(5)
    x = torch.empty(experts * rows, 1, dtype=dtype, device=DEV).normal_(generator=g)
    w = torch.empty(experts, n, 1, dtype=dtype, device=DEV).normal_(generator=g)
    y = torch.full((experts * rows, n), 7.0, dtype=dtype, device=DEV)
    off = torch.arange(0, experts * rows + 1, rows, dtype=torch.int32, device=DEV)
    pf.moe_mm(x, experts * rows, None, 1, w, off, experts, experts * rows, n, 1, y)
    assert outer(x[:, 0], w[:, :, 0], y, rows)


def test_mm_dw_past_a_launch():
    """256 x 256 tiles of 512 work items: one launch ends at 2^23 tiles."""
    experts, n, dtype = 1024, (1 << 21) + 300, torch.bfloat16
    assert experts * -(-n // 256) > 1 << 23
    g = torch.Generator(device=DEV)
    g.manual_seed(6)
    x = torch.empty(experts, 1, dtype=dtype, device=DEV).normal_(generator=g)
    dy = torch.empty(experts, n, dtype=dtype, device=DEV).normal_(generator=g)
    dw = torch.full((experts, n, 1), 7.0, dtype=dtype, device=DEV)
    off = torch.arange(experts + 1, dtype=torch.int32, device=DEV)
    pf.moe_mm_dw(dy, x, experts, None, 1, off, experts, experts, n, 1, dw)
    assert outer(x[:, 0], dy, dw[:, :, 0], 1)


def test_mm_mx4_past_a_launch():
    """4-bit operands behind 4 GiB, by 16 x 16 tiles of 256 work items: one launch ends at 2^32 results."""
    k, n, slots, experts = 64, 2064, 1 << 21, 3
    x_rows = (1 << 27) + 100
    g = torch.Generator(device=DEV)
    g.manual_seed(7)
    codes = torch.randint(0, 256, (x_rows, k // 2), generator=g, device=DEV, dtype=torch.uint8)
    w_codes = torch.randint(0, 256, (experts * n, k // 2), generator=g, device=DEV, dtype=torch.uint8)
    scales, w_scales = (torch.full((v, k // 32), 127, dtype=torch.uint8, device=DEV) for v in (x_rows, experts * n))
    rows = torch.randint(0, x_rows, (slots,), generator=g, device=DEV).int()
    rows[::2] = x_rows - 1 - rows[::2] % 1000
    bounds = [0, 700001, 700001, slots]
    y = torch.full((slots, n), 7.0, dtype=torch.bfloat16, device=DEV)
    off = torch.tensor(bounds, dtype=torch.int32, device=DEV)
    pf.moe_mm_mx4(codes, scales, x_rows, rows, 1, w_codes, w_scales, off, experts, slots, n, k, y)
    w = torch.empty(experts * n, k, device=DEV)
    pf.mx4_dequantize(w_codes, w_scales, experts * n, k, w)
    w = w.view(experts, n, k)
    # all products are multiples of 1/4 of at most 36, so that fp32 holds their sums exactly in any order
    for e in range(experts):
        for b in range(bounds[e], bounds[e + 1], 1 << 18):
            f = min(b + (1 << 18), bounds[e + 1])
            at = rows[b:f].long()
            x = torch.empty(f - b, k, device=DEV)
            pf.mx4_dequantize(codes[at], scales[at], f - b, k, x)
            assert torch.equal(y[b:f], (x @ w[e].t()).bfloat16()), (e, b)
