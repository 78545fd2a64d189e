"""Expert-layer operators (include/prefree_moe.h) on the GPU against plain 64-bit forms (moe_util.py)."""
import numpy as np
import pytest
import torch

import prefree_amd as pf
from moe_util import DEV, NAN, ROUND, TORCH, close, groups, offsets_of, product, route_reference, strided, swiglu

pytestmark = pytest.mark.gpu


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype="f32"):
    return torch.randn(*shape, generator=g, device=DEV).to(TORCH[dtype])


# ---- routing ---------------------------------------------------------------------------------------------------

def logits_for(tokens, experts, dtype, kind, seed):
    g = gen(seed)
    z = torch.randn(tokens, experts, generator=g, device=DEV) * 2
    if kind == "masked":
        z[torch.rand(tokens, experts, generator=g, device=DEV) < 0.4] = -float("inf")
        z[3::5] = -float("inf")
    elif kind == "ties":
        z = torch.round(z)
    elif kind == "equal":
        z[:] = 0.0
        z[::2, ::3] = -0.0
    elif kind == "lowest":        # the type's lowest finite value is a number: chosen when nothing else is left
        z[torch.rand(tokens, experts, generator=g, device=DEV) < 0.8] = torch.finfo(TORCH[dtype]).min
    elif kind == "special":
        z[torch.rand(tokens, experts, generator=g, device=DEV) < 0.1] = NAN
        z[torch.rand(tokens, experts, generator=g, device=DEV) < 0.1] = float("inf")
        z[torch.rand(tokens, experts, generator=g, device=DEV) < 0.2] = -float("inf")
    return z.to(TORCH[dtype])


def route(z, top_k, dtype, normalise=True, ld=0):
    tokens, experts = z.shape
    n = max(1, tokens * top_k)
    out = {"choice": torch.full((n,), 77, dtype=torch.int32, device=DEV),
           "weight": torch.full((n,), NAN, device=DEV), "offsets": torch.full((experts + 1,), 77, dtype=torch.int32, device=DEV),
           "order": torch.full((n,), 77, dtype=torch.int32, device=DEV), "slot": torch.full((n,), 77, dtype=torch.int32, device=DEV)}
    work = torch.full((pf.moe_route_workspace(tokens, experts) // 4 + 1,), 0x7f7f7f7f, dtype=torch.int32, device=DEV)
    pf.moe_route(z, tokens, experts, top_k, out["choice"], out["weight"], out["offsets"], out["order"], out["slot"], work,
                 dtype=dtype, normalise=normalise, ld_logits=ld)
    return out


def check_route(z, top_k, dtype, normalise, ld=0):
    tokens, experts = z.shape
    got = route(z, top_k, dtype, normalise, ld)
    z64 = z.double().cpu().numpy()
    ref = dict(zip(("choice", "weight", "offsets", "order", "slot"), route_reference(z64, top_k, normalise)))
    for name in ("choice", "offsets", "order", "slot"):
        assert np.array_equal(got[name].cpu().numpy()[:ref[name].size], ref[name].reshape(-1)), name
    # exp of a difference d is off by about (|d| + 2) 2^-24, a sum of E terms by E 2^-24, the quotient by one more
    weight = got["weight"].cpu().numpy()[:ref["weight"].size].reshape(ref["weight"].shape)
    with np.errstate(all="ignore"):
        spread = np.nan_to_num(np.where(np.isfinite(z64), np.abs(z64), 0).max(initial=0))
    tol = (experts + 16 + min(2 * spread, 200)) * 2.0 ** -23
    with np.errstate(all="ignore"):
        ok = (np.abs(weight - ref["weight"]) <= tol * np.abs(ref["weight"]) + 2.0 ** -126) | (np.isnan(weight) & np.isnan(ref["weight"]))
    assert ok.all(), (weight[~ok][:3], ref["weight"][~ok][:3])
    return got


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind", ["plain", "masked", "ties", "equal", "lowest", "special"])
@pytest.mark.parametrize("tokens,experts,top_k", [(1, 64, 8), (1, 1, 1), (2, 3, 3), (63, 65, 2), (64, 8, 2), (65, 128, 8), (130, 60, 4)])
def test_route(tokens, experts, top_k, kind, dtype):
    for normalise in (True, False):
        check_route(logits_for(tokens, experts, dtype, kind, tokens + experts), top_k, dtype, normalise)


@pytest.mark.parametrize("tokens,experts,top_k", [(5000, 33, 6), (3001, 256, 16), (1111, 1000, 5), (777, 1024, 16), (500, 300, 1)])
def test_route_many_experts(tokens, experts, top_k):
    for kind in ("plain", "masked"):
        check_route(logits_for(tokens, experts, "f32", kind, 7), top_k, "f32", kind == "plain")


@pytest.mark.parametrize("tokens", [65536, 65537, 70001])
def test_route_beyond_a_thousand_blocks(tokens):
    check_route(logits_for(tokens, 9, "bf16", "masked", 3), 2, "bf16", True)


def test_route_strided_and_empty():
    z = logits_for(100, 20, "bf16", "masked", 5)
    view, ld = strided(z, ld=37, shift=1)
    check_route(view, 3, "bf16", True, ld=ld)
    got = route(torch.empty(0, 12, device=DEV), 2, "f32")
    assert got["offsets"].cpu().tolist() == [0] * 13 and got["order"][0] == 77


def test_route_all_rows_masked():
    z = torch.full((70, 16), -float("inf"), device=DEV)
    got = check_route(z, 4, "f32", False)
    assert got["offsets"].abs().sum() == 0 and (got["order"] == -1).all() and (got["weight"] == 0).all()


def route_loss(z, choice, dweight, normalise):
    """sum of dweight * weight in 64 bits, for a fixed choice (-1: none)."""
    taken = choice >= 0
    e = torch.exp(z - torch.where(torch.isfinite(z), z, torch.tensor(-1e30, dtype=z.dtype)).amax(1, keepdim=True).clamp(min=-1e29))
    top = torch.where(taken, torch.gather(e, 1, choice.clamp(min=0).long()), torch.zeros((), dtype=z.dtype))
    total = top.sum(1, keepdim=True) if normalise else e.sum(1, keepdim=True)
    return (dweight * torch.where(total > 0, top / total.clamp(min=1e-300), torch.zeros((), dtype=z.dtype))).sum()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("normalise", [True, False])
@pytest.mark.parametrize("tokens,experts,top_k,kind", [(1, 64, 8, "plain"), (37, 5, 2, "masked"), (130, 128, 8, "masked"),
                                                       (50, 200, 16, "plain"), (20, 700, 3, "masked"), (9, 1, 1, "plain")])
def test_route_backward(tokens, experts, top_k, kind, normalise, dtype):
    z = logits_for(tokens, experts, dtype, kind, 11)
    got = route(z, top_k, dtype, normalise)
    dweight = randn(gen(4), tokens, top_k)
    view, ld = strided(torch.empty(tokens, experts, dtype=TORCH[dtype], device=DEV), ld=experts + 3, shift=1, fill=5.0)
    pf.moe_route_backward(z, tokens, experts, top_k, got["choice"], got["weight"], dweight, view, dtype=dtype,
                          normalise=normalise, ld_dlogits=ld)
    choice = got["choice"].cpu().view(tokens, top_k)
    z64, dw64 = z.double().cpu(), dweight.double().cpu()
    leaf = z64.clone().requires_grad_()
    finite = torch.isfinite(z64)
    # the formula, by differentiating the 64-bit form (rows of -infinity apart: their gradient is 0)
    safe = torch.where(finite, leaf, torch.full((), -1e4, dtype=torch.float64))
    e = torch.exp(safe - safe.amax(1, keepdim=True).detach())
    e = torch.where(finite, e, torch.zeros((), dtype=torch.float64))
    taken = choice >= 0
    top = torch.where(taken, torch.gather(e, 1, choice.clamp(min=0).long()), torch.zeros((), dtype=torch.float64))
    total = (top if normalise else e).sum(1, keepdim=True)
    loss = (dw64 * top / torch.where(total > 0, total, torch.ones((), dtype=torch.float64))).sum()
    ref = torch.autograd.grad(loss, leaf)[0]
    size = (dw64.abs() * got["weight"].double().cpu().view(tokens, top_k)).sum(1, keepdim=True) + dw64.abs().amax(1, keepdim=True)
    # weights within (E + 40) 2^-23 as in check_route, carried through products and a sum of top_k terms
    close(view.cpu(), ref, (experts + top_k + 64) * 2.0 ** -23 * size, dtype, "dlogits")
    # and by differences: along a direction that leaves the choice alone
    if normalise or kind == "plain":
        g = torch.Generator().manual_seed(1)
        way = torch.where(finite, torch.randn(tokens, experts, generator=g, dtype=torch.float64), torch.zeros((), dtype=torch.float64))
        h = 1e-5
        slope = (route_loss(z64 + h * way, choice, dw64, normalise) - route_loss(z64 - h * way, choice, dw64, normalise)) / (2 * h)
        along = (view.double().cpu() * way).sum()
        # each element rounded to its type, plus the difference's own error h^2 and cancellation 1e-16 / h
        tol = (ROUND[dtype] * (ref.abs() * way.abs()).sum() + ((experts + top_k + 64) * 2.0 ** -23 * size * way.abs()).sum()
               + 1e-8 * (1 + size.sum()) + 1e-11 * size.sum())
        assert abs(slope - along) <= tol, (slope, along, tol)


# ---- the weighted sum back to tokens -----------------------------------------------------------------------------

def combine_inputs(tokens, top_k, width, dtype, seed, drop):
    g = gen(seed)
    n = tokens * top_k
    slot = torch.randperm(n, generator=g, device=DEV).int() if n else torch.empty(0, dtype=torch.int32, device=DEV)
    if drop:
        slot[torch.rand(n, generator=g, device=DEV) < 0.3] = -1
        slot[:top_k] = -1                         # a token without any slot
        if n > top_k:
            slot[-1] = n + 5                      # behind the rows there are: left out as well
    y = randn(g, n, width, dtype=dtype)
    used = torch.zeros(n, dtype=torch.bool, device=DEV)
    good = (slot >= 0) & (slot < n)
    used[slot[good].long()] = True
    y[~used] = NAN                                # rows that no entry names are not read
    return g, slot, good, y, used


SHAPES = [(1, 8, 2048), (5, 8, 2048), (1, 1, 1), (3, 2, 7), (17, 4, 513), (64, 16, 512), (33, 3, 2049), (9, 2, 5001), (130, 1, 4096)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,top_k,width", SHAPES)
@pytest.mark.parametrize("drop", [False, True])
@pytest.mark.parametrize("layout", ["dense", "wide", "shifted"])
def test_combine(tokens, top_k, width, drop, layout, dtype):
    g, slot, good, y, used = combine_inputs(tokens, top_k, width, dtype, 3, drop)
    n = tokens * top_k
    weight = randn(g, tokens, top_k)
    pad, shift = {"dense": (0, 0), "wide": (8, 0), "shifted": (3, 1)}[layout]
    y, ld_y = strided(y, width + pad, shift)
    out, ld_out = strided(torch.zeros(tokens, width, dtype=TORCH[dtype], device=DEV), width + pad, shift, fill=9.0)
    for w in (weight, None):
        pf.moe_combine(y, slot, w, tokens, top_k, width, out, dtype=dtype, ld_y=ld_y, ld_out=ld_out)
        rows = torch.where(good[:, None], y.double()[torch.where(good, slot, 0).long()], 0.0).view(tokens, top_k, width)
        w64 = weight.double() if w is not None else torch.ones(tokens, top_k, dtype=torch.float64, device=DEV)
        ref = (rows * w64[:, :, None]).sum(1)
        close(out, ref, (top_k + 2) * 2.0 ** -23 * (rows.abs() * w64.abs()[:, :, None]).sum(1), dtype, "combine")
    whole = torch.as_strided(out, (tokens, ld_out), (ld_out, 1))[:, width:]
    assert (whole == 9.0).all()                   # the gaps between rows


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,top_k,width", SHAPES)
@pytest.mark.parametrize("drop", [False, True])
@pytest.mark.parametrize("layout", ["dense", "shifted"])
def test_combine_backward(tokens, top_k, width, drop, layout, dtype):
    g, slot, good, y, used = combine_inputs(tokens, top_k, width, dtype, 5, drop)
    n = tokens * top_k
    weight, dout = randn(g, tokens, top_k), randn(g, tokens, width, dtype=dtype)
    pad, shift = {"dense": (0, 0), "shifted": (3, 1)}[layout]
    y, ld_y = strided(y, width + pad, shift)
    dout, ld_dout = strided(dout, width + pad, shift)
    dy, ld_dy = strided(torch.full((n, width), 7.0, dtype=TORCH[dtype], device=DEV), width + pad, shift)
    dweight = torch.full((tokens, top_k), NAN, device=DEV)
    pf.moe_combine_backward(dout, y, slot, weight, tokens, top_k, width, dy, dweight, dtype=dtype, ld_dout=ld_dout, ld_y=ld_y, ld_dy=ld_dy)
    safe = torch.where(good, slot, 0).long()
    rows = torch.where(good[:, None], y.double()[safe], 0.0).view(tokens, top_k, width)
    d64 = dout.double()
    ref = (rows * d64[:, None, :]).sum(2)
    slack = (width + 2) * 2.0 ** -23 * (rows.abs() * d64.abs()[:, None, :]).sum(2)
    close(dweight, ref, slack, "f32", "dweight")
    want = (weight.double()[:, :, None] * d64[:, None, :]).reshape(n, width)
    close(dy[safe[good]], want[good], 2.0 ** -23 * want[good].abs(), dtype, "dy")
    assert (dy[~used] == 7.0).all()               # rows that no entry names keep what they held
    # differences of the 64-bit form along a direction of y and of the weights (it is linear in each: exact)
    way = torch.randn(n, width, generator=g, device=DEV, dtype=torch.float64)
    slope = ((weight.double()[:, :, None] * torch.where(good[:, None], way[safe], 0.0).view(tokens, top_k, width)).sum(1) * d64).sum()
    along = (dy.double()[used] * way[used]).sum()
    assert abs(slope - along) <= 1.01 * (ROUND[dtype] + 2.0 ** -20) * (want.abs() * torch.where(good[:, None], way[safe], 0.0).abs()).sum() + 1e-6


# ---- grouped products --------------------------------------------------------------------------------------------

COUNTS = {
    "one token": [0, 1, 0, 1],
    "few": [3, 0, 17, 1, 16, 0, 5],
    "ragged": [0, 130, 1, 64, 200, 0, 31],
    "one expert": [333],
    "large": [300, 0, 513, 256, 1],
    "empty": [0, 0, 0],
}
NK = [(64, 64), (1, 1), (256, 512), (17, 40), (130, 200), (33, 7), (72, 1000), (129, 257), (520, 96), (8, 0)]


def mm_inputs(counts, n, k, dtype, seed, gather, act, spare=0):
    g = gen(seed)
    e, slots = len(counts), sum(counts) + spare
    top_k = 3
    tokens = max(1, slots // 2)
    rows = torch.randint(0, tokens * top_k, (max(slots, 1),), generator=g, device=DEV).int() if gather else None
    if gather and spare:
        rows[slots - spare:] = -1
    x = randn(g, tokens if gather else max(slots, 1), k, dtype=dtype)
    w = (randn(g, e, (2 if act else 1) * n, k) * max(k, 1) ** -0.5).to(TORCH[dtype])
    return g, e, slots, rows, top_k, x, w


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("case", COUNTS)
@pytest.mark.parametrize("n,k", NK)
def test_mm(case, n, k, dtype):
    counts = COUNTS[case]
    for act, gather, layout in ((0, True, "dense"), (1, False, "wide"), (1, True, "shifted"), (0, False, "shifted")):
        g, e, slots, rows, div, x, w = mm_inputs(counts, n, k, dtype, n + k, gather, act, spare=2)
        pad, shift = {"dense": (0, 0), "wide": (8, 0), "shifted": (1, 1)}[layout]
        x, ld_x = strided(x, k + pad, shift)
        y, ld_y = strided(torch.full((slots, n), 7.0, dtype=TORCH[dtype], device=DEV), n + pad, shift, fill=9.0)
        pre, ld_pre = strided(torch.full((slots, 2 * n), 7.0, dtype=TORCH[dtype], device=DEV), 2 * n + pad, shift, fill=9.0)
        pf.moe_mm(x, x.shape[0], rows, div, w, offsets_of(counts), e, slots, n, k, y, dtype=dtype, act="swiglu" if act else "none",
                  pre=pre if act else None, ld_x=ld_x, ld_y=ld_y, ld_pre=ld_pre if act else 0)
        for i, b, f in groups(counts):
            if b == f:
                continue
            xs = x[(rows[b:f] // div).long()] if gather else x[b:f]
            z, slack = product(xs, w[i])
            if act:
                close(pre[b:f], z, slack, dtype, f"{case} {n}x{k} pre of expert {i}")
                z, slack = swiglu(z[:, :n], z[:, n:], slack[:, :n], slack[:, n:])
            close(y[b:f], z, slack, dtype, f"{case} {n}x{k} act {act} {layout} expert {i}")
        assert (y[slots - 2:] == 7.0).all() and (not act or (pre[slots - 2:] == 7.0).all())
        assert (torch.as_strided(y, (slots, ld_y), (ld_y, 1))[:, n:] == 9.0).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("case", COUNTS)
@pytest.mark.parametrize("n,k", NK)
def test_mm_gradients(case, n, k, dtype):
    counts = COUNTS[case]
    for gather, layout, f32 in ((True, "dense", True), (False, "wide", False), (True, "shifted", False), (False, "shifted", True)):
        g, e, slots, rows, div, x, w = mm_inputs(counts, n, k, dtype, n + k + 1, gather, 0, spare=2)
        dy = randn(g, slots, n, dtype=dtype)
        dy[slots - 2:] = NAN                       # slots of no expert are not read
        pad, shift = {"dense": (0, 0), "wide": (8, 0), "shifted": (1, 1)}[layout]
        x, ld_x = strided(x, k + pad, shift)
        dy, ld_dy = strided(dy, n + pad, shift)
        dx, ld_dx = strided(torch.full((slots, k), 7.0, dtype=TORCH[dtype], device=DEV), k + pad, shift, fill=9.0)
        kind = "f32" if f32 else dtype
        dw = torch.full((e, n, k), NAN, dtype=TORCH[kind], device=DEV)
        off = offsets_of(counts)
        pf.moe_mm_dx(dy, w, off, e, slots, n, k, dx, dtype=dtype, ld_dy=ld_dy, ld_dx=ld_dx)
        pf.moe_mm_dw(dy, x, x.shape[0], rows, div, off, e, slots, n, k, dw, dtype=dtype, dw_dtype=kind, ld_dy=ld_dy, ld_x=ld_x)
        way = torch.randn(e, n, k, generator=g, device=DEV, dtype=torch.float64)
        slope = along = room = 0.0
        for i, b, f in groups(counts):
            xs = x[(rows[b:f] // div).long()] if gather else x[b:f]
            z, slack = product(dy[b:f], w[i].t())
            close(dx[b:f], z, slack, dtype, f"{case} {n}x{k} dx of expert {i}")
            z, slack = product(dy[b:f].t(), xs.t())
            close(dw[i], z, slack, kind, f"{case} {n}x{k} dw of expert {i}")
            # differences: the product is linear in w, so <dy, x (w + way)^T - x w^T> is the slope along `way`
            slope += float((dy[b:f].double() * (xs.double() @ way[i].t())).sum())
            along += float((dw[i].double() * way[i]).sum())
            room += float(((ROUND[kind] * z.abs() + slack) * way[i].abs()).sum())
        assert abs(slope - along) <= 1.01 * room + 1e-6
        assert (dx[slots - 2:] == 7.0).all()
        assert (torch.as_strided(dx, (slots, ld_dx), (ld_dx, 1))[:, k:] == 9.0).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_mm_without_offsets_is_one_product(dtype):
    g = gen(2)
    x, w = randn(g, 300, 520, dtype=dtype), randn(g, 264, 520, dtype=dtype)
    y = torch.empty(300, 264, dtype=TORCH[dtype], device=DEV)
    pf.moe_mm(x, 300, None, 1, w, None, 1, 300, 264, 520, y, dtype=dtype)
    z, slack = product(x, w)
    close(y, z, slack, dtype)


def test_mm_values_outside_the_operands_do_not_matter():
    """Infinities and NaN in rows of other experts, in unused tokens and behind the rows' ends stay out."""
    g = gen(9)
    counts, n, k, dtype = [5, 0, 140, 20], 100, 72, "bf16"
    x = randn(g, 200, k, dtype=dtype)
    rows = torch.randint(0, 100, (165,), generator=g, device=DEV).int() * 2     # odd tokens unused
    x[1::2] = float("inf")
    w = randn(g, 4, n, k, dtype=dtype)
    w[1] = NAN
    x, ld_x = strided(x, k + 8, 0)
    y = torch.empty(165, n, dtype=TORCH[dtype], device=DEV)
    pf.moe_mm(x, 200, rows, 1, w, offsets_of(counts), 4, 165, n, k, y, dtype=dtype, ld_x=ld_x)
    for i, b, f in groups(counts):
        z, slack = product(x[rows[b:f].long()], w[i])
        if b < f:
            close(y[b:f], z, slack, dtype)
    # where they are inside, they come out
    x[rows[7].long(), 3] = float("inf")
    pf.moe_mm(x, 200, rows, 1, w, offsets_of(counts), 4, 165, n, k, y, dtype=dtype, ld_x=ld_x)
    hit = rows == rows[7]
    assert not torch.isfinite(y[hit]).any() and torch.isfinite(y[~hit]).all()


def test_mm_broken_offsets_and_rows_stay_inside():
    """Offsets that decrease or pass the slots, and row indices outside x, give unspecified rows and no fault."""
    g = gen(1)
    for off in ([0, 50, 20, 90], [0, 500, 600, 700], [-5, 10, 40, 60]):
        x, w = randn(g, 30, 64, dtype="bf16"), randn(g, 3, 64, 64, dtype="bf16")
        rows = torch.tensor([-1, 30, 2 ** 31 - 1, -2 ** 31] * 15, dtype=torch.int32, device=DEV)
        y, dw = torch.empty(60, 64, dtype=torch.bfloat16, device=DEV), torch.empty(3, 64, 64, device=DEV)
        o = torch.tensor(off, dtype=torch.int32, device=DEV)
        pf.moe_mm(x, 30, rows, 1, w, o, 3, 60, 64, 64, y)
        pf.moe_mm_dx(y, w, o, 3, 60, 64, 64, torch.empty_like(y))
        pf.moe_mm_dw(y, x, 30, rows, 1, o, 3, 60, 64, 64, dw, dw_dtype="f32")
        torch.cuda.synchronize()


def test_mm_offsets_past_32_bits():
    """Rows of x and of y behind 4 GiB."""
    g = gen(3)
    width, n, tokens = 4096, 64, 600000
    x = torch.zeros(tokens, width, dtype=torch.bfloat16, device=DEV)
    last = randn(g, 40, width, dtype="bf16")
    x[-40:] = last
    rows = torch.arange(tokens - 40, tokens, device=DEV).int()
    w = (randn(g, 2, n, width) * width ** -0.5).to(torch.bfloat16)
    y = torch.empty(40, n, dtype=torch.bfloat16, device=DEV)
    pf.moe_mm(x, tokens, rows, 1, w, offsets_of([15, 25]), 2, 40, n, width, y)
    for i, b, f in groups([15, 25]):
        z, slack = product(last[b:f], w[i])
        close(y[b:f], z, slack, "bf16")
    dw = torch.empty(2, n, width, device=DEV)
    pf.moe_mm_dw(y, x, tokens, rows, 1, offsets_of([15, 25]), 2, 40, n, width, dw, dw_dtype="f32")
    for i, b, f in groups([15, 25]):
        z, slack = product(y[b:f].t(), last[b:f].t())
        close(dw[i], z, slack, "f32")
    out = torch.empty(1, width, dtype=torch.bfloat16, device=DEV)
    slot = torch.tensor([tokens - 1, tokens - 40], dtype=torch.int32, device=DEV)
    pf.moe_combine(x, slot, torch.ones(1, 2, device=DEV), 1, 2, width, out, slots=tokens)
    close(out[0], last[-1].double() + last[0].double(), 2.0 ** -22 * (last[-1].double().abs() + last[0].double().abs()), "bf16")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 7), (65, 512), (130, 1001)])
def test_swiglu_backward(rows, n, dtype):
    g = gen(rows)
    for pad, shift in ((0, 0), (5, 1)):
        dh, ld_dh = strided(randn(g, rows, n, dtype=dtype), n + pad, shift)
        pre, ld_pre = strided(randn(g, rows, 2 * n, dtype=dtype) * 3, 2 * n + pad, shift)
        dpre, ld = strided(torch.empty(rows, 2 * n, dtype=TORCH[dtype], device=DEV), 2 * n + pad, shift, fill=9.0)
        pf.swiglu_backward(dh, pre, rows, n, dpre, dtype=dtype, ld_dh=ld_dh, ld_pre=ld_pre, ld_dpre=ld)
        gate, up, d = pre[:, :n].double(), pre[:, n:].double(), dh.double()
        s = torch.sigmoid(gate)
        # a dozen fp32 roundings of terms that are at most this large
        size = d.abs() * (1 + gate.abs()) * 2.0 ** -23 * 16
        close(dpre[:, :n], d * up * s * (1 + gate * (1 - s)), size * up.abs(), dtype, "gate")
        close(dpre[:, n:], d * gate * s, size, dtype, "up")
        h = 1e-5
        f = lambda a, b: a * torch.sigmoid(a) * b  # noqa: E731
        way = torch.randn(rows, 2 * n, generator=g, device=DEV, dtype=torch.float64)
        p64 = pre.double()
        up_, dn = p64 + h * way, p64 - h * way
        slope = ((f(up_[:, :n], up_[:, n:]) - f(dn[:, :n], dn[:, n:])) * d).sum() / (2 * h)
        along = (dpre.double() * way).sum()
        room = (ROUND[dtype] * dpre.double().abs() * way.abs()).sum() * 1.01 + 1e-4 * (d.abs() * (1 + p64[:, :n].abs()) * (1 + p64[:, n:].abs())).sum()
        assert abs(slope - along) <= room


# ---- 4-bit blocks ------------------------------------------------------------------------------------------------

VALUES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def quantised_reference(x):
    """codes, scales and values of x (float64, CPU) by the definition: the nearest value, ties to the even code."""
    blocks = x.reshape(x.shape[0], -1, 32)
    bad = ~torch.isfinite(blocks).all(2)
    most = torch.where(torch.isfinite(blocks), blocks, torch.zeros_like(blocks)).abs().amax(2)
    e = torch.floor(torch.log2(torch.where(most > 0, most, torch.full_like(most, 2.0 ** -200)))) - 2
    e = e.clamp(min=-127)
    v = torch.where(torch.isfinite(blocks), blocks, torch.zeros_like(blocks)) / torch.exp2(e)[..., None]
    gap = (v.abs()[..., None] - VALUES).abs()
    best = gap.amin(-1, keepdim=True)
    near = gap == best                                   # two of them at a tie: take the even code
    code = torch.where(near, torch.arange(8) + 8 * (torch.arange(8) % 2), torch.full((8,), 99)).amin(-1) % 8
    held = VALUES[code] * torch.exp2(e)[..., None]
    code = code + 8 * torch.signbit(blocks)
    held = torch.where(torch.signbit(blocks), -held, held)
    code[bad] = 0
    held[bad] = NAN
    scale = torch.where(bad, torch.full_like(e, 255.0), e + 127)
    code = code.reshape(x.shape[0], -1, 2)
    return (code[..., 0] + 16 * code[..., 1]).to(torch.uint8), scale.to(torch.uint8), held.reshape(x.shape)


def quantise(x, dtype, pad=0, shift=0):
    rows, k = x.shape
    view, ld = strided(x, k + pad, shift)
    codes = torch.full((max(rows, 1), k // 2), 0x55, dtype=torch.uint8, device=DEV)
    scales = torch.full((max(rows, 1), k // 32), 7, dtype=torch.uint8, device=DEV)
    pf.mx4_quantize(view, rows, k, codes, scales, dtype=dtype, ld_x=ld)
    return codes, scales


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,k", [(1, 32), (3, 64), (65, 96), (7, 1056), (130, 512)])
def test_quantise(rows, k, dtype):
    g = gen(rows + k)
    x = randn(g, rows, k) * torch.exp2(4 * torch.randn(rows, 1, generator=g, device=DEV))
    x.view(-1)[:32] = 0.0
    if rows > 2:
        x[1, :32] = torch.arange(32, device=DEV) * 0.125 - 2            # many ties
        x[2, 32 % k:][:32] = -0.0
        x[2, 5] = 8.0 * 0.999
    x = x.to(TORCH[dtype])
    for pad, shift in ((0, 0), (32, 0), (1, 1)):
        codes, scales = quantise(x, dtype, pad, shift)
        c, s, held = quantised_reference(x.double().cpu())
        assert torch.equal(codes.cpu(), c) and torch.equal(scales.cpu(), s)
        for out in ("f32", "f16", "bf16"):
            y, ld = strided(torch.full((rows, k), 7.0, dtype=TORCH[out], device=DEV), k + pad, shift, fill=9.0)
            pf.mx4_dequantize(codes, scales, rows, k, y, dtype=out, ld_y=ld)
            assert torch.equal(y.cpu(), held.to(TORCH[out])), out
            assert (torch.as_strided(y, (rows, ld), (ld, 1))[:, k:] == 9.0).all()


def test_quantise_extremes():
    x = torch.zeros(8, 64, device=DEV)
    x[0, :32] = torch.finfo(torch.float32).max
    x[1, 3] = float("inf")
    x[2, 40] = NAN
    x[3, :] = 2.0 ** -140                        # below the smallest scale
    x[4, 0] = 2.0 ** -126
    x[5, :32] = torch.linspace(-1.9, 1.9, 32, device=DEV) * 2.0 ** -124
    x[6, 0], x[6, 1] = 1e30, 1e-30
    codes, scales = quantise(x, "f32")
    c, s, held = quantised_reference(x.double().cpu())
    assert torch.equal(scales.cpu(), s) and torch.equal(codes.cpu(), c)
    y = torch.empty(8, 64, device=DEV)
    pf.mx4_dequantize(codes, scales, 8, 64, y)
    assert torch.equal(torch.nan_to_num(y.cpu().double(), nan=123.0), torch.nan_to_num(held, nan=123.0))
    assert scales[1, 0] == 255 and scales[1, 1] == 0 and torch.isnan(y[1, :32]).all()


def mx4_weights(g, e, rows, k):
    w = (randn(g, e * rows, k) * max(k, 1) ** -0.5).to(torch.bfloat16)
    codes, scales = quantise(w, "bf16")
    held = torch.empty(e * rows, k, device=DEV)
    pf.mx4_dequantize(codes, scales, e * rows, k, held)
    return codes, scales, held.view(e, rows, k)


@pytest.mark.parametrize("case", COUNTS)
@pytest.mark.parametrize("n,k", [(64, 64), (1, 32), (256, 512), (17, 96), (130, 1056), (33, 2048), (520, 288), (8, 0)])
def test_mm_mx4(case, n, k):
    counts = COUNTS[case]
    for act, gather, dtype in ((0, True, "f16"), (1, False, "bf16"), (1, True, "bf16"), (0, False, "bf16")):
        g = gen(n + k)
        e, slots = len(counts), sum(counts) + 2
        tokens = max(1, slots // 2)
        rows = torch.randint(0, tokens * 3, (slots,), generator=g, device=DEV).int() if gather else None
        x = randn(g, tokens if gather else slots, k, dtype="bf16")
        xq, xs = quantise(x, "bf16")
        xv = torch.empty(x.shape, device=DEV)
        pf.mx4_dequantize(xq, xs, x.shape[0], k, xv)
        wq, ws, wv = mx4_weights(g, e, (2 if act else 1) * n, k)
        y, ld_y = strided(torch.full((slots, n), 7.0, dtype=TORCH[dtype], device=DEV), n + (3 if act else 0), act, fill=9.0)
        pf.moe_mm_mx4(xq, xs, x.shape[0], rows, 3, wq, ws, offsets_of(counts), e, slots, n, k, y, dtype=dtype,
                      act="swiglu" if act else "none", ld_y=ld_y)
        for i, b, f in groups(counts):
            if b == f:
                continue
            v = xv[(rows[b:f] // 3).long()] if gather else xv[b:f]
            z, slack = product(v, wv[i])
            if act:
                z, slack = swiglu(z[:, :n], z[:, n:], slack[:, :n], slack[:, n:])
            close(y[b:f], z, slack, dtype, f"{case} {n}x{k} act {act} expert {i}")
        assert (y[slots - 2:] == 7.0).all()


def test_mm_mx4_scales_and_nan():
    """Scales from 2^-127 up count as what they stand for, and a block of scale 255 makes its row NaN."""
    g = gen(6)
    k, n, m = 160, 40, 20
    xq = torch.randint(0, 256, (m, k // 2), generator=g, device=DEV, dtype=torch.int32).to(torch.uint8)
    wq = torch.randint(0, 256, (n, k // 2), generator=g, device=DEV, dtype=torch.int32).to(torch.uint8)
    xs = torch.randint(100, 150, (m, k // 32), generator=g, device=DEV, dtype=torch.int32).to(torch.uint8)
    ws = torch.randint(100, 150, (n, k // 32), generator=g, device=DEV, dtype=torch.int32).to(torch.uint8)
    xs[3], ws[5] = 0, 200
    xs[4] = 255
    xv, wv = torch.empty(m, k, device=DEV), torch.empty(n, k, device=DEV)
    pf.mx4_dequantize(xq, xs, m, k, xv)
    pf.mx4_dequantize(wq, ws, n, k, wv)
    y = torch.empty(m, n, dtype=torch.bfloat16, device=DEV)
    pf.moe_mm_mx4(xq, xs, m, None, 1, wq, ws, None, 1, m, n, k, y)
    z, slack = product(xv, wv)
    keep = [i for i in range(m) if i != 4]
    close(y[keep], z[keep], slack[keep] + 2.0 ** -126, "bf16")
    assert torch.isnan(y[4]).all()


# ---- streams, graphs, repetition ---------------------------------------------------------------------------------

def layer(s, stream):
    t, e, k, d, n = 50, 8, 2, 128, 192
    pf.moe_route(s["z"], t, e, k, s["choice"], s["weight"], s["offsets"], s["order"], s["slot"], s["work"], dtype="bf16", stream=stream)
    pf.moe_mm(s["x"], t, s["order"], k, s["w1"], s["offsets"], e, t * k, n, d, s["h"], act="swiglu", pre=s["pre"], stream=stream)
    pf.moe_mm(s["h"], t * k, None, 1, s["w2"], s["offsets"], e, t * k, d, n, s["y"], stream=stream)
    pf.moe_combine(s["y"], s["slot"], s["weight"], t, k, d, s["out"], stream=stream)
    pf.moe_combine_backward(s["dout"], s["y"], s["slot"], s["weight"], t, k, d, s["dy"], s["dweight"], stream=stream)
    pf.moe_mm_dx(s["dy"], s["w2"], s["offsets"], e, t * k, d, n, s["dh"], stream=stream)
    pf.moe_mm_dw(s["dy"], s["h"], t * k, None, 1, s["offsets"], e, t * k, d, n, s["dw2"], dw_dtype="f32", stream=stream)
    pf.swiglu_backward(s["dh"], s["pre"], t * k, n, s["dpre"], stream=stream)
    pf.moe_mm_dx(s["dpre"], s["w1"], s["offsets"], e, t * k, 2 * n, d, s["dxs"], stream=stream)
    pf.moe_mm_dw(s["dpre"], s["x"], t, s["order"], k, s["offsets"], e, t * k, 2 * n, d, s["dw1"], dw_dtype="f32", stream=stream)
    pf.moe_combine(s["dxs"], s["slot"], None, t, k, d, s["dx"], stream=stream)
    pf.moe_route_backward(s["z"], t, e, k, s["choice"], s["weight"], s["dweight"], s["dz"], dtype="bf16", stream=stream)
    pf.mx4_quantize(s["x"], t, d, s["xq"], s["xs"], stream=stream)
    pf.moe_mm_mx4(s["xq"], s["xs"], t, s["order"], k, s["wq"], s["ws"], s["offsets"], e, t * k, n, d, s["h4"], act="swiglu", stream=stream)
    return {k_: s[k_] for k_ in ("choice", "weight", "offsets", "order", "slot", "out", "dw1", "dw2", "dx", "dz", "h4")}


def layer_state():
    g = gen(8)
    t, e, k, d, n = 50, 8, 2, 128, 192
    b = lambda *shape: torch.zeros(*shape, dtype=torch.bfloat16, device=DEV)  # noqa: E731
    i = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=DEV)  # noqa: E731
    u = lambda *shape: torch.zeros(*shape, dtype=torch.uint8, device=DEV)  # noqa: E731
    s = {"z": randn(g, t, e, dtype="bf16"), "x": randn(g, t, d, dtype="bf16"), "dout": randn(g, t, d, dtype="bf16"),
         "w1": randn(g, e, 2 * n, d, dtype="bf16") * 0.1, "w2": randn(g, e, d, n, dtype="bf16") * 0.1,
         "choice": i(t, k), "weight": torch.zeros(t, k, device=DEV), "offsets": i(e + 1), "order": i(t * k), "slot": i(t * k),
         "work": i(max(1, pf.moe_route_workspace(t, e) // 4)), "h": b(t * k, n), "pre": b(t * k, 2 * n), "y": b(t * k, d), "out": b(t, d),
         "dy": b(t * k, d), "dweight": torch.zeros(t, k, device=DEV), "dh": b(t * k, n), "dpre": b(t * k, 2 * n), "dxs": b(t * k, d),
         "dx": b(t, d), "dz": b(t, e), "dw1": torch.zeros(e, 2 * n, d, device=DEV), "dw2": torch.zeros(e, d, n, device=DEV),
         "xq": u(t, d // 2), "xs": u(t, d // 32), "h4": b(t * k, n)}
    s["wq"], s["ws"], _ = mx4_weights(g, e, 2 * n, d)
    return s


def test_layer_on_another_stream_and_in_a_graph():
    s = layer_state()
    torch.cuda.synchronize()
    first = {k: v.clone() for k, v in layer(s, None).items()}
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    outputs = list(first)

    def wipe():
        for name in outputs:
            s[name].fill_(3)

    with torch.cuda.stream(stream):
        wipe()
        layer(s, stream)
        stream.synchronize()
        assert all(torch.equal(s[k], first[k]) for k in outputs), "another stream"
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            layer(s, stream)
        for replay in range(4):
            wipe()
            graph.replay()
            stream.synchronize()
            assert all(torch.equal(s[k], first[k]) for k in outputs), f"replay {replay}"
            layer(s, stream)                       # eager work between the replays
            stream.synchronize()
