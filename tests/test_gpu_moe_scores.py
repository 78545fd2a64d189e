"""Routing by scores (include/prefree_moe.h) against plain 64-bit forms; the gradient also against differences."""
import numpy as np
import pytest
import torch

import prefree_amd as pf
from moe_util import DEV, NAN, ROUND, TORCH, strided

pytestmark = pytest.mark.gpu


def scores(z, score):
    z = np.asarray(z, dtype=np.float64)
    with np.errstate(all="ignore"):
        if score == "sigmoid":
            return 1 / (1 + np.exp(-z))
        most = z.max(1, keepdims=True)
        part = np.exp(z - np.where(most > -np.inf, most, 0))
        return part / np.where(part.sum(1, keepdims=True) > 0, part.sum(1, keepdims=True), 1)


def best_first(v, k):
    """The k largest of each row, of equal ones the lowest index, NaN before all."""
    nan = np.isnan(v)
    first = np.argsort(-np.where(nan, np.inf, v), axis=1, kind="stable")
    second = np.argsort(~np.take_along_axis(nan, first, 1), axis=1, kind="stable")
    return np.take_along_axis(first, second, 1)[:, :k]


def reference(z, k, score="sigmoid", bias=None, groups=1, kept=1, best=2, normalise=True, scale=1.0):
    """choice, weight, offsets, order, slot."""
    z = np.asarray(z, dtype=np.float64)
    tokens, experts = z.shape
    s = scores(z, score)
    with np.errstate(all="ignore"):
        if bias is None and (groups == 1 or best == 1):
            r = z.copy()
        else:
            r = s + (0 if bias is None else np.asarray(bias, dtype=np.float64))
    r[z == -np.inf] = -np.inf
    if groups > 1:
        in_groups = r.reshape(tokens, groups, -1)
        order = np.sort(np.where(np.isnan(in_groups), np.inf, in_groups), axis=2)[:, :, ::-1][:, :, :best]
        value = np.where(order > -np.inf, order, 0).sum(2)
        value[order[:, :, 0] == -np.inf] = -np.inf
        value[np.isnan(in_groups).any(2)] = np.nan
        stays = np.zeros((tokens, groups), dtype=bool)
        np.put_along_axis(stays, best_first(value, kept), True, 1)
        r = np.where(stays[:, :, None], in_groups, -np.inf).reshape(tokens, experts)
    index = best_first(r, k)
    chosen = ~(np.take_along_axis(r, index, 1) == -np.inf)
    choice = np.where(chosen, index, -1).astype(np.int32)
    zc = np.take_along_axis(z, index, 1)
    with np.errstate(all="ignore"):
        if not normalise:
            weight = np.take_along_axis(s, index, 1)
        elif score == "softmax":
            part = np.where(chosen, np.exp(zc - np.where(chosen, zc, -np.inf).max(1, keepdims=True)), 0)
            weight = part / part.sum(1, keepdims=True)
        else:
            # the ratio of sigmoids, by their logarithms
            log = np.where(chosen, -np.logaddexp(0, -zc), -np.inf)
            part = np.exp(log - log.max(1, keepdims=True))
            weight = part / part.sum(1, keepdims=True)
        weight = np.where(chosen, scale * weight, 0)
    flat = choice.reshape(-1)
    order = np.argsort(np.where(flat < 0, experts, flat), kind="stable")
    used = int((flat >= 0).sum())
    offsets = np.zeros(experts + 1, dtype=np.int32)
    offsets[1:] = np.cumsum(np.bincount(flat[flat >= 0], minlength=experts))
    slot = np.full(flat.size, -1, dtype=np.int32)
    slot[order[:used]] = np.arange(used)
    order = np.where(np.arange(flat.size) < used, order, -1).astype(np.int32)
    return choice, weight, offsets, order, slot


def route(z, k, dtype="f32", ld=0, shift=0, bias=None, stream=None, **kw):
    tokens, experts = z.shape
    view, ld = strided(z.to(TORCH[dtype]), ld, shift)
    i = lambda *n: torch.full(n, 99, dtype=torch.int32, device=DEV)  # noqa: E731
    choice, weight, offsets, order, slot = i(tokens, k), torch.full((tokens, k), NAN, device=DEV), i(experts + 1), i(tokens * k), i(tokens * k)
    work = torch.full((pf.moe_route_workspace(tokens, experts) + 4,), 0x5a, dtype=torch.uint8, device=DEV)
    pf.moe_route_scores(view, tokens, experts, k, choice, weight, offsets, order, slot, work, dtype=dtype, bias=bias, ld_logits=ld, stream=stream, **kw)
    torch.cuda.synchronize()
    return [v.cpu().numpy() for v in (choice, weight, offsets, order, slot)], view


def check(z, k, dtype="f32", bias=None, ld=0, shift=0, **kw):
    got, held = route(z, k, dtype, ld, shift, bias, **kw)
    ref_kw = dict(kw)
    ref_kw["kept"] = ref_kw.pop("groups_kept", kw.get("groups", 1))
    ref_kw["best"] = ref_kw.pop("group_best", 2)
    want = reference(held.double().cpu().numpy(), k, bias=None if bias is None else bias.cpu().numpy(), **ref_kw)
    for name, g, w in zip(("choice", "weight", "offsets", "order", "slot"), got, want):
        if name == "weight":
            # exp, sum, quotients and the scale: each at most two roundings of fp32, and of a sum over all experts 2^-24 a term,
            # at most 2^-20 for 16 to a lane; exp's argument is rounded too, |z - m| 2^-24
            off = np.abs(np.where(np.isnan(w), 0, g) - np.where(np.isnan(w), 0, w))
            span = np.abs(np.where(np.isfinite(held.double().cpu().numpy()), held.double().cpu().numpy(), 0)).max() if held.numel() else 0
            assert np.array_equal(np.isnan(g), np.isnan(w)) and (off <= (2.0 ** -19 + span * 2.0 ** -22) * np.abs(np.where(np.isnan(w), 0, w)) + 2.0 ** -126).all()
        else:
            assert np.array_equal(g, w), (name, np.argwhere(g != w)[:5], g[g != w][:5], w[g != w][:5])
    return got


def logits(tokens, experts, seed, masked=False):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    z = torch.randn(tokens, experts, generator=g, device=DEV) * 1.5 + torch.randn(experts, generator=g, device=DEV) * 0.5
    if masked:
        z[torch.rand(tokens, experts, generator=g, device=DEV) < 0.3] = -float("inf")
        z[3::8] = -float("inf")
    return z


def biases(experts, seed=9):
    return torch.randn(experts, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV) * 0.1


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tokens,experts,k,groups,kept,best", [
    (1, 64, 8, 8, 4, 2), (5, 1, 1, 1, 1, 1), (67, 8, 2, 1, 1, 2), (130, 60, 6, 4, 2, 1), (64, 96, 6, 8, 3, 2), (65, 256, 8, 8, 4, 2),
    (300, 160, 6, 8, 3, 1), (200, 255, 16, 5, 2, 2), (77, 320, 8, 16, 5, 2), (66, 512, 3, 16, 1, 1), (129, 1024, 16, 16, 7, 2), (40, 16, 4, 16, 3, 2)])
def test_route(tokens, experts, k, groups, kept, best, dtype, score):
    for bias in (None, biases(experts)):
        for normalise, scale, masked in ((True, 1.0, False), (False, 2.5, True)):
            check(logits(tokens, experts, tokens + experts, masked), k, dtype, bias, score=score, groups=groups, groups_kept=kept, group_best=best,
                  normalise=normalise, scale=scale)


@pytest.mark.parametrize("tokens", [4161, 65537])
def test_many_tokens(tokens):
    """Several launches; among so many scores some lie next to each other."""
    check(logits(tokens, 32, 1, True), 4, bias=biases(32), groups=4, groups_kept=2)


def test_scores_next_to_each_other():
    """Sums that 32 bits do not tell apart, or tell wrongly: logits and biases a few steps of fp32 apart."""
    g = torch.Generator(device=DEV).manual_seed(3)
    for score, experts in (("sigmoid", 256), ("softmax", 64), ("sigmoid", 600)):
        z = torch.randint(-3, 4, (3000, experts), generator=g, device=DEV).float() * 2.0 ** -21 + torch.randint(0, 4, (3000, experts), generator=g, device=DEV)
        bias = torch.randint(-2, 3, (experts,), generator=g, device=DEV).float() * 2.0 ** -25 + 0.25
        check(z, 8, bias=bias, score=score, groups=8, groups_kept=3)
        check(z, 8, bias=bias, score=score)
        check(z, 8, score=score, groups=8, groups_kept=3)
        check(z, 8, bias=torch.zeros(experts, device=DEV), score=score, groups=4, groups_kept=2, group_best=1)


def test_ties_go_to_the_lowest_index():
    z = torch.zeros(130, 48, device=DEV)
    for kw in ({}, {"bias": torch.zeros(48, device=DEV)}, {"groups": 4, "groups_kept": 2}, {"bias": torch.ones(48, device=DEV), "groups": 8, "groups_kept": 3}):
        got = check(z, 5, **kw)
        assert (got[0] == np.arange(5)).all()
    z = torch.randint(-2, 3, (500, 240), generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).float()
    for groups, kept, best in ((1, 1, 2), (8, 3, 2), (8, 3, 1), (16, 2, 2)):
        check(z, 7, bias=torch.zeros(240, device=DEV), groups=groups, groups_kept=kept, group_best=best)
        check(z, 7, "bf16", groups=groups, groups_kept=kept, group_best=best)


@pytest.mark.parametrize("groups,kept", [(1, 1), (4, 2)])
def test_masks_and_values_without_an_order(groups, kept):
    inf = float("inf")
    z = logits(70, 32, 5)
    z[0], z[1, 1:], z[2, :30] = -inf, -inf, -inf          # nothing, one, two left
    z[3, 5], z[4, :] = NAN, NAN
    z[5, 9] = inf
    bias = biases(32)
    bias[7] = -inf                                         # out of service
    bias[9] = inf                                          # in whatever its score
    for b in (None, bias):
        check(z, 4, bias=b, groups=groups, groups_kept=kept)
        check(z, 4, bias=b, groups=groups, groups_kept=kept, normalise=False)
    got = check(z, 4, bias=bias, groups=groups, groups_kept=kept)
    assert not (got[0] == 7).any()
    few = torch.full((70, 32), -inf, device=DEV)           # fewer in the kept groups than are asked for
    few[:, ::8] = 1
    check(few, 4, bias=biases(32), groups=groups, groups_kept=kept)


def test_far_logits():
    """Sigmoids that are no normal numbers: their ratios are."""
    z = logits(100, 16, 6) * 3 - 120
    got = check(z, 4)
    assert np.allclose(got[1].sum(1), 1, atol=2.0 ** -20)
    check(z + 300, 4)
    check(logits(100, 16, 6) * 40, 4, score="softmax")


@pytest.mark.parametrize("ld,shift", [(50, 0), (49, 1), (0, 3)])
def test_strides(ld, shift):
    for dtype in ("f32", "bf16"):
        check(logits(90, 48, 7), 5, dtype, biases(48), ld, shift, groups=8, groups_kept=4)


def test_no_tokens():
    got = route(logits(0, 24, 1), 3)[0]
    assert not got[2].any()


def test_agrees_with_the_plain_routing():
    z = logits(700, 128, 8, True)
    i = lambda *n: torch.empty(n, dtype=torch.int32, device=DEV)  # noqa: E731
    for normalise in (True, False):
        got, _ = route(z, 8, score="softmax", normalise=normalise)
        out = [i(700, 8), torch.empty(700, 8, device=DEV), i(129), i(5600), i(5600)]
        pf.moe_route(z, 700, 128, 8, *out, torch.empty(pf.moe_route_workspace(700, 128), dtype=torch.uint8, device=DEV), normalise=normalise)
        torch.cuda.synchronize()
        for a, b in zip(got, out):
            assert np.array_equal(a, b.cpu().numpy()) or (a.dtype == np.float32 and np.allclose(a, b.cpu().numpy(), rtol=2.0 ** -19, atol=0))


def weights_of(z, choice, score, normalise, scale):
    """Weights of a fixed choice, in 64 bits, for derivatives."""
    s = torch.sigmoid(z) if score == "sigmoid" else torch.softmax(z, 1)
    part = torch.where(choice >= 0, s.gather(1, choice.clamp(min=0).long()), 0.0)
    return scale * (part / part.sum(1, keepdim=True).clamp(min=1e-300) if normalise else part)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("normalise", [True, False])
@pytest.mark.parametrize("dtype,tokens,experts,k,ld", [("f32", 100, 64, 6, 0), ("bf16", 37, 96, 8, 0), ("f16", 65, 17, 3, 0), ("f32", 33, 1024, 16, 1030),
                                                       ("bf16", 18, 33, 4, 35), ("f32", 16, 1, 1, 0), ("bf16", 1, 256, 8, 256)])
def test_gradient(score, normalise, dtype, tokens, experts, k, ld):
    scale = 2.5
    z = logits(tokens, experts, 11)
    if experts > 4:
        z[0], z[tokens // 2, 3:] = -float("inf"), -float("inf")
    (choice, weight, *_), held = route(z, k, dtype, ld, bias=biases(experts), score=score, normalise=normalise, scale=scale)
    choice, weight = torch.from_numpy(choice).to(DEV), torch.from_numpy(weight).to(DEV)
    dweight = torch.randn(tokens, k, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV)
    out, ld_d = strided(torch.full((tokens, experts), NAN, dtype=TORCH[dtype], device=DEV), ld + (3 if ld else 0), 0, fill=7.0)
    pf.moe_route_scores_backward(held, tokens, experts, k, choice, weight, dweight, out, dtype=dtype, score=score, normalise=normalise, scale=scale,
                                 ld_logits=ld, ld_dlogits=ld_d)
    torch.cuda.synchronize()
    z64 = held.double().contiguous().requires_grad_()
    live = z64.detach().max(1)[0] > -float("inf")
    full = weights_of(z64[live], choice[live], score, normalise, scale)
    want = torch.zeros(tokens, experts, dtype=torch.float64, device=DEV)
    want[live] = torch.autograd.grad((full * dweight[live].double()).sum(), z64)[0][live].nan_to_num()
    # w, 1 - s and the sum over the chosen are off by 2^-20 of themselves and of the sum's terms
    slack = 2.0 ** -18 * scale * dweight.abs().sum(1, keepdim=True).double()
    assert ((out.double() - want).abs() <= ROUND[dtype] * want.abs() + slack + 2.0 ** -24).all()
    assert not out[~live].any()
    if ld_d > experts:
        assert (out.as_strided((tokens - 1, ld_d - experts), (ld_d, 1), experts) == 7).all()
    # along a direction, against the difference of the weights
    if dtype == "f32" and experts > 1:
        way = torch.randn(tokens, experts, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV).double()
        base, h = held.double()[live], 1e-5
        f = lambda z: (weights_of(z, choice[live], score, normalise, scale) * dweight[live].double()).sum()  # noqa: E731
        slope = (f(base + h * way[live]) - f(base - h * way[live])) / (2 * h)
        along = (out.double() * way).sum()
        assert abs(slope - along) <= (slack * way.abs().sum(1, keepdim=True)).sum() + 1e-6


def test_balance():
    counts = torch.tensor([5, 0, 3, 4, 3, 3], dtype=torch.int32, device=DEV)       # a mean of 3
    offsets = torch.cat([torch.zeros(1, dtype=torch.int32, device=DEV), counts.cumsum(0).int()])
    bias = torch.randn(6, device=DEV)
    want = bias + 0.25 * torch.tensor([-1, 1, 0, -1, 0, 0], device=DEV)
    out = torch.empty(6, device=DEV)
    pf.moe_balance(offsets, 6, 0.25, bias, out)
    pf.moe_balance(offsets, 6, 0.25, bias, bias)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(bias, want)
    counts = torch.randint(0, 1 << 19, (1023,), generator=torch.Generator(device=DEV).manual_seed(4), device=DEV)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), counts.cumsum(0)]).int()
    bias, out = torch.zeros(1023, device=DEV), torch.empty(1023, device=DEV)
    pf.moe_balance(offsets, 1023, 1.0, bias, out)
    torch.cuda.synchronize()
    assert torch.equal(out, torch.sign(offsets[-1].long() - counts * 1023).float())


def test_balancing_evens_the_load():
    """Routing and its bias's step in turn, as training has them: the busiest expert's share falls to near the mean."""
    tokens, experts, k = 2048, 32, 4
    z = logits(tokens, experts, 12) + torch.linspace(-1, 1, experts, device=DEV)
    bias = torch.zeros(experts, device=DEV)
    most = []
    for _ in range(150):
        got, _ = route(z, k, bias=bias, groups=4, groups_kept=2)
        offsets = torch.from_numpy(got[2]).to(DEV)
        most.append(int(np.diff(got[2]).max()))
        pf.moe_balance(offsets, experts, 5e-3, bias, bias)
    mean = tokens * k / experts
    assert most[0] > 1.5 * mean and most[-1] < 1.25 * mean


def test_equal_and_nearly_equal_at_the_end_of_the_choice():
    """Behind the last chosen: one with the same logit, then one that 32 bits cannot tell from both and 64 bits put first."""
    k, experts = 6, 40
    z = torch.full((64, experts), -4.0, device=DEV)
    z[:, 30:30 + k - 1] = torch.linspace(2, 1, k - 1, device=DEV)
    step = 2.0 ** -24                                       # of a logit of 0.5; of its sigmoid a quarter
    z[:, 3], z[:, 9], z[:, 20] = 0.5, 0.5, 0.5 + 2 * step
    z[1::2, 21] = 0.5 + step
    z[2::4, 22:29] = 0.5
    for bias in (None, torch.zeros(experts, device=DEV), torch.full((experts,), 0.125, device=DEV)):
        got = check(z, k, bias=bias)
        assert (got[0][:, k - 1] == 20).all()
        check(z, k, bias=bias, score="softmax")
        for groups, kept in ((4, 2), (8, 5), (10, 4)):
            check(z, k, bias=bias, groups=groups, groups_kept=kept, group_best=1)
            check(z, k, bias=bias, groups=groups, groups_kept=kept)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("experts,groups,kept", [(255, 3, 2), (256, 8, 4), (96, 16, 3), (1020, 3, 1), (1024, 4, 2), (640, 5, 2), (24, 8, 8), (7, 7, 3)])
def test_layouts_of_groups_over_lanes(experts, groups, kept, dtype):
    for top_k in (1, 14, 15, 16):
        if top_k <= experts:
            check(logits(70, experts, experts, True), top_k, dtype, biases(experts), groups=groups, groups_kept=kept)
            check(logits(70, experts, experts), top_k, dtype, groups=groups, groups_kept=kept, group_best=1, score="softmax", normalise=False)


def test_wide_biases_and_logits():
    """Biases far larger than scores, and logits over the whole range of fp32: fixed point with little room between them."""
    z, g = logits(300, 64, 21), torch.Generator(device=DEV).manual_seed(5)
    check(z, 8, bias=torch.randn(64, generator=g, device=DEV) * 1e4, groups=8, groups_kept=4)
    check(z, 8, bias=torch.randint(-2, 3, (64,), generator=g, device=DEV).float() * 1e6, groups=8, groups_kept=4)
    wild = z * torch.exp2(torch.randint(-60, 60, (300, 64), generator=g, device=DEV).float())
    check(wild, 8)
    check(wild, 8, groups=8, groups_kept=2, group_best=1)
    huge = z.sign() * 3e38
    check(huge, 8)
    check(huge, 8, bias=biases(64), groups=4, groups_kept=2)


@pytest.mark.parametrize("level", [0.0, -0.3, 0.3, 50.0, -50.0, 3e7, -3e7])
def test_groups_with_one_expert_left(level):
    """A group of which one expert can be chosen counts its score alone, above or below the sums of two."""
    g = torch.Generator(device=DEV).manual_seed(6)
    z = logits(2000, 32, 13)
    z[torch.rand(2000, 32, generator=g, device=DEV) < 0.8] = -float("inf")
    check(z, 4, bias=biases(32) + level, groups=8, groups_kept=3)
    check(z, 4, bias=biases(32) + level, groups=4, groups_kept=2, score="softmax")


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("scale", [1.0, 2.5, 0.3, 7.7e-5])
def test_gradient_of_one_expert_is_none(score, scale):
    """Its weight is the scale, whatever its logit."""
    tokens, experts = 300, 24
    z = logits(tokens, experts, 5)
    (choice, weight, *_), held = route(z, 1, score=score, scale=scale)
    assert (weight == np.float32(scale)).all()
    dz = torch.full((tokens, experts), NAN, device=DEV)
    dweight = torch.randn(tokens, 1, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    pf.moe_route_scores_backward(held, tokens, experts, 1, torch.from_numpy(choice).to(DEV), torch.from_numpy(weight).to(DEV), dweight, dz, score=score, scale=scale)
    torch.cuda.synchronize()
    assert (dz == 0).all()
