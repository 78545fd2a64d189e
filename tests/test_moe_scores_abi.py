"""Routing by scores (include/prefree_moe.h) — CPU only: refusals before any launch."""
import pytest

import prefree_amd as pf
from test_moe_abi import ALIGN, INVALID, P, refused


def route(logits=P, tokens=100, experts=8, top_k=2, choice=P, weight=P, offsets=P, order=P, slot=P, work=P, work_bytes=1 << 20, ld=0, **kw):
    pf.moe_route_scores(logits, tokens, experts, top_k, choice, weight, offsets, order, slot, work, workspace_bytes=work_bytes, ld_logits=ld, **kw)


@pytest.mark.parametrize("kw", [{"tokens": -1}, {"experts": 0}, {"experts": 1025}, {"top_k": 0}, {"top_k": 9}, {"experts": 64, "top_k": 17},
                                {"logits": None}, {"choice": None}, {"weight": None}, {"offsets": None}, {"order": None}, {"slot": None},
                                {"dtype": "f64"}, {"work": None}, {"work_bytes": 63}, {"ld": 7}, {"ld": -1}, {"tokens": 1 << 30},
                                {"score": 2}, {"groups": 0}, {"groups": 3}, {"groups": 17, "experts": 34}, {"groups": 4, "groups_kept": 5},
                                {"groups": 4, "groups_kept": 0}, {"group_best": 0}, {"group_best": 3}, {"scale": 0.0}, {"scale": -1.0},
                                {"scale": float("inf")}, {"scale": float("nan")}])
def test_route_refusals(kw):
    refused(INVALID, route, **kw)


def test_route_alignment_and_names():
    for kw in ({"logits": P + 2}, {"work": P + 2}, {"bias": P + 1}, {"choice": P + 1}, {"weight": P + 2}, {"offsets": P + 2}, {"order": P + 2},
               {"slot": P + 2}, {"logits": P + 1, "dtype": "bf16"}):
        refused(ALIGN, route, **kw)
    with pytest.raises(KeyError):
        route(score="tanh")
    torch = pytest.importorskip("torch")
    with pytest.raises(TypeError):
        route(bias=torch.zeros(8, dtype=torch.float64))
    with pytest.raises(TypeError):
        route(bias=torch.zeros(8))                       # not on the GPU


def test_backward_refusals():
    back = lambda z=P, tokens=4, experts=8, choice=P, weight=P, dweight=P, d=P, **kw: pf.moe_route_scores_backward(  # noqa: E731
        z, tokens, experts, 2, choice, weight, dweight, d, **kw)
    for kw in ({"z": None}, {"choice": None}, {"weight": None}, {"dweight": None}, {"d": None}, {"dtype": "f64"}, {"ld_dlogits": 7}, {"ld_logits": 7},
               {"score": 5}, {"scale": 0.0}, {"tokens": -1}, {"experts": 1}):
        refused(INVALID, back, **kw)
    for kw in ({"z": P + 1}, {"d": P + 2}, {"choice": P + 2}, {"weight": P + 1}, {"dweight": P + 1}):
        refused(ALIGN, back, **kw)
    back(tokens=0)


def test_balance_refusals():
    b = lambda offsets=P, experts=8, rate=0.1, bias=P, out=P: pf.moe_balance(offsets, experts, rate, bias, out)  # noqa: E731
    for kw in ({"offsets": None}, {"bias": None}, {"out": None}, {"experts": 0}, {"experts": 1025}):
        refused(INVALID, b, **kw)
    for kw in ({"offsets": P + 1}, {"bias": P + 2}, {"out": P + 2}):
        refused(ALIGN, b, **kw)
