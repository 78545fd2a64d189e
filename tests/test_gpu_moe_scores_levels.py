"""Routing by scores with biases around a far level: sums of 64 bits, in which scores may be equal that are not alone."""
import pytest
import torch

from moe_util import DEV
from test_gpu_moe_scores import biases, check, logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("level", [1e8, -1e9, 3e9, 1e10, -1e11, 1e12, -1e14, 1e16, -1e30])
def test_biases_of_a_far_level(level, score):
    """From 10^10 on sums of neighbouring scores are equal: the lowest index."""
    z, bias = logits(700, 64, 31), biases(64) + level
    check(z, 6, bias=bias, score=score)
    check(z, 6, bias=bias, score=score, groups=8, groups_kept=3)
    check(z, 6, bias=bias, score=score, groups=8, groups_kept=3, group_best=1)
    z[torch.rand(700, 64, generator=torch.Generator(device=DEV).manual_seed(7), device=DEV) < 0.8] = -float("inf")
    check(z, 4, bias=bias, score=score, groups=16, groups_kept=5)


@pytest.mark.parametrize("level,between", [(1e12, 65536.0), (-3e12, 2.0 ** 19), (1e10, 1024.0), (1e30, 1e30), (-1e38, 2e38)])
def test_levels_some_way_apart(level, between):
    """The sums of each level are equal or not as 64 bits have them, and the levels lie one behind the other."""
    z = logits(700, 64, 32)
    bias = torch.full((64,), level, device=DEV)
    bias[::3] += between
    check(z, 8, bias=bias)
    check(z, 8, bias=bias, groups=8, groups_kept=4)
    bias[::5] = -float("inf")
    check(z, 30 // 2, bias=bias)
