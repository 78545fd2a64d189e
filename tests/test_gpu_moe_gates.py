"""SwiGLU and its gradient (include/prefree_moe.h) where the gate's sigmoid leaves the range of normal numbers, on the GPU.

silu(g) is within (8 + |g|) 2^-23 of itself (roundings of the exponent, the exponential, the reciprocal and products), and
where sigmoid(g) is under 2^-142 it may count as 0: with |g| < 110 that is less than 2^-134."""
import pytest
import torch

import prefree_amd as pf
from moe_util import DEV, close, offsets_of

pytestmark = pytest.mark.gpu

FLOOR = 2.0 ** -134


def gates(n):
    """n gates from -109.5 to -80 and some around 0, over and over, as bf16 holds them."""
    values = torch.cat([torch.arange(-109.5, -80, 0.5), torch.tensor([-87.375, -88.75, -20.0, -1.0, -0.0, 0.0, 0.5, 3.0, 90.0, 120.0])])
    return values.bfloat16().float()[torch.arange(n) % values.numel()].to(DEV)


def silu(g, u):
    h = g * torch.sigmoid(g) * u
    return h, (8 + g.abs()) * 2.0 ** -23 * h.abs() + FLOOR * u.abs()


# rows of an expert, experts, n, k: products with few rows, small tiles, tiles a workgroup each, tiles over all CUs
@pytest.mark.parametrize("rows,experts,n,k", [(3, 2, 72, 16), (3, 2, 71, 17), (40, 4, 136, 24), (40, 4, 135, 25), (700, 3, 140, 31),
                                              (300, 16, 520, 32)])
def test_swiglu_at_the_ends_of_the_sigmoid(rows, experts, n, k):
    g = torch.Generator(device=DEV)
    g.manual_seed(n)
    slots = rows * experts
    rest = torch.exp2(torch.randint(-3, 12, (n,), generator=g, device=DEV).float()) * (1 - 2 * (torch.arange(n, device=DEV) % 2))
    w = torch.zeros(experts, 2 * n, k, dtype=torch.bfloat16, device=DEV)
    w[:, :n, 0], w[:, n:, 0] = gates(n), rest
    x = torch.zeros(slots, k, dtype=torch.bfloat16, device=DEV)
    x[:, 0] = 1
    y, pre = (torch.empty(slots, c, dtype=torch.bfloat16, device=DEV) for c in (n, 2 * n))
    pf.moe_mm(x, slots, None, 1, w, offsets_of([rows] * experts), experts, slots, n, k, y, act="swiglu", pre=pre)
    assert (pre == w[0, :, 0]).all()
    h, slack = silu(gates(n).double(), rest.double())
    close(y, h.expand(slots, n), slack.expand(slots, n), "bf16", "silu(gate) * rest")
    big = rest.abs().double() * FLOOR < 2.0 ** -9 * h.abs()
    assert (y[:, big] != 0).all() and int((gates(n) < -87)[big].sum()) > 5


@pytest.mark.parametrize("rows,n,k", [(2, 64, 32), (200, 136, 64), (2000, 1024, 96)])
def test_swiglu_of_4_bit_products_at_the_ends_of_the_sigmoid(rows, n, k):
    gate = -(64.0 + torch.tensor([16.0, 24.0, 32.0], device=DEV)[torch.arange(n, device=DEV) % 3])   # -80, -88, -96
    w = torch.zeros(2 * n, k, device=DEV)
    w[:n, 0], w[:n, 1], w[n:, 0] = -64, gate + 64, 1024   # of scale 16, elements 4 and 1, 3/2 or 2
    x = torch.zeros(rows, k, device=DEV)
    x[:, :2] = 1
    held = []
    for v in (x, w):
        codes = torch.empty(v.shape[0], k // 2, dtype=torch.uint8, device=DEV)
        scales = torch.empty(v.shape[0], k // 32, dtype=torch.uint8, device=DEV)
        pf.mx4_quantize(v, v.shape[0], k, codes, scales, dtype="f32")
        held += [codes, scales]
    y = torch.empty(rows, n, dtype=torch.bfloat16, device=DEV)
    pf.moe_mm_mx4(held[0], held[1], rows, None, 1, held[2], held[3], None, 1, rows, n, k, y, act="swiglu")
    h, slack = silu(gate.double(), torch.full_like(gate, 1024.0).double())
    close(y, h.expand(rows, n), slack.expand(rows, n), "bf16", "silu(gate) * rest")
    assert (y != 0).all()


@pytest.mark.parametrize("n", [136, 77])
def test_swiglu_backward_at_the_ends_of_the_sigmoid(n):
    rows = 65
    g = torch.Generator(device=DEV)
    g.manual_seed(n)
    pre = torch.empty(rows, 2 * n, device=DEV)
    pre[:, :n] = gates(rows * n).view(rows, n)
    pre[:, n:] = torch.randn(rows, n, generator=g, device=DEV) * torch.exp2(torch.randint(-3, 12, (rows, n), generator=g, device=DEV).float())
    pre = pre.bfloat16()
    dh = torch.randn(rows, n, generator=g, device=DEV).bfloat16()
    dpre = torch.empty_like(pre)
    pf.swiglu_backward(dh, pre, rows, n, dpre)
    gate, up, d = pre[:, :n].double(), pre[:, n:].double(), dh.double()
    s = torch.sigmoid(gate)
    # two dozen fp32 roundings, those of the exponent times |g|, of terms that are at most this large
    size = (24 + gate.abs()) * 2.0 ** -23 * d.abs() * (1 + gate.abs()) * s + FLOOR * d.abs()
    close(dpre[:, :n], d * up * s * (1 + gate * (1 - s)), size * up.abs(), "bf16", "gate")
    close(dpre[:, n:], d * gate * s, size, "bf16", "up")
    big = FLOOR < 2.0 ** -9 * (gate * s).abs()
    small = (gate < -88.75) & big & (d.abs() > 0.1)
    assert int(small.sum()) > 50 and (dpre[:, n:][small] != 0).all()
