"""Grouped products (include/prefree_moe.h) with more experts and tiles than workgroups, on the GPU against plain 64-bit
forms: several tiles a workgroup, tiles with half their rows, short and odd k, and the sizes where another kernel takes
over."""
import numpy as np
import pytest
import torch

import prefree_amd as pf
from moe_util import DEV, NAN, ROUND, TORCH, close, groups, offsets_of, product, strided, swiglu

pytestmark = pytest.mark.gpu


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def counts_for(experts, mean, seed):
    """Uneven counts: some experts without rows, some with one, with a tile's rows and a few around it."""
    r = np.random.RandomState(seed)
    c = r.poisson(mean * r.uniform(0.2, 1.8, experts))
    for at, n in ((0, 0), (3, 1), (5, 256), (6, 257), (7, 128), (8, 129), (experts // 2, 0), (experts - 1, 0)):
        if at < experts:
            c[at] = n if n < 2 or mean >= 64 else c[at]
    return [int(v) for v in c]


# experts, mean rows, n, k: from a few rows an expert to several tiles, k under a tile's, odd in pieces, long
SHAPES = [
    (300, 100, 64, 40), (300, 100, 520, 8), (300, 20, 264, 72), (1024, 2, 256, 64), (700, 30, 24, 136),
    (70, 97, 512, 200), (2, 9000, 1032, 104), (1, 4097, 2064, 264), (300, 8, 40, 512), (600, 1, 264, 2048), (65, 9, 2000, 96),
]


def operands(experts, mean, n, k, dtype, act, gather, seed):
    g = gen(seed)
    counts = counts_for(experts, mean, seed)
    slots = sum(counts) + 3
    tokens = max(1, slots // 2) if gather else slots
    rows = torch.randint(0, tokens * 3, (slots,), generator=g, device=DEV).int() if gather else None
    x = torch.randn(tokens, k, generator=g, device=DEV).to(TORCH[dtype])
    w = (torch.randn(experts, (2 if act else 1) * n, k, generator=g, device=DEV) * k ** -0.5).to(TORCH[dtype])
    return g, counts, slots, rows, x, w


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("experts,mean,n,k", SHAPES)
def test_mm(experts, mean, n, k, dtype):
    for act, gather in ((0, True), (1, False), (1, True)):
        g, counts, slots, rows, x, w = operands(experts, mean, n, k, dtype, act, gather, experts + n)
        x, ld_x = strided(x, k + 8)
        y, ld_y = strided(torch.full((slots, n), 7.0, dtype=TORCH[dtype], device=DEV), n + 8, fill=9.0)
        pre, ld_pre = strided(torch.full((slots, 2 * n), 7.0, dtype=TORCH[dtype], device=DEV), 2 * n + 8, fill=9.0)
        pf.moe_mm(x, x.shape[0], rows, 3, w, offsets_of(counts), experts, slots, n, k, y, dtype=dtype,
                  act="swiglu" if act else "none", pre=pre if act else None, ld_x=ld_x, ld_y=ld_y, ld_pre=ld_pre if act else 0)
        for i, b, f in groups(counts):
            if b == f:
                continue
            z, slack = product(x[(rows[b:f] // 3).long()] if gather else x[b:f], w[i])
            if act:
                close(pre[b:f], z, slack, dtype, f"pre of expert {i}, {f - b} rows")
                z, slack = swiglu(z[:, :n], z[:, n:], slack[:, :n], slack[:, n:])
            close(y[b:f], z, slack, dtype, f"expert {i}, {f - b} rows")
        assert (y[slots - 3:] == 7.0).all() and (not act or (pre[slots - 3:] == 7.0).all())
        assert (torch.as_strided(y, (slots, ld_y), (ld_y, 1))[:, n:] == 9.0).all()
        assert (torch.as_strided(pre, (slots, ld_pre), (ld_pre, 1))[:, 2 * n:] == 9.0).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("experts,mean,n,k", SHAPES)
def test_gradients(experts, mean, n, k, dtype):
    for gather, kind in ((True, "f32"), (False, dtype)):
        g, counts, slots, rows, x, w = operands(experts, mean, n, k, dtype, 0, gather, experts + k)
        dy = torch.randn(slots, n, generator=g, device=DEV).to(TORCH[dtype])
        dy[slots - 3:] = NAN
        dx = torch.full((slots, k), 7.0, dtype=TORCH[dtype], device=DEV)
        dw = torch.full((experts, n, k), NAN, dtype=TORCH[kind], device=DEV)
        off = offsets_of(counts)
        pf.moe_mm_dx(dy, w, off, experts, slots, n, k, dx, dtype=dtype)
        pf.moe_mm_dw(dy, x, x.shape[0], rows, 3, off, experts, slots, n, k, dw, dtype=dtype, dw_dtype=kind)
        for i, b, f in groups(counts):
            xs = x[(rows[b:f] // 3).long()] if gather else x[b:f]
            z, slack = product(dy[b:f], w[i].t())
            close(dx[b:f], z, slack, dtype, f"dx of expert {i}, {f - b} rows")
            z, slack = product(dy[b:f].t(), xs.t())
            close(dw[i], z, slack, kind, f"dw of expert {i}, {f - b} rows")
        assert (dx[slots - 3:] == 7.0).all()


@pytest.mark.parametrize("experts,mean,n,k", [(300, 100, 64, 32), (300, 100, 520, 160), (1024, 2, 256, 64), (70, 97, 512, 224),
                                              (2, 9000, 1032, 96), (300, 8, 40, 512), (600, 1, 264, 2048), (65, 9, 2000, 544)])
def test_mm_mx4(experts, mean, n, k):
    for act, gather, dtype in ((0, True, "f16"), (1, True, "bf16"), (1, False, "bf16")):
        g, counts, slots, rows, x, w = operands(experts, mean, n, k, "bf16", act, gather, experts + n + k)
        x = x * torch.exp2(3 * torch.randn(x.shape[0], 1, generator=g, device=DEV)).to(x.dtype)
        held = []
        for v in (x, w.view(-1, k)):
            codes = torch.empty(v.shape[0], k // 2, dtype=torch.uint8, device=DEV)
            scales = torch.empty(v.shape[0], k // 32, dtype=torch.uint8, device=DEV)
            values = torch.empty(v.shape, device=DEV)
            pf.mx4_quantize(v, v.shape[0], k, codes, scales, dtype="bf16")
            pf.mx4_dequantize(codes, scales, v.shape[0], k, values)
            held.append((codes, scales, values))
        (xq, xs, xv), (wq, ws, wv) = held
        wv = wv.view(w.shape)
        y = torch.full((slots, n), 7.0, dtype=TORCH[dtype], device=DEV)
        pf.moe_mm_mx4(xq, xs, x.shape[0], rows, 3, wq, ws, offsets_of(counts), experts, slots, n, k, y, dtype=dtype,
                      act="swiglu" if act else "none")
        for i, b, f in groups(counts):
            if b == f:
                continue
            z, slack = product(xv[(rows[b:f] // 3).long()] if gather else xv[b:f], wv[i])
            if act:
                z, slack = swiglu(z[:, :n], z[:, n:], slack[:, :n], slack[:, n:])
            close(y[b:f], z, slack, dtype, f"act {act} expert {i}, {f - b} rows")
        assert (y[slots - 3:] == 7.0).all()


@pytest.mark.parametrize("mean", [7, 8, 9, 31, 32, 33, 95, 96, 127, 128])
@pytest.mark.parametrize("n,k,shift", [(136, 264, 0), (135, 263, 0), (135, 263, 1)])
def test_mm_around_the_rows_where_another_kernel_takes_over(mean, n, k, shift):
    g, dtype, experts = gen(mean), "bf16", 150
    counts = [mean] * experts
    counts[4], counts[9], counts[11] = 0, 2 * mean - 1, 1   # the mean stays
    slots = mean * experts
    x, ld_x = strided(torch.randn(slots, k, generator=g, device=DEV).to(TORCH[dtype]), k, shift)
    flat = (torch.randn(experts * n * k + 8, generator=g, device=DEV) * k ** -0.5).to(TORCH[dtype])
    w = flat[shift:shift + experts * n * k].view(experts, n, k)
    y, ld_y = strided(torch.full((slots, n), 7.0, dtype=TORCH[dtype], device=DEV), n, shift)
    pf.moe_mm(x, slots, None, 1, w, offsets_of(counts), experts, slots, n, k, y, dtype=dtype, ld_x=ld_x, ld_y=ld_y)
    for i, b, f in groups(counts):
        if b < f:
            z, slack = product(x[b:f], w[i])
            close(y[b:f], z, slack, dtype, f"expert {i}")


@pytest.mark.parametrize("experts", [5, 150])
@pytest.mark.parametrize("mean", [3, 4, 5, 23, 24, 25, 300])
def test_mm_unaligned_around_the_rows_where_another_kernel_takes_over(mean, experts):
    g, dtype, n, k = gen(mean), "f16", 70, 331
    counts = [mean] * experts
    counts[1], counts[3], counts[4] = 0, 2 * mean - 1, 1
    slots = mean * experts
    x = torch.randn(slots, k, generator=g, device=DEV).to(TORCH[dtype])
    for act in (0, 1):
        w = (torch.randn(experts, (1 + act) * n, k, generator=g, device=DEV) * k ** -0.5).to(TORCH[dtype])
        y, ld_y = strided(torch.full((slots, n), 7.0, dtype=TORCH[dtype], device=DEV), n, 1)
        pf.moe_mm(x, slots, None, 1, w, offsets_of(counts), experts, slots, n, k, y, dtype=dtype, act="swiglu" if act else "none", ld_y=ld_y)
        for i, b, f in groups(counts):
            if b == f:
                continue
            z, slack = product(x[b:f], w[i])
            if act:
                z, slack = swiglu(z[:, :n], z[:, n:], slack[:, :n], slack[:, n:])
            close(y[b:f], z, slack, dtype, f"expert {i}")


def test_mm_values_behind_unaligned_rows_do_not_matter():
    """Rows of odd length that start at odd elements, with NaN around them: the words that are loaded hold some of it."""
    g, dtype = gen(8), "bf16"
    for experts, mean, n, k in ((5, 3, 9, 31), (5, 40, 67, 33), (40, 200, 70, 97), (3, 700, 33, 1)):
        counts = [mean] * experts
        slots = mean * experts
        x, ld_x = strided(torch.randn(slots, k, generator=g, device=DEV).to(TORCH[dtype]), k + 2, 1)
        flat = torch.full((experts * n * k + 9,), NAN, dtype=TORCH[dtype], device=DEV)
        w = flat[3:3 + experts * n * k].view(experts, n, k)
        w.copy_(torch.randn(experts, n, k, generator=g, device=DEV) * k ** -0.5)
        dy, ld_dy = strided(torch.randn(slots, n, generator=g, device=DEV).to(TORCH[dtype]), n + 2, 1)
        y, dx, dw = (torch.empty(*s, dtype=t, device=DEV) for s, t in (((slots, n), TORCH[dtype]), ((slots, k), TORCH[dtype]), ((experts, n, k), torch.float32)))
        off = offsets_of(counts)
        pf.moe_mm(x, slots, None, 1, w, off, experts, slots, n, k, y, dtype=dtype, ld_x=ld_x)
        pf.moe_mm_dx(dy, w, off, experts, slots, n, k, dx, dtype=dtype, ld_dy=ld_dy)
        pf.moe_mm_dw(dy, x, slots, None, 1, off, experts, slots, n, k, dw, dtype=dtype, dw_dtype="f32", ld_dy=ld_dy, ld_x=ld_x)
        for i, b, f in groups(counts):
            close(y[b:f], *product(x[b:f], w[i]), dtype, "y")
            close(dx[b:f], *product(dy[b:f], w[i].t()), dtype, "dx")
            close(dw[i], *product(dy[b:f].t(), x[b:f].t()), "f32", "dw")


def test_same_bits_each_time():
    g, counts, slots, rows, x, w = operands(300, 60, 264, 136, "bf16", 1, True, 5)
    off = offsets_of(counts)
    got = []
    for _ in range(3):
        y, pre = (torch.empty(slots, c, dtype=torch.bfloat16, device=DEV).fill_(1.0) for c in (264, 528))
        dw, dx = torch.empty_like(w), torch.empty(slots, 136, dtype=torch.bfloat16, device=DEV).fill_(1.0)
        pf.moe_mm(x, x.shape[0], rows, 3, w, off, 300, slots, 264, 136, y, act="swiglu", pre=pre)
        pf.moe_mm_dx(pre, w, off, 300, slots, 528, 136, dx)
        pf.moe_mm_dw(pre, x, x.shape[0], rows, 3, off, 300, slots, 528, 136, dw)
        got.append((y, pre, dx, dw))
    for again in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], again))


def test_broken_offsets_and_rows_stay_inside():
    """Offsets that decrease or pass the slots, and row indices outside x: unspecified rows, and no fault."""
    g, experts, slots, n, k = gen(1), 300, 3000, 264, 64
    r = np.random.RandomState(2)
    x, w = (torch.randn(*s, generator=g, device=DEV).bfloat16() for s in ((30, k), (experts, n, k)))
    rows = torch.tensor([-1, 30, 2 ** 31 - 1, -2 ** 31] * (slots // 4), dtype=torch.int32, device=DEV)
    xq, wq = (torch.randint(0, 256, (v, k // 2), generator=g, device=DEV).to(torch.uint8) for v in (30, experts * n))
    xs, ws = (torch.full((v, k // 32), 127, dtype=torch.uint8, device=DEV) for v in (30, experts * n))
    for off in (r.randint(0, slots, experts + 1), r.randint(-2 ** 31, 2 ** 31 - 1, experts + 1), np.arange(experts + 1) % 2 * 10 * slots):
        o = torch.tensor(off.astype(np.int32), device=DEV)
        y, dx, dw = torch.empty(slots, n, dtype=torch.bfloat16, device=DEV), torch.empty(slots, k, dtype=torch.bfloat16, device=DEV), torch.empty(experts, n, k, device=DEV)
        y.fill_(1.0)
        pf.moe_mm(x, 30, rows, 1, w, o, experts, slots, n, k, y)
        pf.moe_mm_dx(y, w, o, experts, slots, n, k, dx)
        pf.moe_mm_dw(y, x, 30, rows, 1, o, experts, slots, n, k, dw, dw_dtype="f32")
        pf.moe_mm_mx4(xq, xs, 30, rows, 1, wq, ws, o, experts, slots, n, k, y)
        torch.cuda.synchronize()


def test_mx4_codes_past_32_bits():
    """Rows of x, and rows of one expert's weights, behind 4 GiB of codes."""
    g, k, m, n = gen(4), 4096, 40, 48
    rows_all = 2 ** 21 + 100
    codes = torch.zeros(rows_all, k // 2, dtype=torch.uint8, device=DEV)
    scales = torch.full((rows_all, k // 32), 127, dtype=torch.uint8, device=DEV)
    small = torch.randn(m, k, generator=g, device=DEV)
    pf.mx4_quantize(small, m, k, codes[-m:], scales[-m:], dtype="f32")
    held = torch.empty(m, k, device=DEV)
    pf.mx4_dequantize(codes[-m:], scales[-m:], m, k, held)
    other = torch.randn(n, k, generator=g, device=DEV) * k ** -0.5
    oc, os_ = torch.empty(n, k // 2, dtype=torch.uint8, device=DEV), torch.empty(n, k // 32, dtype=torch.uint8, device=DEV)
    ov = torch.empty(n, k, device=DEV)
    pf.mx4_quantize(other, n, k, oc, os_, dtype="f32")
    pf.mx4_dequantize(oc, os_, n, k, ov)
    rows = torch.arange(rows_all - m, rows_all, device=DEV).int()
    y = torch.empty(m, n, dtype=torch.bfloat16, device=DEV)
    pf.moe_mm_mx4(codes, scales, rows_all, rows, 1, oc, os_, None, 1, m, n, k, y)
    z, slack = product(held, ov)
    close(y, z, slack, "bf16", "x")
    y = torch.empty(n, rows_all, dtype=torch.bfloat16, device=DEV)
    pf.moe_mm_mx4(oc, os_, n, None, 1, codes, scales, None, 1, n, rows_all, k, y)
    z, slack = product(ov, held)
    close(y[:, -m:], z, slack, "bf16", "w")
    assert (y[:, :-m] == 0).all()
