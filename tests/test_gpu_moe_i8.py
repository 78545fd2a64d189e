"""8-bit integers with a scale a row (include/prefree_moe.h): both directions, and products grouped by expert, against 64-bit forms."""
import pytest
import torch

import prefree_amd as pf
from moe_util import DEV, NAN, TORCH, close, groups, offsets_of, strided, swiglu

pytestmark = pytest.mark.gpu


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def integers(x):
    """The integers and scales of rows of x, by whole numbers: 127 |x| / most is compared with halves without a quotient's rounding."""
    x = x.double()
    most = x.abs().amax(dim=1, keepdim=True).clamp(min=2.0 ** -100)
    low = torch.floor(127 * x.abs() / most)
    low = torch.where(low * most > 127 * x.abs(), low - 1, low)
    rest = 127 * x.abs() - low * most                 # 127 x has 31 bits, low * most as many: exact
    up = (2 * rest > most) | ((2 * rest == most) & (low % 2 == 1))
    return (torch.sign(x) * (low + up)).to(torch.int8), most[:, 0]


def quantised(x, rows, k, dtype, ld=0, stream=None):
    codes = torch.full((rows, pf.i8_row(k)), 77, dtype=torch.int8, device=DEV)
    scales = torch.full((rows,), NAN, device=DEV)
    pf.i8_quantize(x, rows, k, codes, scales, dtype=dtype, ld_x=ld, stream=stream)
    torch.cuda.synchronize()
    return codes, scales


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,k,ld,shift", [(1, 1, 0, 0), (3, 7, 0, 0), (5, 16, 0, 0), (2, 17, 0, 1), (1, 2048, 0, 0), (65, 1111, 0, 0),
                                             (7, 4096, 4100, 3), (2, 4097, 0, 0), (3, 9000, 9001, 1), (2049, 130, 0, 0), (2050, 2049, 0, 0),
                                             (2100, 2500, 2512, 0), (2111, 4096, 0, 0), (2051, 5001, 0, 0)])
def test_integers(dtype, rows, k, ld, shift):
    g = gen(rows * 7919 + k)
    x = torch.randn(rows, k, generator=g, device=DEV) * torch.exp2(torch.randint(-9, 9, (rows, 1), generator=g, device=DEV).float())
    x = x.to(TORCH[dtype])
    # halves between integers: the largest magnitude a power of two times 127, elements its multiples of 1/254
    halves = torch.randint(-254, 255, (k,), generator=g, device=DEV) / 2
    halves[0] = -127
    x[0] = halves.to(x.dtype)
    if rows > 2:
        x[1] = 0
        x[2, 0] = 3 * x[2].abs().max()
    view, ld = strided(x, ld, shift)
    codes, scales = quantised(view, rows, k, dtype, ld)
    want, most = integers(x)
    assert torch.equal(codes[:, :k], want)
    assert not codes[:, k:].any()
    assert torch.equal(scales, (most / 127).float())
    for out in ("f32", dtype):
        y, ld_y = strided(torch.full((rows, k), NAN, dtype=TORCH[out], device=DEV), ld, shift, fill=5.0)
        pf.i8_dequantize(codes, scales, rows, k, y, dtype=out, ld_y=ld_y)
        torch.cuda.synchronize()
        assert torch.equal(y, (want.float() * scales[:, None]).to(TORCH[out]))
        assert (y.as_strided((rows - 1, ld_y - k), (ld_y, 1), y.storage_offset() + k) == 5).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,k", [(6, 40), (2500, 40), (6, 3000), (6, 20000)])
def test_rows_without_an_answer(dtype, rows, k):
    x = torch.randn(rows, k, generator=gen(1), device=DEV).to(TORCH[dtype])
    x[0, k - 1], x[1, 3], x[2, k // 2] = float("inf"), float("nan"), -float("inf")
    x[3] = 0
    x[4] *= torch.finfo(x.dtype).tiny
    codes, scales = quantised(x, rows, k, dtype)
    assert scales[:3].isnan().all() and not codes[:3].any()
    want, most = integers(x[3:])
    assert torch.equal(codes[3:, :k], want) and torch.equal(scales[3:], (most / 127).float())


def test_long_rows_and_offsets_past_32_bits():
    rows, k = 3, 1 << 24
    x = torch.randn(rows, k, generator=gen(2), device=DEV).bfloat16()
    codes, scales = quantised(x, rows, k, "bf16")
    for r in range(rows):
        want, most = integers(x[r:r + 1])
        assert torch.equal(codes[r:r + 1], want) and scales[r] == (most[0] / 127).float()
    rows, k = (1 << 20) + 1, 4100            # more than 2^32 bytes of codes
    x = torch.randn(64, k, generator=gen(3), device=DEV).bfloat16()
    big = x.repeat(rows // 64 + 1, 1)[:rows]
    codes, scales = quantised(big, rows, k, "bf16")
    want, most = integers(x)
    for r in (0, 64, 64 * 8189, rows // 64 * 64 - 64):
        assert torch.equal(codes[r:r + 64, :k], want[:min(64, rows - r)])
    assert torch.equal(codes[-1:, :k], want[:1]) and scales[-1] == (most[0] / 127).float()
    y = torch.empty(rows, k, dtype=torch.bfloat16, device=DEV)
    pf.i8_dequantize(codes, scales, rows, k, y, dtype="bf16")
    torch.cuda.synchronize()
    assert torch.equal(y[-1], (want[0].float() * scales[-1]).bfloat16())


def reference(xq, xs, wq, ws, act, n):
    """(y, slack): sums of whole numbers are exact; four roundings of fp32 to scale them."""
    y = (xq.double() @ wq.double().t()) * xs.double()[:, None] * ws.double()
    slack = 4 * 2.0 ** -24 * y.abs()
    if act == "none":
        return y, slack
    return swiglu(y[:, :n], y[:, n:], slack[:, :n], slack[:, n:])


def check(counts, n, k, act="none", dtype="bf16", gather=0, ld_extra=0, tail=0, seed=0, stream=None):
    g = gen(seed + n * 31 + k)
    experts, used = len(counts), sum(counts)
    slots, rows_w = used + tail, (2 if act == "swiglu" else 1) * n
    x_rows = gather or max(slots, 1)
    kp = pf.i8_row(k)
    xq = torch.zeros(x_rows, kp, dtype=torch.int8, device=DEV)
    wq = torch.zeros(experts, rows_w, kp, dtype=torch.int8, device=DEV)
    xq[:, :k] = torch.randint(-127, 128, (x_rows, k), generator=g, device=DEV)
    wq[:, :, :k] = torch.randint(-128, 128, (experts, rows_w, k), generator=g, device=DEV)
    xs = torch.rand(x_rows, generator=g, device=DEV) * 0.02 / k ** 0.5
    ws = torch.rand(experts, rows_w, generator=g, device=DEV) * 0.02
    rows, div = None, 1
    if gather:
        div = 2
        rows = torch.randint(0, x_rows * div, (slots,), generator=g, device=DEV, dtype=torch.int32)
    y, ld = strided(torch.full((slots, n), NAN, dtype=TORCH[dtype], device=DEV), n + ld_extra, 0, fill=NAN)
    offsets = offsets_of(counts)
    pf.moe_mm_i8(xq, xs, x_rows, rows, div, wq, ws, offsets, experts, slots, n, k, y, dtype=dtype, act=act, ld_y=ld, stream=stream)
    torch.cuda.synchronize()
    for e, b, f in groups(counts):
        if f == b:
            continue
        at = rows[b:f].long() // div if gather else torch.arange(b, f, device=DEV)
        ref, slack = reference(xq[at], xs[at], wq[e], ws[e], act, n)
        close(y[b:f], ref, slack, dtype, f"expert {e}")
    assert y[used:].isnan().all()
    if ld_extra:
        assert y.as_strided((slots - 1, ld_extra), (ld, 1), y.storage_offset() + n).isnan().all()


@pytest.mark.parametrize("act", ["none", "swiglu"])
@pytest.mark.parametrize("counts,n,k", [
    ([1], 1, 1), ([1], 16, 64), ([1, 0, 1], 33, 17), ([2, 0, 5, 1], 64, 500), ([8] * 6, 130, 1111),          # few rows: weights to registers
    ([30, 0, 70, 129], 96, 256), ([40, 17, 1, 200], 131, 130), ([64, 64], 257, 48), ([100, 300], 128, 1),    # tiles of 128 x 128
    ([256] * 20, 1024, 512), ([300, 0, 77, 1030, 513] * 8, 520, 100), ([129] * 40, 640, 16),                # 256 x 256, a workgroup a CU
])
def test_product(counts, n, k, act):
    check(counts, n, k, act)


@pytest.mark.parametrize("act", ["none", "swiglu"])
@pytest.mark.parametrize("counts,n,k", [([1, 3, 0, 2], 40, 100), ([60, 90, 0], 100, 333), ([500] * 12, 800, 300)])
def test_gathered_f16_gaps_and_rest(counts, n, k, act):
    check(counts, n, k, act, dtype="f16", gather=37, ld_extra=3, tail=5)


def test_one_expert_without_offsets_and_nothing():
    check([0, 0], 8, 8, tail=3)
    n, k = 24, 40
    xq = torch.randint(-127, 128, (4, pf.i8_row(k)), device=DEV, dtype=torch.int8)
    xq[:, k:] = 0
    one = torch.ones(64, device=DEV)
    y = torch.zeros(4, n, dtype=torch.bfloat16, device=DEV)
    wq = torch.randint(-127, 128, (n, pf.i8_row(k)), device=DEV, dtype=torch.int8)
    wq[:, k:] = 0
    pf.moe_mm_i8(xq, one, 4, None, 1, wq, one, None, 1, 4, n, k, y)
    torch.cuda.synchronize()
    assert torch.equal(y, (xq.double() @ wq.double().t()).bfloat16())
    pf.moe_mm_i8(None, one, 4, None, 1, None, one, None, 1, 4, n, 0, y)
    torch.cuda.synchronize()
    assert not y.any()


@pytest.mark.parametrize("rows", [3, 200])
def test_largest_sums_and_scales_without_a_number(rows):
    """Every product -128 * -128, as many as fit: 2^31 - 2^18; a NaN scale reaches its row or its column alone."""
    n, k = 40, 131056
    xq = torch.full((rows, k), -128, dtype=torch.int8, device=DEV)
    wq = torch.full((n, k), -128, dtype=torch.int8, device=DEV)
    xs, ws = torch.ones(rows, device=DEV), torch.ones(n, device=DEV)
    xs[1], ws[2] = NAN, NAN
    y = torch.zeros(rows, n, dtype=torch.bfloat16, device=DEV)
    pf.moe_mm_i8(xq, xs, rows, None, 1, wq, ws, None, 1, rows, n, k, y)
    torch.cuda.synchronize()
    want = torch.full((rows, n), 16384.0 * k, device=DEV).bfloat16()
    want[1], want[:, 2] = NAN, NAN
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.nan_to_num(), want.nan_to_num())


def test_operand_past_4_gib():
    """Rows behind 32-bit offsets: a product that gathers the last of them."""
    x_rows, k, n = (1 << 20) + 7, 4112, 32
    xq = torch.zeros(x_rows, k, dtype=torch.int8, device=DEV)
    at = torch.tensor([x_rows - 1, 0, x_rows - 7, 12345], dtype=torch.int32, device=DEV)
    xq[at.long()] = torch.randint(-127, 128, (4, k), generator=gen(4), device=DEV, dtype=torch.int8)
    wq = torch.randint(-127, 128, (n, k), generator=gen(5), device=DEV, dtype=torch.int8)
    xs, ws = torch.rand(x_rows, device=DEV), torch.rand(n, device=DEV)
    y = torch.zeros(4, n, dtype=torch.bfloat16, device=DEV)
    pf.moe_mm_i8(xq, xs, x_rows, at, 1, wq, ws, None, 1, 4, n, k, y)
    torch.cuda.synchronize()
    ref, slack = reference(xq[at.long()], xs[at.long()], wq, ws, "none", n)
    close(y, ref, slack, "bf16")


def test_rows_outside_and_offsets_that_decrease_stay_inside():
    """Unspecified rows, but nothing outside of x is read and slots behind the last expert are left."""
    n, k, slots = 64, 128, 40
    xq = torch.randint(-127, 128, (8, k), device=DEV, dtype=torch.int8)
    wq = torch.randint(-127, 128, (3, n, k), device=DEV, dtype=torch.int8)
    one = torch.ones(3 * n, device=DEV)
    rows = torch.tensor([-5, 1 << 30, 8, 7] * 10, dtype=torch.int32, device=DEV)
    y = torch.full((slots, n), NAN, dtype=torch.bfloat16, device=DEV)
    pf.moe_mm_i8(xq, one, 8, rows, 1, wq, one, torch.tensor([0, 20, 10, 30], dtype=torch.int32, device=DEV), 3, slots, n, k, y)
    torch.cuda.synchronize()
    assert y[30:].isnan().all() and y[3].isfinite().all()
    assert torch.equal(y[3].double(), (xq[7].double() @ wq[0].double().t()).bfloat16().double())


@pytest.mark.parametrize("slots", [3, 70, 300])
@pytest.mark.parametrize("x_scale,w_scale", [(2.0 ** 70, 2.0 ** 70), (2.0 ** -90, 2.0 ** -40), (2.0 ** -40, 2.0 ** -90)])
def test_scales_whose_product_is_no_number(slots, x_scale, w_scale):
    """Sums of 0 stay 0, and small scales one after the other lose nothing."""
    n, k = 256, 64
    xq = torch.randint(-127, 128, (slots, k), generator=gen(slots), device=DEV).to(torch.int8)
    wq = torch.randint(-127, 128, (n, k), generator=gen(n), device=DEV).to(torch.int8)
    xq[1], wq[5] = 0, 0
    xs, ws = torch.full((slots,), x_scale, device=DEV), torch.full((n,), w_scale, device=DEV)
    y = torch.full((slots, n), NAN, dtype=torch.bfloat16, device=DEV)
    pf.moe_mm_i8(xq, xs, slots, None, 1, wq, ws, None, 1, slots, n, k, y)
    torch.cuda.synchronize()
    ref = (xq.double() @ wq.double().t()) * x_scale * w_scale
    assert torch.equal(y, ref.float().bfloat16())        # sums under 2^24 and powers of two: one rounding
