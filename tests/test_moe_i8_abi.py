"""8-bit integers (include/prefree_moe.h) — CPU only: refusals before any launch."""
import pytest

import prefree_amd as pf
from test_moe_abi import ALIGN, INVALID, P, refused


def quantize(x=P, rows=2, k=40, codes=P, scales=P, **kw):
    pf.i8_quantize(x, rows, k, codes, scales, **kw)


@pytest.mark.parametrize("kw", [{"x": None}, {"codes": None}, {"scales": None}, {"k": 0}, {"k": -1}, {"k": (1 << 24) + 1}, {"rows": -1},
                                {"dtype": "f64"}, {"ld_x": 39}, {"ld_x": -1}])
def test_quantize_refusals(kw):
    refused(INVALID, quantize, **kw)


def test_quantize_alignment_and_nothing_to_do():
    refused(ALIGN, quantize, codes=P + 8)
    refused(ALIGN, quantize, scales=P + 2)
    refused(ALIGN, quantize, x=P + 1)
    refused(ALIGN, quantize, x=P + 2, dtype="f32")
    quantize(rows=0)


def test_dequantize_refusals():
    d = lambda codes=P, scales=P, rows=2, k=40, y=P, **kw: pf.i8_dequantize(codes, scales, rows, k, y, **kw)  # noqa: E731
    for kw in ({"codes": None}, {"scales": None}, {"y": None}, {"k": 0}, {"rows": -1}, {"ld_y": 39}, {"dtype": "f64"}):
        refused(INVALID, d, **kw)
    for kw in ({"codes": P + 1}, {"scales": P + 1}, {"y": P + 2}):
        refused(ALIGN, d, **kw)
    d(rows=0)


def mm(xq=P, xs=P, x_rows=10, rows=P, row_div=1, wq=P, ws=P, offsets=P, experts=4, slots=10, n=64, k=64, y=P, **kw):
    pf.moe_mm_i8(xq, xs, x_rows, rows, row_div, wq, ws, offsets, experts, slots, n, k, y, **kw)


@pytest.mark.parametrize("kw", [{"xq": None}, {"xs": None}, {"wq": None}, {"ws": None}, {"y": None}, {"k": 131057}, {"k": -1}, {"n": -1},
                                {"dtype": "f32"}, {"x_rows": 0}, {"rows": None, "x_rows": 9}, {"row_div": 0}, {"act": 5}, {"ld_y": 5},
                                {"offsets": None}, {"experts": 0}, {"experts": 1025}, {"slots": -1}])
def test_mm_refusals(kw):
    refused(INVALID, mm, **kw)


def test_mm_alignment_and_nothing_to_do():
    for kw in ({"xq": P + 8}, {"wq": P + 4}, {"y": P + 1}, {"xs": P + 2}, {"ws": P + 1}, {"rows": P + 2}, {"offsets": P + 2}):
        refused(ALIGN, mm, **kw)
    mm(slots=0)
    mm(n=0)


def test_wrong_tensor_types_are_refused_in_python():
    torch = pytest.importorskip("torch")
    with pytest.raises(TypeError):
        quantize(codes=torch.zeros(2, 48, dtype=torch.uint8))
    with pytest.raises(TypeError):
        quantize(codes=torch.zeros(2, 48, dtype=torch.int8))        # not on the GPU
    with pytest.raises(TypeError):
        mm(xs=torch.zeros(10, dtype=torch.float64))
    assert [pf.i8_row(k) for k in (1, 16, 17, 1111)] == [16, 16, 32, 1120]
