"""C ABI of the expert-layer operators (include/prefree_moe.h) — CPU only: exports, and refusals before any launch."""
import os
import re
import subprocess

import pytest

import prefree_amd as pf

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 4096       # a pointer that is never followed: every call here is refused, or has nothing to do


def declared(header):
    text = open(os.path.join(REPO, "include", header)).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"\b(pfk?_[a-z0-9_]+)\s*\(", text)))


@pytest.mark.parametrize("header,path", [("prefree_moe.h", pf.LIB_PATH), ("prefree_moe_kernels.h", pf.KLIB_PATH)])
def test_declared_functions_are_exported(header, path):
    out = subprocess.run(["nm", "-D", "--defined-only", path], capture_output=True, text=True, check=True).stdout
    have = {line.split()[-1] for line in out.splitlines() if line.strip()}
    names = declared(header)
    assert len(names) >= 11 and not [n for n in names if n not in have]
    assert not [n for n in have if "internal" in n]


def test_header_is_c():
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-fsyntax-only", "-x", "c",
                    os.path.join(REPO, "include", "prefree_moe.h")], check=True)


def refused(status, call, *args, **kwargs):
    with pytest.raises(pf.PrefreeError) as e:
        call(*args, **kwargs)
    assert e.value.status == status
    assert str(e.value)


INVALID, ALIGN = 1, 2


def route(tokens=100, experts=8, top_k=2, logits=P, dtype="f32", work=P, work_bytes=1 << 20, ld=0, offsets=P):
    pf.moe_route(logits, tokens, experts, top_k, P, P, offsets, P, P, work, dtype=dtype, workspace_bytes=work_bytes, ld_logits=ld)


@pytest.mark.parametrize("kw", [{"tokens": -1}, {"experts": 0}, {"experts": 1025}, {"top_k": 0}, {"top_k": 9}, {"experts": 64, "top_k": 17},
                                {"logits": None}, {"offsets": None}, {"dtype": "f64"}, {"work": None}, {"work_bytes": 63}, {"ld": 7},
                                {"ld": -1}, {"tokens": 1 << 30}])
def test_route_refusals(kw):
    refused(INVALID, route, **kw)


def test_route_alignment():
    refused(ALIGN, route, logits=P + 2)
    refused(ALIGN, route, work=P + 2)


def mm(n=64, k=64, slots=10, experts=4, offsets=P, x_rows=10, rows=P, row_div=1, x=P, w=P, y=P, dtype="bf16", act="none", pre=None, **ld):
    pf.moe_mm(x, x_rows, rows, row_div, w, offsets, experts, slots, n, k, y, dtype=dtype, act=act, pre=pre, **ld)


@pytest.mark.parametrize("kw", [{"n": -1}, {"k": -1}, {"slots": -1}, {"experts": 0}, {"experts": 2000}, {"offsets": None}, {"x_rows": 0},
                                {"rows": None, "x_rows": 9}, {"row_div": 0}, {"x": None}, {"w": None}, {"y": None}, {"dtype": "f32"},
                                {"act": 2}, {"pre": P}, {"ld_x": 63}, {"ld_y": 3}, {"act": "swiglu", "pre": P, "ld_pre": 64}, {"n": 1 << 25}])
def test_mm_refusals(kw):
    refused(INVALID, mm, **kw)


def test_mm_alignment_and_nothing_to_do():
    for name in ("x", "w", "y"):
        refused(ALIGN, mm, **{name: P + 1})
    mm(slots=0)
    mm(n=0)


def test_gradient_refusals():
    dx = lambda n=64, k=64, dy=P, w=P, out=P, dtype="bf16", **ld: pf.moe_mm_dx(dy, w, P, 4, 10, n, k, out, dtype=dtype, **ld)  # noqa: E731
    for kw in ({"n": -1}, {"dy": None}, {"w": None}, {"out": None}, {"dtype": "f32"}, {"ld_dy": 1}, {"ld_dx": 1}):
        refused(INVALID, dx, **kw)
    refused(ALIGN, dx, dy=P + 1)
    dw = lambda dy=P, x=P, x_rows=10, rows=P, div=1, out=P, slots=10, dtype="bf16", dw_dtype="f32", **ld: pf.moe_mm_dw(  # noqa: E731
        dy, x, x_rows, rows, div, P, 4, slots, 64, 64, out, dtype=dtype, dw_dtype=dw_dtype, **ld)
    for kw in ({"dy": None}, {"x": None}, {"out": None}, {"x_rows": 0}, {"rows": None, "x_rows": 3}, {"div": 0}, {"dw_dtype": "f16"},
               {"dtype": "f32"}, {"slots": -1}, {"ld_x": 2}, {"ld_dy": 2}):
        refused(INVALID, dw, **kw)
    refused(ALIGN, dw, out=P + 2)
    refused(INVALID, pf.swiglu_backward, P, P, -1, 4, P)
    refused(INVALID, pf.swiglu_backward, None, P, 1, 4, P)
    refused(INVALID, pf.swiglu_backward, P, P, 1, 4, P, ld_pre=7)
    refused(ALIGN, pf.swiglu_backward, P, P + 1, 1, 4, P)


def test_combine_refusals():
    c = lambda y=P, slot=P, w=P, t=4, k=2, width=64, out=P, **kw: pf.moe_combine(y, slot, w, t, k, width, out, **kw)  # noqa: E731
    for kw in ({"y": None}, {"slot": None}, {"out": None}, {"t": -1}, {"k": 0}, {"k": 17}, {"width": -1}, {"dtype": "f32"}, {"slots": -1}, {"ld_y": 5}):
        refused(INVALID, c, **kw)
    refused(ALIGN, c, out=P + 1)
    c(t=0)
    b = lambda dout=P, y=P, slot=P, w=P, dy=P, dw=P, **kw: pf.moe_combine_backward(dout, y, slot, w, 4, 2, 64, dy, dw, **kw)  # noqa: E731
    for kw in ({"dout": None}, {"y": None}, {"slot": None}, {"dy": None}, {"dw": None}, {"dtype": "f64"}, {"ld_dy": 5}):
        refused(INVALID, b, **kw)
    refused(ALIGN, b, dy=P + 1)
    back = lambda z=P, choice=P, d=P, **kw: pf.moe_route_backward(z, 4, 8, 2, choice, P, P, d, **kw)  # noqa: E731
    for kw in ({"z": None}, {"choice": None}, {"d": None}, {"dtype": "f64"}, {"ld_dlogits": 7}):
        refused(INVALID, back, **kw)


def test_mx4_refusals():
    q = lambda x=P, rows=2, k=64, codes=P, scales=P, **kw: pf.mx4_quantize(x, rows, k, codes, scales, **kw)  # noqa: E731
    for kw in ({"x": None}, {"codes": None}, {"scales": None}, {"k": 40}, {"rows": -1}, {"dtype": "f64"}, {"ld_x": 32}):
        refused(INVALID, q, **kw)
    refused(ALIGN, q, codes=P + 4)
    refused(ALIGN, q, x=P + 1)
    q(rows=0)
    d = lambda codes=P, scales=P, k=64, y=P, **kw: pf.mx4_dequantize(codes, scales, 2, k, y, **kw)  # noqa: E731
    for kw in ({"codes": None}, {"scales": None}, {"y": None}, {"k": 33}, {"ld_y": 2}):
        refused(INVALID, d, **kw)
    m = lambda xq=P, xs=P, wq=P, ws=P, k=64, y=P, x_rows=10, **kw: pf.moe_mm_mx4(xq, xs, x_rows, P, 1, wq, ws, P, 4, 10, 64, k, y, **kw)  # noqa: E731
    for kw in ({"xq": None}, {"xs": None}, {"wq": None}, {"ws": None}, {"y": None}, {"k": 48}, {"dtype": "f32"}, {"x_rows": 0}, {"act": 5}, {"ld_y": 5}):
        refused(INVALID, m, **kw)
    refused(ALIGN, m, wq=P + 8)


def test_wrong_tensor_types_are_refused_in_python():
    torch = pytest.importorskip("torch")
    host = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        pf.mx4_quantize(host, 4, 64, P, P)                          # not on the GPU
    with pytest.raises(TypeError):
        pf.mx4_quantize(host.float(), 4, 64, P, P, dtype="bf16")
    with pytest.raises(TypeError):
        pf.moe_combine(P, torch.zeros(8, dtype=torch.int64), P, 4, 2, 64, P)


def test_spmv_refuses_bf16():
    with pytest.raises(pf.PrefreeError) as e:
        pf.spmv(P, P, P, P, P, 4, 4, 4, dtype="bf16")
    assert e.value.status == INVALID
