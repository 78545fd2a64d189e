"""Expert-layer operators of the MI355X library: routing, products grouped by expert, 4-bit blocks.

The same calls as include/prefree_moe.h, which says what each computes, on device buffers as in the rest of this
package: anything with ``data_ptr()``, outputs given by the caller, sizes as numbers, ``stream=None`` the null stream,
errors raised as PrefreeError.  Sizes are not read from the tensors, but a tensor's type and device are checked against
what the call takes.  Leading dimensions (``ld_*``) count elements, 0 standing for the row's length.  No counterpart in
the reference.
"""
from __future__ import annotations

import ctypes

from . import BF16, F16, F32, _check, _s, dtype_code, lib

ACTIVATIONS = {"none": 0, "swiglu": 1}

_vp = ctypes.c_void_p
_i = ctypes.c_int
_ll = ctypes.c_longlong

_SIGNATURES = {
    "pf_moe_route": [_vp, _ll, _i, _i, _i, _i, _i, _vp, _vp, _vp, _vp, _vp, _vp, ctypes.c_size_t, _vp],
    "pf_moe_route_backward": [_vp, _ll, _i, _i, _i, _i, _i, _vp, _vp, _vp, _vp, _ll, _vp],
    "pf_moe_combine": [_vp, _ll, _i, _i, _vp, _vp, _i, _i, _i, _vp, _ll, _vp],
    "pf_moe_combine_backward": [_vp, _ll, _vp, _ll, _i, _i, _vp, _vp, _i, _i, _i, _vp, _ll, _vp, _vp],
    "pf_moe_mm": [_vp, _ll, _i, _vp, _i, _vp, _vp, _i, _i, _i, _i, _i, _i, _vp, _ll, _vp, _ll, _vp],
    "pf_moe_mm_dx": [_vp, _ll, _vp, _vp, _i, _i, _i, _i, _i, _vp, _ll, _vp],
    "pf_moe_mm_dw": [_vp, _ll, _vp, _ll, _i, _vp, _i, _vp, _i, _i, _i, _i, _i, _vp, _i, _vp],
    "pf_swiglu_backward": [_vp, _ll, _vp, _ll, _i, _i, _i, _vp, _ll, _vp],
    "pf_mx4_quantize": [_vp, _ll, _i, _i, _i, _vp, _vp, _vp],
    "pf_mx4_dequantize": [_vp, _vp, _i, _i, _i, _vp, _ll, _vp],
    "pf_moe_mm_mx4": [_vp, _vp, _i, _vp, _i, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _vp, _ll, _vp],
}


def _signatures(L):
    for name, args in _SIGNATURES.items():
        f = getattr(L, name)
        f.argtypes = args
        f.restype = _i
    L.pf_moe_route_workspace.argtypes = [_i, _i]
    L.pf_moe_route_workspace.restype = ctypes.c_size_t


# Type of a buffer, by what its `dtype` is: kept per type object, since these calls are a few microseconds long.
_KINDS = {}


def _kind(dtype):
    text = str(dtype)
    if text.endswith("int32") and "uint32" not in text:
        return "i32"
    if text.endswith("uint8"):
        return "u8"
    if any(w in text for w in ("int", "bool", "complex", "float8")):
        return text
    try:
        return dtype_code(dtype)
    except ValueError:
        return text


def _buf(obj, kind, name):
    """Raw pointer of `obj`, whose type (where it says one) has to be `kind`: a code of this package, "i32" or "u8"."""
    try:
        if _KINDS[obj.dtype] == kind and obj.is_cuda:
            return obj.data_ptr()
    except (AttributeError, KeyError):
        pass
    return _buf_checked(obj, kind, name)


def _buf_checked(obj, kind, name):
    """_buf for what it has not seen; kind None: of any type."""
    if obj is None or isinstance(obj, int):
        return obj
    dtype = getattr(obj, "dtype", None)
    if dtype is not None and kind is not None:
        if dtype not in _KINDS:
            _KINDS[dtype] = _kind(dtype)
        if _KINDS[dtype] != kind:
            raise TypeError(f"{name} is {dtype}")
    if not getattr(obj, "is_cuda", True):
        raise TypeError(f"{name} is on {obj.device}, not on the GPU")
    return obj.data_ptr()


def _act(act):
    return act if isinstance(act, int) else ACTIVATIONS[act]


def moe_route_workspace(tokens, experts) -> int:
    """Bytes of workspace that moe_route takes."""
    return int(lib().pf_moe_route_workspace(int(tokens), int(experts)))


def moe_route(logits, tokens, experts, top_k, choice, weight, offsets, order, slot, workspace, dtype="f32",
              normalise=True, workspace_bytes=None, ld_logits=0, stream=None):
    """The top_k experts of each token with their weights, and the chosen entries ordered by expert."""
    d = dtype_code(dtype)
    if workspace_bytes is None:
        workspace_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    _check(lib().pf_moe_route(_buf(logits, d, "logits"), ld_logits, d, int(tokens), int(experts), int(top_k),
                              int(bool(normalise)), _buf(choice, "i32", "choice"), _buf(weight, F32, "weight"),
                              _buf(offsets, "i32", "offsets"), _buf(order, "i32", "order"), _buf(slot, "i32", "slot"),
                              _buf_checked(workspace, None, "workspace"), int(workspace_bytes), _s(stream)), "pf_moe_route")


def moe_route_backward(logits, tokens, experts, top_k, choice, weight, dweight, dlogits, dtype="f32", normalise=True,
                       ld_logits=0, ld_dlogits=0, stream=None):
    """dlogits from dweight, with the choice and the weights that moe_route wrote."""
    d = dtype_code(dtype)
    _check(lib().pf_moe_route_backward(_buf(logits, d, "logits"), ld_logits, d, int(tokens), int(experts), int(top_k),
                                       int(bool(normalise)), _buf(choice, "i32", "choice"), _buf(weight, F32, "weight"),
                                       _buf(dweight, F32, "dweight"), _buf(dlogits, d, "dlogits"), ld_dlogits,
                                       _s(stream)), "pf_moe_route_backward")


def moe_combine(y, slot, weight, tokens, top_k, width, out, dtype="bf16", slots=None, ld_y=0, ld_out=0, stream=None):
    """out[t] = sum over j of weight[t, j] * y[slot[t, j]]; weight None: all 1.  slots: rows of y (tokens * top_k)."""
    d = dtype_code(dtype)
    slots = int(tokens) * int(top_k) if slots is None else int(slots)
    _check(lib().pf_moe_combine(_buf(y, d, "y"), ld_y, d, slots, _buf(slot, "i32", "slot"), _buf(weight, F32, "weight"),
                                int(tokens), int(top_k), int(width), _buf(out, d, "out"), ld_out, _s(stream)),
           "pf_moe_combine")


def moe_combine_backward(dout, y, slot, weight, tokens, top_k, width, dy, dweight, dtype="bf16", slots=None, ld_dout=0,
                         ld_y=0, ld_dy=0, stream=None):
    """dy[slot[t, j]] = weight[t, j] * dout[t] and dweight[t, j] = <dout[t], y[slot[t, j]]>."""
    d = dtype_code(dtype)
    slots = int(tokens) * int(top_k) if slots is None else int(slots)
    _check(lib().pf_moe_combine_backward(_buf(dout, d, "dout"), ld_dout, _buf(y, d, "y"), ld_y, d, slots,
                                         _buf(slot, "i32", "slot"), _buf(weight, F32, "weight"), int(tokens),
                                         int(top_k), int(width), _buf(dy, d, "dy"), ld_dy,
                                         _buf(dweight, F32, "dweight"), _s(stream)), "pf_moe_combine_backward")


def moe_mm(x, x_rows, rows, row_div, w, offsets, experts, slots, n, k, y, dtype="bf16", act="none", pre=None, ld_x=0,
           ld_y=0, ld_pre=0, stream=None):
    """y[s] = act(x[rows[s] // row_div] w[e]^T) for the slots s of each expert e; rows None: x has a row a slot."""
    d = dtype_code(dtype)
    _check(lib().pf_moe_mm(_buf(x, d, "x"), ld_x, int(x_rows), _buf(rows, "i32", "rows"), int(row_div), _buf(w, d, "w"),
                           _buf(offsets, "i32", "offsets"), int(experts), int(slots), int(n), int(k), d, _act(act),
                           _buf(y, d, "y"), ld_y, _buf(pre, d, "pre"), ld_pre, _s(stream)), "pf_moe_mm")


def moe_mm_dx(dy, w, offsets, experts, slots, n, k, dx, dtype="bf16", ld_dy=0, ld_dx=0, stream=None):
    """dx[s] = dy[s] w[e] for the slots s of each expert e."""
    d = dtype_code(dtype)
    _check(lib().pf_moe_mm_dx(_buf(dy, d, "dy"), ld_dy, _buf(w, d, "w"), _buf(offsets, "i32", "offsets"), int(experts),
                              int(slots), int(n), int(k), d, _buf(dx, d, "dx"), ld_dx, _s(stream)), "pf_moe_mm_dx")


def moe_mm_dw(dy, x, x_rows, rows, row_div, offsets, experts, slots, n, k, dw, dtype="bf16", dw_dtype=None, ld_dy=0,
              ld_x=0, stream=None):
    """dw[e] = sum over the slots s of e of dy[s]^T x[rows[s] // row_div]; dw_dtype: dtype (None) or "f32"."""
    d = dtype_code(dtype)
    dw_d = d if dw_dtype is None else dtype_code(dw_dtype)
    _check(lib().pf_moe_mm_dw(_buf(dy, d, "dy"), ld_dy, _buf(x, d, "x"), ld_x, int(x_rows), _buf(rows, "i32", "rows"),
                              int(row_div), _buf(offsets, "i32", "offsets"), int(experts), int(slots), int(n), int(k), d,
                              _buf(dw, dw_d, "dw"), dw_d, _s(stream)), "pf_moe_mm_dw")


def swiglu_backward(dh, pre, rows, n, dpre, dtype="bf16", ld_dh=0, ld_pre=0, ld_dpre=0, stream=None):
    """dpre [rows, 2n] from dh [rows, n] and the pre-activations [rows, 2n] that moe_mm wrote."""
    d = dtype_code(dtype)
    _check(lib().pf_swiglu_backward(_buf(dh, d, "dh"), ld_dh, _buf(pre, d, "pre"), ld_pre, d, int(rows), int(n),
                                    _buf(dpre, d, "dpre"), ld_dpre, _s(stream)), "pf_swiglu_backward")


def mx4_quantize(x, rows, k, codes, scales, dtype="bf16", ld_x=0, stream=None):
    """x [rows, k] to 4-bit blocks: codes [rows, k/2] and scales [rows, k/32], both uint8."""
    d = dtype_code(dtype)
    _check(lib().pf_mx4_quantize(_buf(x, d, "x"), ld_x, d, int(rows), int(k), _buf(codes, "u8", "codes"),
                                 _buf(scales, "u8", "scales"), _s(stream)), "pf_mx4_quantize")


def mx4_dequantize(codes, scales, rows, k, y, dtype="f32", ld_y=0, stream=None):
    """What 4-bit blocks stand for, in y [rows, k]."""
    d = dtype_code(dtype)
    _check(lib().pf_mx4_dequantize(_buf(codes, "u8", "codes"), _buf(scales, "u8", "scales"), int(rows), int(k), d,
                                   _buf(y, d, "y"), ld_y, _s(stream)), "pf_mx4_dequantize")


def moe_mm_mx4(x_codes, x_scales, x_rows, rows, row_div, w_codes, w_scales, offsets, experts, slots, n, k, y,
               dtype="bf16", act="none", ld_y=0, stream=None):
    """moe_mm of 4-bit operands; y in `dtype`."""
    d = dtype_code(dtype)
    _check(lib().pf_moe_mm_mx4(_buf(x_codes, "u8", "x_codes"), _buf(x_scales, "u8", "x_scales"), int(x_rows),
                               _buf(rows, "i32", "rows"), int(row_div), _buf(w_codes, "u8", "w_codes"),
                               _buf(w_scales, "u8", "w_scales"), _buf(offsets, "i32", "offsets"), int(experts),
                               int(slots), int(n), int(k), d, _act(act), _buf(y, d, "y"), ld_y, _s(stream)),
           "pf_moe_mm_mx4")


__all__ = ["BF16", "F16", "ACTIVATIONS", "moe_route_workspace", "moe_route", "moe_route_backward", "moe_combine",
           "moe_combine_backward", "moe_mm", "moe_mm_dx", "moe_mm_dw", "swiglu_backward", "mx4_quantize",
           "mx4_dequantize", "moe_mm_mx4"]
