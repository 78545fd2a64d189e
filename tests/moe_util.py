"""Plain 64-bit forms of the expert-layer operators and what their tests share.

Tolerances come from the number formats.  A sum of K products of 16-bit values formed in fp32 in any order is off by at
most (K + 2) 2^-23 sum|a b| (2^-23, twice the rounding of one addition, covers matrix units that truncate), and the
result is rounded once: relative 2^-8 (bf16) or 2^-11 (f16), absolute 2^-25 where f16 is subnormal.
"""
import numpy as np
import torch

import prefree_amd as pf

DEV = "cuda:0"
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ROUND = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}
TINY = {"f16": 2.0 ** -24, "bf16": 2.0 ** -126, "f32": 2.0 ** -126}
NAN = float("nan")


def strided(t, ld=0, shift=0, fill=NAN):
    """`t` [rows, cols] in rows of `ld` elements that start `shift` elements into an allocation; the gaps hold `fill`.

    Returns the tensor view and the ld to pass."""
    rows, cols = t.shape
    ld = max(ld or cols, 1)
    flat = torch.full((rows * ld + shift + 64,), fill, dtype=t.dtype, device=t.device)
    view = flat[shift:shift + rows * ld].view(rows, ld)[:, :cols]
    view.copy_(t)
    return view, ld


def route_reference(z, top_k, normalise):
    """choice, weight, offsets, order, slot of logits z [tokens, experts] (float64, -inf and NaN allowed), by numpy."""
    z = np.asarray(z, dtype=np.float64)
    tokens, experts = z.shape
    nan = np.isnan(z)
    first = np.argsort(-np.where(nan, np.inf, z), axis=1, kind="stable")
    second = np.argsort(~np.take_along_axis(nan, first, 1), axis=1, kind="stable")
    index = np.take_along_axis(first, second, 1)[:, :top_k]
    top = np.take_along_axis(z, index, 1)
    chosen = ~(top == -np.inf)
    choice = np.where(chosen, index, -1).astype(np.int32)
    with np.errstate(all="ignore"):
        base = np.where(chosen[:, :1], top[:, :1], 0.0)
        part = np.exp(top - base)
        total = np.where(chosen, part, 0.0).sum(1, keepdims=True) if normalise else np.exp(z - base).sum(1, keepdims=True)
        weight = np.where(chosen, part / total, 0.0)
    flat = choice.reshape(-1)
    order = np.argsort(np.where(flat < 0, experts, flat), kind="stable")
    used = int((flat >= 0).sum())
    offsets = np.zeros(experts + 1, dtype=np.int32)
    offsets[1:] = np.cumsum(np.bincount(flat[flat >= 0], minlength=experts))
    slot = np.full(flat.size, -1, dtype=np.int32)
    slot[order[:used]] = np.arange(used)
    order = np.where(np.arange(flat.size) < used, order, -1).astype(np.int32)
    return choice, weight, offsets, order, slot


def offsets_of(counts):
    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32), device=DEV)


def groups(counts):
    at = np.concatenate([[0], np.cumsum(counts)])
    return [(e, int(at[e]), int(at[e + 1])) for e in range(len(counts))]


def close(got, ref, slack, dtype, what=""):
    """|got - ref| <= rounding of ref to dtype + slack, element by element."""
    got, ref = got.double(), ref.double()
    tol = ROUND[dtype] * ref.abs() + slack + TINY[dtype]
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: " \
                          f"{got[bad][0].item()} for {ref[bad][0].item()}"


def product(x, w):
    """(x w^T, its fp32 summation slack) in 64 bits."""
    x, w = x.double(), w.double()
    return x @ w.t(), (x.shape[1] + 2) * 2.0 ** -23 * (x.abs() @ w.abs().t())


def swiglu(g, u, dg, du):
    """(silu(g) u, slack from slacks dg, du of its inputs): |silu'| <= 1.1, |silu(g)| <= |g|; eight fp32 roundings of
    exp, sum, quotient and products."""
    s = torch.sigmoid(g)
    h = g * s * u
    return h, 1.1 * dg * u.abs() + g.abs() * du + 1.1 * dg * du + (8 + g.abs()) * 2.0 ** -23 * h.abs()
