"""A layer of experts: its routing, its ragged products and its 4-bit form, as cases to time and to check.

Every case is one pass through one operator, as a program calls it that holds the layer's weights on the GPU.

  route     the choice of `top_k` of `experts` for each token, its weights, and the order of the chosen by expert;
            with `train` also the gradient of the logits from that of the weights
  combine   the weighted sum of the experts' rows back to tokens; with `train` also both gradients
  mm        the product of ragged row groups with one weight matrix each, the rows gathered from the tokens on the
            way, with SwiGLU (`act`) or without
  mm_grad   the gradients of that product (without an activation) for its rows and its weights
  quant     a matrix to 4-bit blocks and back
  mm_mx4    tokens to 4-bit blocks, and their product with weights held in 4-bit blocks

`tokens` is 1 for one sequence that answers token by token, up to a few hundred for a batch of such, and thousands
for prompts and training. `width` is the tokens' length, `inner` the experts'. The choices are uneven, as a router's
are: each expert has a popularity of its own. `masked` marks logits of -infinity: one expert in eight for each token,
and every sixteenth token whole, as padding has it.
"""
import math

import torch

own = False

TYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
INF = float("inf")
LARGEST = 2.0 * 32768 * 2048 * 4096   # operations of the largest listed product


def _pf():
    import importlib
    return importlib.import_module("prefree-public_amd")


def _case(op, tokens, experts, top_k, width=0, inner=0, dtype="bf16", act=False, train=False, masked=False,
          normalise=True):
    return {"op": op, "tokens": tokens, "experts": experts, "top_k": top_k, "width": width, "inner": inner,
            "dtype": dtype, "act": act, "train": train, "masked": masked, "normalise": normalise}


def _named(name, *args, **kwargs):
    return {"name": name, **_case(*args, **kwargs)}


def listed():
    return [
        # one token of one sequence: the smallest call there is, all of it latency
        _named("route_1_of_64_bf16", "route", 1, 64, 8),
        # a training batch, forward and backward, with padding and experts that are out of reach
        _named("route_16384_of_128_f32_train", "route", 16384, 128, 8, dtype="f32", train=True, masked=True),
        # a few sequences that answer side by side
        _named("combine_5_bf16", "combine", 5, 64, 8, 2048),
        # a training batch of an odd number of tokens
        _named("combine_8191_f16_train", "combine", 8191, 32, 4, 2048, dtype="f16", train=True),
        # one token: eight experts' weights are read for one row each
        _named("mm_1_bf16_act", "mm", 1, 64, 8, 2048, 1024, act=True),
        # a batch of sequences that answer: every expert has some rows, none has many
        _named("mm_67_bf16_act", "mm", 67, 64, 8, 2048, 1024, act=True),
        # odd sizes in half precision: rows that start at odd addresses
        _named("mm_311_odd_f16", "mm", 311, 12, 2, 1111, 717, dtype="f16"),
        # prompts: the matrix cores' case, and the largest
        _named("mm_8192_bf16_act", "mm", 8192, 32, 4, 2048, 2048, act=True),
        # a training batch's gradients
        _named("mm_grad_8192_bf16", "mm_grad", 8192, 16, 2, 2048, 2048),
        # a layer's weights, quantised as they are loaded
        _named("quant_65536_bf16", "quant", 65536, 1, 1, 2048),
        # one token, and prompts, with 4-bit weights
        _named("mm_mx4_1_act", "mm_mx4", 1, 64, 8, 2048, 1024, act=True),
        _named("mm_mx4_8192_act", "mm_mx4", 8192, 32, 4, 2048, 2048, act=True),
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step`: one time in four a power of two times it, else an odd multiple, which no tile divides."""
    n = max(lo, min(hi, lo * (hi / lo) ** rng.random())) / step
    return step * (1 << int(math.log2(n)) if rng.random() < 0.25 else int(n - 1) | 1)


def draw(rng):
    op = rng.choice(["route", "combine", "mm", "mm", "mm", "mm_grad", "mm_grad", "quant", "mm_mx4", "mm_mx4"])
    experts = rng.choice([4, 8, 12, 16, 24, 32, 60, 64, 96, 128])
    top_k = min(rng.choice([1, 2, 2, 4, 4, 6, 8]), experts)
    dtype = rng.choice(["bf16", "bf16", "f16"])
    train = rng.random() < 0.5
    if op == "route":
        return _case(op, _log(rng, 1, 32768), experts, top_k, dtype=rng.choice(["f32", "f32", "bf16", "f16"]),
                     train=train, masked=rng.random() < 0.5, normalise=rng.random() < 0.7)
    if op == "combine":
        return _case(op, _log(rng, 1, 16384), experts, top_k, _log(rng, 500, 4096), dtype=dtype, train=train)
    if op == "quant":
        return _case(op, _log(rng, 1, 65536), 1, 1, _log(rng, 128, 4096, 32), dtype=rng.choice(["bf16", "f16", "f32"]))
    step = 8 if rng.random() < 0.75 else 1
    width = _log(rng, 512, 4096, 32 if op == "mm_mx4" else step)
    inner = _log(rng, 256, 2048, step)
    act = op != "mm_grad" and rng.random() < 0.6
    # no more than the largest listed case: fewer tokens, and no more than 2^29 weights
    rows = (2 if act else 1) * inner
    while experts * rows * width > 1 << 29:
        experts //= 2
    top_k = min(top_k, experts)
    tokens = int(LARGEST / (2.0 * top_k * width * rows * (2 if op == "mm_grad" else 1)))
    tokens = _log(rng, 1 if op != "mm_grad" else 64, min(8192, tokens))
    return _case(op, tokens, experts, top_k, width, inner, dtype=dtype, act=act)


# ---- inputs ----------------------------------------------------------------------------------------------------

def _logits(case, g, device):
    t, e = case["tokens"], case["experts"]
    z = torch.randn(t, e, generator=g, device=device) * 1.5 + torch.randn(e, generator=g, device=device) * 0.5
    if case["masked"]:
        z[torch.rand(t, e, generator=g, device=device) < 0.125] = -INF
        z[15::16] = -INF
    return z


def _routing(choice, experts):
    """(offsets, order, slot) of a choice [tokens, top_k] of experts (-1: none)."""
    flat = choice.reshape(-1).long()
    key = torch.where(flat < 0, experts, flat)
    by, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(by, torch.arange(experts + 1, device=flat.device))
    place = torch.arange(flat.numel(), device=flat.device)
    slot = torch.empty_like(place).scatter_(0, order, torch.where(by < experts, place, -1))
    order = torch.where(by < experts, order, -1)
    return offsets.int(), order.int(), slot.int()


def _randn(g, device, dtype, *shape):
    out = torch.empty(shape, dtype=dtype, device=device)
    return out.normal_(generator=g)


def prepare(case, seed):
    device = "cuda"
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    c = dict(case)
    op, t, e, k, width, inner = (c[n] for n in ("op", "tokens", "experts", "top_k", "width", "inner"))
    dtype = TYPE[c["dtype"]]
    s = {"case": c}
    f32, i32 = {"dtype": torch.float32, "device": device}, {"dtype": torch.int32, "device": device}
    if op == "route":
        s["logits"] = _logits(c, g, device).to(dtype)
        s["dweight"] = torch.randn(t, k, generator=g, device=device)
        s["choice"], s["weight"] = torch.empty(t, k, **i32), torch.empty(t, k, **f32)
        s["offsets"], s["order"], s["slot"] = torch.empty(e + 1, **i32), torch.empty(t * k, **i32), torch.empty(t * k, **i32)
        s["dlogits"] = torch.empty(t, e, dtype=dtype, device=device)
        s["workspace"] = torch.empty(e * (-(-t // 64)), **i32)
        return s
    if op == "quant":
        s["x"] = _randn(g, device, dtype, t, width) * torch.exp2(2 * torch.randn(t, 1, generator=g, device=device)).to(dtype)
        s["codes"] = torch.empty(t, width // 2, dtype=torch.uint8, device=device)
        s["scales"] = torch.empty(t, width // 32, dtype=torch.uint8, device=device)
        s["values"] = torch.empty(t, width, **f32)
        return s
    choice = torch.sort(_logits(c, g, device), dim=1, descending=True, stable=True)[1][:, :k]
    s["offsets"], s["order"], s["slot"] = _routing(choice, e)
    s["capacity"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())
    n = t * k
    if op == "combine":
        s["weight"] = torch.softmax(torch.randn(t, k, generator=g, device=device), dim=1)
        s["y"] = _randn(g, device, dtype, n, width)
        s["out"] = torch.empty(t, width, dtype=dtype, device=device)
        s["dout"] = _randn(g, device, dtype, t, width)
        s["dy"], s["dweight"] = torch.empty(n, width, dtype=dtype, device=device), torch.empty(t, k, **f32)
        return s
    rows = (2 if c["act"] else 1) * inner
    s["x"] = _randn(g, device, dtype, t, width)
    s["y"] = torch.empty(n, inner, dtype=dtype, device=device)
    w = _randn(g, device, dtype, e, rows, width) * width ** -0.5
    if op == "mm_mx4":
        s["wq"], s["ws"] = _quantised(w.reshape(e * rows, width))
        s["wq"], s["ws"] = s["wq"].reshape(e, rows, -1), s["ws"].reshape(e, rows, -1)
        s["xq"] = torch.empty(t, width // 2, dtype=torch.uint8, device=device)
        s["xs"] = torch.empty(t, width // 32, dtype=torch.uint8, device=device)
        return s
    s["w"] = w
    if op == "mm_grad":
        s["dy"] = _randn(g, device, dtype, n, inner)
        s["dx"] = torch.empty(n, width, dtype=dtype, device=device)
        s["dw"] = torch.empty(e, inner, width, **f32)
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------

def _route_plain(s):
    c, z = s["case"], s["logits"].float()
    k, e = c["top_k"], c["experts"]
    top, index = torch.sort(z, dim=1, descending=True, stable=True)
    top, index = top[:, :k], index[:, :k]
    chosen = top > -INF
    most = torch.where(chosen[:, :1], top[:, :1], 0.0)
    part = torch.exp(top - most)
    whole = torch.exp(z - most)
    total = (part if c["normalise"] else whole).sum(dim=1, keepdim=True)
    weight = torch.where(chosen, part / total, 0.0)
    choice = torch.where(chosen, index, -1)
    out = [choice.int(), weight, *_routing(choice, e)]
    if c["train"]:
        grad = weight * s["dweight"]
        inner = grad.sum(dim=1, keepdim=True)
        if c["normalise"]:
            dz = torch.zeros_like(z).scatter_(1, index, grad - weight * inner)
        else:
            share = torch.where(z > -INF, whole / total, 0.0)
            dz = torch.zeros_like(z).scatter_(1, index, grad) - share * inner
        out.append(dz.to(s["logits"].dtype))
    return out


def _combine_plain(s):
    c = s["case"]
    y = s["y"].float()[s["slot"].long()].reshape(c["tokens"], c["top_k"], -1)
    out = [(y * s["weight"][:, :, None]).sum(dim=1).to(s["out"].dtype)]
    if c["train"]:
        dout = s["dout"].float()
        dy = (dout[:, None, :] * s["weight"][:, :, None]).reshape(-1, c["width"])
        out.append(dy[s["order"].long()].to(s["dy"].dtype))
        out.append((dout[:, None, :] * y).sum(dim=2))
    return out


def _padded(s):
    """The slots of every expert as [experts, capacity], and which of them there are."""
    at = s["offsets"][:-1, None].long() + torch.arange(s["capacity"], device=s["offsets"].device)
    there = at < s["offsets"][1:, None]
    return torch.where(there, at, 0), there


def _product_plain(s, x, w):
    c = s["case"]
    at, there = _padded(s)
    rows = torch.where(there[:, :, None], x[s["order"].long()[at] // c["top_k"]], 0.0)
    y = torch.matmul(rows, w.transpose(1, 2))
    if c["act"]:
        gate, up = y[:, :, :c["inner"]], y[:, :, c["inner"]:]
        y = gate / (1 + torch.exp(-gate)) * up
    out = torch.empty_like(s["y"], dtype=torch.float32)
    out[at[there]] = y[there]
    return out.to(s["y"].dtype)


def _grad_plain(s):
    c = s["case"]
    at, there = _padded(s)
    there = there[:, :, None]
    rows = torch.where(there, s["x"].float()[s["order"].long()[at] // c["top_k"]], 0.0)
    dy = torch.where(there, s["dy"].float()[at], 0.0)
    dx = torch.empty_like(s["dx"], dtype=torch.float32)
    there = there[:, :, 0]
    dx[at[there]] = torch.matmul(dy, s["w"].float())[there]
    return [dx.to(s["dx"].dtype), torch.matmul(dy.transpose(1, 2), rows)]


def _quantised(x):
    """4-bit blocks of x [rows, columns]: codes, two a byte with the first in the low half, and scales."""
    blocks = x.float().reshape(x.shape[0], -1, 32)
    most = blocks.abs().amax(dim=2, keepdim=True)
    exponent = torch.frexp(most)[1] - 3          # most = m 2^e, m in [1/2, 1): floor(log2) is e - 1
    exponent = torch.where(most > 0, exponent, -127).clamp(-127, 127)
    size = torch.ldexp(blocks.abs(), -exponent)
    # nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6; a tie goes to the even code
    code = ((size > 0.25).byte() + (size >= 0.75) + (size > 1.25) + (size >= 1.75) + (size > 2.5) + (size >= 3.5) + (size > 5.0))
    code = code + 8 * torch.signbit(blocks).byte()
    code = code.reshape(x.shape[0], -1, 2)
    scale = (exponent + 127).byte().reshape(x.shape[0], -1)
    return code[:, :, 0] + 16 * code[:, :, 1], scale


def _values(codes, scales):
    """What 4-bit blocks stand for, in 32 bits."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    table = torch.cat([table, -table])
    v = table[torch.stack([codes & 15, codes >> 4], dim=-1).int()].reshape(*scales.shape, 32)
    return torch.ldexp(v, scales.int()[..., None] - 127).reshape(*codes.shape[:-1], -1)


def run(s):
    c = s["case"]
    if own:
        return _run_own(s)
    if c["op"] == "route":
        return _route_plain(s)
    if c["op"] == "combine":
        return _combine_plain(s)
    if c["op"] == "mm":
        return _product_plain(s, s["x"].float(), s["w"].float())
    if c["op"] == "mm_grad":
        return _grad_plain(s)
    if c["op"] == "quant":
        return _values(*_quantised(s["x"]))
    return _product_plain(s, _values(*_quantised(s["x"])), _values(s["wq"], s["ws"]))


def _run_own(s):
    pf, c = _pf(), s["case"]
    op, t, e, k, width, inner = (c[n] for n in ("op", "tokens", "experts", "top_k", "width", "inner"))
    act = "swiglu" if c["act"] else "none"
    if op == "route":
        pf.moe_route(s["logits"], t, e, k, s["choice"], s["weight"], s["offsets"], s["order"], s["slot"], s["workspace"],
                     dtype=c["dtype"], normalise=c["normalise"])
        out = [s["choice"], s["weight"], s["offsets"], s["order"], s["slot"]]
        if c["train"]:
            pf.moe_route_backward(s["logits"], t, e, k, s["choice"], s["weight"], s["dweight"], s["dlogits"],
                                  dtype=c["dtype"], normalise=c["normalise"])
            out.append(s["dlogits"])
        return out
    if op == "combine":
        pf.moe_combine(s["y"], s["slot"], s["weight"], t, k, width, s["out"], dtype=c["dtype"])
        if not c["train"]:
            return [s["out"]]
        pf.moe_combine_backward(s["dout"], s["y"], s["slot"], s["weight"], t, k, width, s["dy"], s["dweight"],
                                dtype=c["dtype"])
        return [s["out"], s["dy"], s["dweight"]]
    if op == "mm":
        pf.moe_mm(s["x"], t, s["order"], k, s["w"], s["offsets"], e, t * k, inner, width, s["y"], dtype=c["dtype"],
                  act=act)
        return s["y"]
    if op == "mm_grad":
        pf.moe_mm_dx(s["dy"], s["w"], s["offsets"], e, t * k, inner, width, s["dx"], dtype=c["dtype"])
        pf.moe_mm_dw(s["dy"], s["x"], t, s["order"], k, s["offsets"], e, t * k, inner, width, s["dw"],
                     dtype=c["dtype"], dw_dtype="f32")
        return [s["dx"], s["dw"]]
    if op == "quant":
        pf.mx4_quantize(s["x"], t, width, s["codes"], s["scales"], dtype=c["dtype"])
        pf.mx4_dequantize(s["codes"], s["scales"], t, width, s["values"], dtype="f32")
        return s["values"]
    pf.mx4_quantize(s["x"], t, width, s["xq"], s["xs"], dtype=c["dtype"])
    pf.moe_mm_mx4(s["xq"], s["xs"], t, s["order"], k, s["wq"], s["ws"], s["offsets"], e, t * k, inner, width, s["y"],
                  dtype=c["dtype"], act=act)
    return s["y"]


# ---- what a pass cannot do without -------------------------------------------------------------------------------

def work(case):
    op, t, e, k, width, inner = (case[n] for n in ("op", "tokens", "experts", "top_k", "width", "inner"))
    b, n = SIZE[case["dtype"]], t * k
    if op == "route":
        both = 2 if case["train"] else 1
        return {"bytes": both * t * e * b + 16 * n + 4 * (e + 1) + (both - 1) * 4 * n, "flops": both * 4 * t * e}
    if op == "combine":
        if case["train"]:
            return {"bytes": b * width * (2 * t + 2 * n) + 16 * n, "flops": 6 * n * width}
        return {"bytes": b * width * (t + n) + 8 * n, "flops": 2 * n * width}
    if op == "quant":
        return {"bytes": t * width * (b + 2 * (0.5 + 1 / 32) + 4), "flops": 4 * t * width}
    rows = (2 if case["act"] else 1) * inner
    used = e * (1 - (1 - 1 / e) ** n)            # experts with a row, were all alike
    if op == "mm":
        return {"bytes": b * (used * rows * width + t * width + n * inner) + 4 * n, "flops": 2 * n * rows * width}
    if op == "mm_grad":
        return {"bytes": b * (used * rows * width + t * width + n * (inner + width)) + 4 * e * rows * width + 4 * n,
                "flops": 4 * n * rows * width}
    held = width * (0.5 + 1 / 32)
    return {"bytes": used * rows * held + t * (b * width + held) + b * n * inner + 4 * n, "flops": 2 * n * rows * width}


# ---- the definitions, in 64 bits -----------------------------------------------------------------------------------

def _blocks64(x):
    """Each block of 32 of x rounded to the nearest multiple of its scale that e2m1 has."""
    blocks = x.double().reshape(-1, 32)
    most = blocks.abs().amax(dim=1, keepdim=True)
    scale = torch.exp2(torch.floor(torch.log2(torch.where(most > 0, most, 1.0))) - 2)
    v = (blocks / scale).abs()
    step = torch.where(v < 2, 0.5, torch.where(v < 4, 1.0, 2.0)).double()   # torch.round takes ties to even multiples
    return (torch.clamp(torch.round(v / step) * step, max=6.0) * torch.sign(blocks) * scale).reshape(x.shape)


def _held64(codes, scales):
    sign = 1.0 - 2.0 * ((codes >> 3) & 1).double()
    e, m = ((codes >> 1) & 3).double(), (codes & 1).double()
    low = sign * torch.where(e > 0, (1 + m / 2) * torch.exp2(e - 1), m / 2)
    hi = codes >> 4
    sign = 1.0 - 2.0 * ((hi >> 3) & 1).double()
    e, m = ((hi >> 1) & 3).double(), (hi & 1).double()
    high = sign * torch.where(e > 0, (1 + m / 2) * torch.exp2(e - 1), m / 2)
    v = torch.stack([low, high], dim=-1).reshape(*scales.shape, 32)
    return (v * torch.exp2(scales.double() - 127)[..., None]).reshape(*codes.shape[:-1], -1)


def exact(case, seed):
    s = prepare(case, seed)
    op, t, e, k, width, inner = (case[n] for n in ("op", "tokens", "experts", "top_k", "width", "inner"))
    if op == "route":
        z = s["logits"].double()
        # rank of each logit in its row: those above it, and equal ones before it
        rank = torch.empty(t, e, dtype=torch.int64, device=z.device)
        for i in range(e):
            above = z > z[:, i:i + 1]
            above[:, :i] |= z[:, :i] == z[:, i:i + 1]
            rank[:, i] = above.sum(dim=1)
        chosen = (rank < k) & (z > -INF)
        top = torch.where(chosen.any(dim=1, keepdim=True), z.amax(dim=1, keepdim=True), 0.0)
        p = torch.exp(z - top)
        p = torch.where(chosen, p, 0.0) if case["normalise"] else p
        p = p / p.sum(dim=1, keepdim=True).clamp(min=1e-300)
        spot = torch.where(chosen, rank, k)
        weight = torch.zeros(t, k + 1, dtype=torch.float64, device=z.device).scatter_(1, spot, torch.where(chosen, p, 0.0))[:, :k]
        out = [None, weight, None, None, None]
        if case["train"]:
            full = torch.zeros_like(z)
            for j in range(k):
                full += torch.where(spot == j, s["dweight"][:, j:j + 1].double(), 0.0)
            out.append(p * (full - (weight * s["dweight"].double()).sum(dim=1, keepdim=True)))
        return out
    if op == "quant":
        return _blocks64(s["x"])
    slot = s["slot"].long().reshape(t, k)
    if op == "combine":
        weight, y, dout = s["weight"].double(), s["y"].double(), s["dout"].double()
        out = [sum(weight[:, j:j + 1] * y[slot[:, j]] for j in range(k))]
        if case["train"]:
            dy = torch.zeros_like(y)
            for j in range(k):
                dy[slot[:, j]] = weight[:, j:j + 1] * dout
            out += [dy, torch.stack([(dout * y[slot[:, j]]).sum(dim=1) for j in range(k)], dim=1)]
        return out
    bounds = s["offsets"].tolist()
    token = s["order"].long() // k
    x = _blocks64(s["x"]) if op == "mm_mx4" else s["x"].double()
    out, dw = [], []
    for i in range(e):
        rows = x[token[bounds[i]:bounds[i + 1]]]
        w = _held64(s["wq"][i], s["ws"][i]) if op == "mm_mx4" else s["w"][i].double()
        if op == "mm_grad":
            dy = s["dy"][bounds[i]:bounds[i + 1]].double()
            out.append(dy @ w)
            dw.append(dy.t() @ rows)
        else:
            y = rows @ w.t()
            out.append(y[:, :inner] * torch.sigmoid(y[:, :inner]) * y[:, inner:] if case["act"] else y)
    out = torch.cat(out)
    return [out, torch.stack(dw)] if op == "mm_grad" else out
