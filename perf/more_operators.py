"""More of a layer of experts: routing by scores, products in 8-bit integers, orthogonal updates of its weights.

Every case is one pass through one operator, as a program calls it that holds the layer's weights on the GPU.

  route   the choice of `top_k` of `experts` by sigmoid or softmax scores plus a bias that balances the load, out of the
          best groups of experts, its weights from the scores alone, and the order of the chosen by expert; with
          `train` also the gradient of the logits from that of the weights, and the bias for the next step
  quant   a matrix to 8-bit integers with a scale a row, and back
  mm      tokens to 8-bit integers, and their product by expert with weights held in 8-bit integers with a scale a
          row, with SwiGLU (`act`) or without
  orth    the update of `experts` matrices made orthogonal by five Newton-Schulz steps, out of their momentum

`tokens` is 1 for one sequence that answers token by token, up to a few hundred for a batch of such, and thousands for
prompts and training.  `width` is the tokens' length, `inner` the experts'.  The choices are uneven, as a router's are.
`masked` marks logits of -infinity: one expert in eight for each token, and every sixteenth token whole, as padding has it.
"""
import math

import torch

own = False

TYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
INF = float("inf")
LARGEST = 2.0 * 32768 * 2048 * 4096   # operations of the largest listed product
STEPS = [(3.4445, -4.7750, 2.0315)] * 5   # x (a + b x^2 + c x^4), near 1 after five times for x from 0.01 to 1


def _pf():
    import importlib
    return importlib.import_module("prefree-public_amd")


def _route(tokens, experts, top_k, score="sigmoid", dtype="f32", bias=True, groups=1, kept=1, best=2, normalise=True,
           scale=1.0, train=False, masked=False):
    return {"op": "route", "tokens": tokens, "experts": experts, "top_k": top_k, "score": score, "dtype": dtype, "bias": bias,
            "groups": groups, "kept": kept, "best": best, "normalise": normalise, "scale": scale, "train": train, "masked": masked}


def _quant(tokens, width, dtype="bf16"):
    return {"op": "quant", "tokens": tokens, "width": width, "dtype": dtype}


def _mm(tokens, experts, top_k, width, inner, dtype="bf16", act=False):
    return {"op": "mm", "tokens": tokens, "experts": experts, "top_k": top_k, "width": width, "inner": inner, "dtype": dtype,
            "act": act}


def _orth(experts, inner, width, dtype="f32", result="bf16"):
    return {"op": "orth", "experts": experts, "inner": inner, "width": width, "dtype": dtype, "result": result}


def listed():
    return [
        # one token of one sequence: all of it latency
        {"name": "route_1_of_64", **_route(1, 64, 8, dtype="bf16", groups=8, kept=4, scale=2.5)},
        # a training batch with padding: forward, backward and the next bias
        {"name": "route_16384_of_256_train", **_route(16384, 256, 8, groups=8, kept=4, scale=2.5, train=True, masked=True)},
        # softmax scores, not renormalised, groups by their best expert; an odd batch
        {"name": "route_4097_of_96_softmax", **_route(4097, 96, 6, "softmax", "bf16", False, 8, 3, 1, False, 16.0)},
        # activations on their way into a product
        {"name": "quant_32768_bf16", **_quant(32768, 2048)},
        # rows that start at odd addresses
        {"name": "quant_1023_odd_f16", **_quant(1023, 1111, "f16")},
        # one token: eight experts' weights are read for one row each
        {"name": "mm_1_act", **_mm(1, 64, 8, 2048, 1024, act=True)},
        # a batch of sequences that answer: every expert has some rows, none has many
        {"name": "mm_67_act", **_mm(67, 64, 8, 2048, 1024, act=True)},
        # odd sizes in half precision
        {"name": "mm_311_odd_f16", **_mm(311, 12, 2, 1111, 717, "f16")},
        # prompts: the matrix cores' case
        {"name": "mm_8192_act", **_mm(8192, 32, 4, 2048, 2048, act=True)},
        # a router's update: one flat matrix
        {"name": "orth_64x2048_f32", **_orth(1, 64, 2048)},
        # a small layer's experts, more rows than columns, of odd sizes
        {"name": "orth_12x1111x717_bf16", **_orth(12, 1111, 717, "bf16")},
        # a layer's experts from their fp32 momentum: the largest
        {"name": "orth_16x2048x2048_f32", **_orth(16, 2048, 2048)},
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step`: one time in four a power of two times it, else an odd multiple, which no tile divides."""
    n = max(lo, min(hi, lo * (hi / lo) ** rng.random())) / step
    return step * (1 << int(math.log2(n)) if rng.random() < 0.25 else int(n - 1) | 1)


def draw(rng):
    op = rng.choice(["route", "route", "route", "quant", "mm", "mm", "mm", "orth", "orth"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        kept = rng.randint(1, groups)
        experts = groups * rng.choice([4, 6, 8, 12, 16, 20, 32])
        top_k = min(rng.choice([1, 2, 4, 6, 8]), kept * (experts // groups))
        return _route(_log(rng, 1, 32768), experts, top_k, rng.choice(["sigmoid", "sigmoid", "softmax"]),
                      rng.choice(["f32", "f32", "bf16", "f16"]), rng.random() < 0.75, groups, kept, rng.choice([1, 2]),
                      rng.random() < 0.7, rng.choice([1.0, 2.5, 16.0]), rng.random() < 0.5, rng.random() < 0.5)
    if op == "quant":
        return _quant(_log(rng, 1, 32768), _log(rng, 128, 4096), rng.choice(["bf16", "f16", "f32"]))
    experts = rng.choice([4, 8, 12, 16, 24, 32, 60, 64, 96, 128])
    if op == "orth":
        inner, width = _log(rng, 32, 2048), _log(rng, 32, 4096)
        while experts > 1 and experts * min(inner, width) ** 2 * max(inner, width) > 16 * 2048 ** 3:
            experts //= 2
        if min(inner, width) ** 2 * max(inner, width) > 2 * 2048 ** 3:
            width = 2048
        return _orth(rng.choice([1, experts]), inner, width, rng.choice(["f32", "bf16", "f16"]), dtype)
    top_k = min(rng.choice([1, 2, 2, 4, 4, 6, 8]), experts)
    step = 16 if rng.random() < 0.75 else 1
    width, inner, act = _log(rng, 512, 4096, step), _log(rng, 256, 2048, step), rng.random() < 0.6
    # no more than the largest listed case: fewer tokens, and no more than 2^29 weights
    rows = (2 if act else 1) * inner
    while experts * rows * width > 1 << 29:
        experts //= 2
    top_k = min(top_k, experts)
    tokens = _log(rng, 1, min(8192, int(LARGEST / (2.0 * top_k * width * rows))))
    return _mm(tokens, experts, top_k, width, inner, dtype, act)


# ---- inputs ----------------------------------------------------------------------------------------------------

def _logits(tokens, experts, masked, g):
    z = torch.randn(tokens, experts, generator=g, device="cuda") * 1.5 + torch.randn(experts, generator=g, device="cuda") * 0.5
    if masked:
        z[torch.rand(tokens, experts, generator=g, device="cuda") < 0.125] = -INF
        z[15::16] = -INF
    return z


def _order(choice, experts):
    """(offsets, order, slot) of a choice [tokens, top_k] of experts (-1: none)."""
    flat = choice.reshape(-1).long()
    key = torch.where(flat < 0, experts, flat)
    by, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(by, torch.arange(experts + 1, device=flat.device))
    place = torch.arange(flat.numel(), device=flat.device)
    slot = torch.empty_like(place).scatter_(0, order, torch.where(by < experts, place, -1))
    order = torch.where(by < experts, order, -1)
    return offsets.int(), order.int(), slot.int()


def _randn(g, dtype, *shape):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=g)


def _row(k):
    """Bytes of a row of k 8-bit integers: whole pieces of 16, zeros behind the k."""
    return (k + 15) // 16 * 16


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c = dict(case)
    op, dtype = c["op"], TYPE[c["dtype"]]
    s = {"case": c}
    f32, i32, i8 = ({"dtype": t, "device": "cuda"} for t in (torch.float32, torch.int32, torch.int8))
    if op == "orth":
        e, m, n = c["experts"], c["inner"], c["width"]
        # a momentum: few directions carry most of it, the rest is noise
        few = max(1, min(m, n) // 8)
        g32 = torch.matmul(_randn(g, torch.float32, e, m, few), _randn(g, torch.float32, e, few, n)) * few ** -0.5
        s["g"] = ((g32 + 0.3 * _randn(g, torch.float32, e, m, n)) * 2e-3).to(dtype)
        s["out"] = torch.empty(e, m, n, dtype=TYPE[c["result"]], device="cuda")
        pieces = (-(-m // 64) * 64) * (-(-n // 64) * 64)
        s["workspace"] = torch.empty(16 * e * pieces + (1 << 26), dtype=torch.uint8, device="cuda")
        return s
    t = c["tokens"]
    if op == "route":
        e, k = c["experts"], c["top_k"]
        s["logits"] = _logits(t, e, c["masked"], g).to(dtype)
        s["bias"] = torch.randn(e, generator=g, device="cuda") * 0.05 if c["bias"] else None
        s["dweight"] = torch.randn(t, k, generator=g, device="cuda")
        s["choice"], s["weight"] = torch.empty(t, k, **i32), torch.empty(t, k, **f32)
        s["offsets"], s["order"], s["slot"] = torch.empty(e + 1, **i32), torch.empty(t * k, **i32), torch.empty(t * k, **i32)
        s["dlogits"], s["next"] = torch.empty(t, e, dtype=dtype, device="cuda"), torch.empty(e, **f32)
        s["workspace"] = torch.empty(e * (-(-t // 64)), **i32)
        return s
    k = c["width"]
    if op == "quant":
        s["x"] = _randn(g, dtype, t, k) * torch.exp2(2 * torch.randn(t, 1, generator=g, device="cuda")).to(dtype)
        s["codes"], s["scales"] = torch.empty(t, _row(k), **i8), torch.empty(t, **f32)
        s["values"] = torch.empty(t, k, **f32)
        return s
    e, top_k, inner = c["experts"], c["top_k"], c["inner"]
    choice = torch.sort(_logits(t, e, False, g), dim=1, descending=True, stable=True)[1][:, :top_k]
    s["offsets"], s["order"], s["slot"] = _order(choice, e)
    s["capacity"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())
    s["x"] = _randn(g, dtype, t, k)
    rows = (2 if c["act"] else 1) * inner
    codes, scales = _quantised(_randn(g, torch.bfloat16, e * rows, k) * k ** -0.5)
    s["wq"] = torch.nn.functional.pad(codes, (0, _row(k) - k)).reshape(e, rows, -1).contiguous()
    s["ws"] = scales.reshape(e, rows).contiguous()
    s["xq"], s["xs"] = torch.empty(t, _row(k), **i8), torch.empty(t, **f32)
    s["y"] = torch.empty(t * top_k, inner, dtype=dtype, device="cuda")
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------

def _scores(c, z):
    """Scores of logits in 64 bits: sums that lie next to each other decide the choice."""
    z = z.double()
    if c["score"] == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    most = z.amax(dim=1, keepdim=True)
    part = torch.exp(z - torch.where(most > -INF, most, 0.0))
    return part / part.sum(dim=1, keepdim=True).clamp(min=1e-300)


def _route_plain(s):
    c, z = s["case"], s["logits"]
    t, e = z.shape
    k, groups = c["top_k"], c["groups"]
    score = _scores(c, z)
    rank = score if s["bias"] is None else score + s["bias"].double()
    rank = torch.where(z > -INF, rank, -INF)
    if groups > 1:
        best = torch.sort(rank.reshape(t, groups, -1), dim=2, descending=True)[0][:, :, :c["best"]]
        total = torch.where(best > -INF, best, 0.0).sum(dim=2)
        total = torch.where(best[:, :, 0] > -INF, total, -INF)
        first = torch.sort(total, dim=1, descending=True, stable=True)[1][:, :c["kept"]]
        kept = torch.zeros(t, groups, dtype=torch.bool, device=z.device).scatter_(1, first, True)
        rank = torch.where(kept[:, :, None], rank.reshape(t, groups, -1), -INF).reshape(t, e)
    top, index = torch.sort(rank, dim=1, descending=True, stable=True)
    top, index = top[:, :k], index[:, :k]
    chosen = top > -INF
    part = torch.where(chosen, score.gather(1, index), 0.0)
    total = part.sum(dim=1, keepdim=True).clamp(min=1e-300)
    weight = c["scale"] * (part / total if c["normalise"] else part)
    choice = torch.where(chosen, index, -1)
    offsets, order, slot = _order(choice, e)
    out = [choice.int(), weight.float(), offsets, order, slot]
    if c["train"]:
        g = s["dweight"].double()
        inner = (weight * g).sum(dim=1, keepdim=True) / c["scale"]
        if c["score"] == "sigmoid":
            dz = weight * (1 - score.gather(1, index)) * (g - inner if c["normalise"] else g)
            dz = torch.zeros_like(score).scatter_(1, index, dz)
        elif c["normalise"]:
            dz = torch.zeros_like(score).scatter_(1, index, weight * (g - inner))
        else:
            dz = torch.zeros_like(score).scatter_(1, index, weight * g) - score * inner * c["scale"]
        out.append(dz.to(z.dtype))
        if s["bias"] is not None:
            count = (offsets[1:] - offsets[:-1]).long()
            out.append(s["bias"] + 1e-3 * torch.sign(offsets[-1] - count * e).float())
    return out


def _quantised(x):
    """Rows of x as integers from -127 to 127 and a scale each; in 64 bits, where a quotient between two integers is one."""
    most = x.float().abs().amax(dim=1, keepdim=True).clamp(min=2.0 ** -100)
    return torch.round(x.double() * 127 / most.double()).to(torch.int8), (most / 127)[:, 0]


def _product_plain(s):
    c = s["case"]
    codes, scales = _quantised(s["x"])
    at = s["offsets"][:-1, None].long() + torch.arange(s["capacity"], device=codes.device)
    there = at < s["offsets"][1:, None]
    at = torch.where(there, at, 0)
    row = s["order"].long()[at] // c["top_k"]
    y = torch.matmul(torch.where(there[:, :, None], codes[row].float(), 0.0), s["wq"][:, :, :c["width"]].float().transpose(1, 2))
    y = y * scales[row][:, :, None] * s["ws"][:, None, :]
    if c["act"]:
        gate, up = y[:, :, :c["inner"]], y[:, :, c["inner"]:]
        y = gate / (1 + torch.exp(-gate)) * up
    out = torch.empty_like(s["y"], dtype=torch.float32)
    out[at[there]] = y[there]
    return out.to(s["y"].dtype)


def _orth_plain(s):
    x = s["g"].float()
    flat = x.shape[1] <= x.shape[2]
    x = x if flat else x.transpose(1, 2).contiguous()
    x = x / x.double().square().sum(dim=(1, 2), keepdim=True).sqrt().clamp(min=1e-300).float()
    for a, b, c in STEPS:
        square = torch.matmul(x, x.transpose(1, 2))
        x = a * x + torch.matmul(b * square + c * torch.matmul(square, square), x)
    return (x if flat else x.transpose(1, 2).contiguous()).to(s["out"].dtype)


def run(s):
    c = s["case"]
    if own:
        return _run_own(s)
    if c["op"] == "route":
        return _route_plain(s)
    if c["op"] == "quant":
        codes, scales = _quantised(s["x"])
        return codes.float() * scales[:, None]
    return _product_plain(s) if c["op"] == "mm" else _orth_plain(s)


def _run_own(s):
    pf, c = _pf(), s["case"]
    op = c["op"]
    if op == "orth":
        e, m, n = c["experts"], c["inner"], c["width"]
        pf.orthogonalize(s["g"], e, m, n, s["out"], s["workspace"], dtype=c["dtype"], out_dtype=c["result"], steps=STEPS)
        return s["out"]
    t = c["tokens"]
    if op == "route":
        e, k = c["experts"], c["top_k"]
        pf.moe_route_scores(s["logits"], t, e, k, s["choice"], s["weight"], s["offsets"], s["order"], s["slot"], s["workspace"],
                            dtype=c["dtype"], score=c["score"], bias=s["bias"], groups=c["groups"], groups_kept=c["kept"],
                            group_best=c["best"], normalise=c["normalise"], scale=c["scale"])
        out = [s["choice"], s["weight"], s["offsets"], s["order"], s["slot"]]
        if c["train"]:
            pf.moe_route_scores_backward(s["logits"], t, e, k, s["choice"], s["weight"], s["dweight"], s["dlogits"],
                                         dtype=c["dtype"], score=c["score"], normalise=c["normalise"], scale=c["scale"])
            out.append(s["dlogits"])
            if s["bias"] is not None:
                pf.moe_balance(s["offsets"], e, 1e-3, s["bias"], s["next"])
                out.append(s["next"])
        return out
    k = c["width"]
    if op == "quant":
        pf.i8_quantize(s["x"], t, k, s["codes"], s["scales"], dtype=c["dtype"])
        pf.i8_dequantize(s["codes"], s["scales"], t, k, s["values"], dtype="f32")
        return s["values"]
    top_k, inner = c["top_k"], c["inner"]
    pf.i8_quantize(s["x"], t, k, s["xq"], s["xs"], dtype=c["dtype"])
    pf.moe_mm_i8(s["xq"], s["xs"], t, s["order"], top_k, s["wq"], s["ws"], s["offsets"], c["experts"], t * top_k, inner, k,
                 s["y"], dtype=c["dtype"], act="swiglu" if c["act"] else "none")
    return s["y"]


# ---- what a pass cannot do without -------------------------------------------------------------------------------

def work(case):
    op, b = case["op"], SIZE[case["dtype"]]
    if op == "orth":
        e, m, n = case["experts"], *sorted((case["inner"], case["width"]))
        # squares are symmetric: half their results
        return {"bytes": e * m * n * (b + SIZE[case["result"]]), "flops": len(STEPS) * e * (m * m * n + m ** 3 + 2 * m * m * n)}
    t = case["tokens"]
    if op == "route":
        e, n = case["experts"], t * case["top_k"]
        both = 2 if case["train"] else 1
        return {"bytes": both * t * e * b + 16 * n + 4 * (2 * e + 1) + (both - 1) * (4 * n + 8 * e), "flops": (4 + 6 * both) * t * e}
    k = case["width"]
    if op == "quant":
        return {"bytes": t * (k * (b + 1 + 1 + 4) + 8), "flops": 4 * t * k}
    e, n, inner = case["experts"], t * case["top_k"], case["inner"]
    rows = (2 if case["act"] else 1) * inner
    used = e * (1 - (1 - 1 / e) ** n)            # experts with a row, were all alike
    return {"bytes": used * rows * (k + 4) + t * (k * (b + 1) + 4) + b * n * inner + 4 * n, "flops": 2 * n * rows * k}


# ---- the definitions, in 64 bits -----------------------------------------------------------------------------------

def _exact_route(s):
    c, z = s["case"], s["logits"].double()
    t, e = z.shape
    k, groups = c["top_k"], c["groups"]
    score = torch.sigmoid(z) if c["score"] == "sigmoid" else torch.nan_to_num(torch.softmax(z, dim=1), nan=0.0)
    rank = torch.where(z > -INF, score + (0 if s["bias"] is None else s["bias"].double()), -INF)
    size = e // groups
    if groups > 1:
        value = []
        for i in range(groups):
            top = torch.topk(rank[:, i * size:(i + 1) * size], c["best"], dim=1)[0]
            value.append(torch.where(top[:, 0] > -INF, torch.where(top > -INF, top, 0.0).sum(dim=1), -INF))
        value = torch.stack(value, dim=1)
        for i in range(groups):      # a group is out if as many as are kept come before it
            before = (value > value[:, i:i + 1]).sum(dim=1) + (value[:, :i] == value[:, i:i + 1]).sum(dim=1)
            rank[:, i * size:(i + 1) * size] = torch.where((before < c["kept"])[:, None], rank[:, i * size:(i + 1) * size], -INF)
    place = torch.empty(t, e, dtype=torch.int64, device=z.device)
    for i in range(e):
        place[:, i] = (rank > rank[:, i:i + 1]).sum(dim=1) + (rank[:, :i] == rank[:, i:i + 1]).sum(dim=1)
    chosen = (place < k) & (rank > -INF)
    part = torch.where(chosen, score, 0.0)
    total = part.sum(dim=1, keepdim=True).clamp(min=1e-300)
    full = c["scale"] * (part / total if c["normalise"] else part)
    spot = torch.where(chosen, place, k)
    weight = torch.zeros(t, k + 1, dtype=torch.float64, device=z.device).scatter_(1, spot, full)[:, :k]
    out = [None, weight, None, None, None]
    if not c["train"]:
        return out
    # of each weight by each score, then of each score by each logit
    g = torch.zeros_like(z)
    for j in range(k):
        g += torch.where(spot == j, s["dweight"][:, j:j + 1].double(), 0.0)
    if c["normalise"]:
        g = torch.where(chosen, (g - (g * part).sum(dim=1, keepdim=True) / total) / total, 0.0)
    g = g * c["scale"]
    if c["score"] == "sigmoid":
        out.append(g * score * (1 - score))
    else:
        out.append(score * (g - (g * score).sum(dim=1, keepdim=True)))
    return out + [None] * (s["bias"] is not None)


def _integers(x):
    x = x.double()
    most = x.abs().amax(dim=1, keepdim=True).clamp(min=2.0 ** -100)
    low = torch.floor(127 * x / most)
    rest = 127 * x - low * most       # exact for values of 24 bits, so that a half is a half
    up = (2 * rest > most) | ((2 * rest == most) & (low % 2 != 0))
    return low + up, most / 127


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(s)
    if case["op"] == "quant":
        whole, step = _integers(s["x"])
        return whole * step
    if case["op"] == "orth":
        out = []
        for g in s["g"].double():
            x = g / torch.linalg.matrix_norm(g).clamp(min=1e-300)
            for a, b, c in STEPS:
                if x.shape[0] <= x.shape[1]:
                    q = x @ x.t()
                    x = a * x + b * (q @ x) + c * (q @ (q @ x))
                else:
                    q = x.t() @ x
                    x = a * x + b * (x @ q) + c * ((x @ q) @ q)
            out.append(x)
        return torch.stack(out)
    e, inner, k = case["experts"], case["inner"], case["width"]
    bounds, token = s["offsets"].tolist(), s["order"].long() // case["top_k"]
    whole, step = _integers(s["x"])
    out = []
    for i in range(e):
        rows = token[bounds[i]:bounds[i + 1]]
        y = (whole[rows] * step[rows]) @ (s["wq"][i, :, :k].double() * s["ws"][i].double()[:, None]).t()
        out.append(y[:, :inner] * torch.sigmoid(y[:, :inner]) * y[:, inner:] if case["act"] else y)
    return torch.cat(out)
