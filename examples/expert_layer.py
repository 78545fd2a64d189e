"""A layer of experts, trained and then served from 4-bit weights, on the library's expert-layer operators.

    python examples/expert_layer.py [--tokens N] [--width N] [--inner N] [--experts N] [--top-k N] [--steps N]
                                    [--scores sigmoid] [--update orthogonal] [--bits 8]

Training fits the layer to a fixed random layer of the same shape: routing, the gathered product with SwiGLU, the second
product, the weighted sum, and the gradients of each, from this package; the update of the weights is torch's.  Serving
holds the trained weights in 4-bit blocks and answers tokens one at a time.  Prints the loss on the way and how far the
4-bit answers are from the 16-bit ones.

--scores sigmoid routes by sigmoid scores and a bias of the choice that each step moves towards even loads.  --update
orthogonal moves the experts' weights by their momentum made nearly orthogonal, the router's as before.  --bits 8 serves
from 8-bit integers with a scale a row.
"""
import argparse
import importlib
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
pf = importlib.import_module("prefree-public_amd")

BF16, F32, I32, I8, U8 = torch.bfloat16, torch.float32, torch.int32, torch.int8, torch.uint8


def empty(*shape, dtype=BF16):
    return torch.empty(*shape, dtype=dtype, device="cuda")


class Buffers:
    """What one pass over `tokens` tokens writes; allocated once."""

    def __init__(self, layer, tokens):
        t, e, k, d, n = tokens, layer.experts, layer.top_k, layer.width, layer.inner
        self.tokens, self.slots = t, t * k
        self.logits, self.weight = empty(t, e), empty(t, k, dtype=F32)
        self.choice, self.order, self.slot = (empty(t * k, dtype=I32) for _ in range(3))
        self.offsets, self.work = empty(e + 1, dtype=I32), empty(max(1, pf.moe_route_workspace(t, e)), dtype=U8)
        self.hidden, self.pre, self.y, self.out = empty(t * k, n), empty(t * k, 2 * n), empty(t * k, d), empty(t, d)


class ExpertLayer:
    def __init__(self, width, inner, experts, top_k, seed=0, scores=None):
        self.width, self.inner, self.experts, self.top_k, self.scores = width, inner, experts, top_k, scores
        self.bias = torch.zeros(experts, dtype=F32, device="cuda")       # of the choice by sigmoid scores
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)

        def weights(*shape):
            return (torch.randn(*shape, generator=g, device="cuda") * shape[-1] ** -0.5)
        # held in fp32 for the updates; the products take the 16-bit copies
        self.master = {"router": weights(experts, width), "up": weights(experts, 2 * inner, width), "down": weights(experts, width, inner)}
        self.w = {name: v.to(BF16) for name, v in self.master.items()}

    def choose(self, x, b):
        """The experts of each token: logits, then the choice, its weights and the order by expert."""
        t, e, k, d = b.tokens, self.experts, self.top_k, self.width
        pf.moe_mm(x, t, None, 1, self.w["router"], None, 1, t, e, d, b.logits)
        if self.scores == "sigmoid":
            pf.moe_route_scores(b.logits, t, e, k, b.choice, b.weight, b.offsets, b.order, b.slot, b.work, dtype="bf16", bias=self.bias)
        else:
            pf.moe_route(b.logits, t, e, k, b.choice, b.weight, b.offsets, b.order, b.slot, b.work, dtype="bf16")

    def forward(self, x, b):
        t, e, k, d, n = b.tokens, self.experts, self.top_k, self.width, self.inner
        self.choose(x, b)
        pf.moe_mm(x, t, b.order, k, self.w["up"], b.offsets, e, b.slots, n, d, b.hidden, act="swiglu", pre=b.pre)
        pf.moe_mm(b.hidden, b.slots, None, 1, self.w["down"], b.offsets, e, b.slots, d, n, b.y)
        pf.moe_combine(b.y, b.slot, b.weight, t, k, d, b.out)
        return b.out

    def backward(self, x, dout, b):
        """Gradients of the weights (fp32) and of x from that of the result, after forward(x, b)."""
        t, e, k, d, n = b.tokens, self.experts, self.top_k, self.width, self.inner
        dy, dweight, dhidden, dpre = empty(b.slots, d), empty(t, k, dtype=F32), empty(b.slots, n), empty(b.slots, 2 * n)
        dslots, dx, dlogits, dx_router = empty(b.slots, d), empty(t, d), empty(t, e), empty(t, d)
        grad = {name: torch.empty_like(v) for name, v in self.master.items()}
        pf.moe_combine_backward(dout, b.y, b.slot, b.weight, t, k, d, dy, dweight)
        pf.moe_mm_dw(dy, b.hidden, b.slots, None, 1, b.offsets, e, b.slots, d, n, grad["down"], dw_dtype="f32")
        pf.moe_mm_dx(dy, self.w["down"], b.offsets, e, b.slots, d, n, dhidden)
        pf.swiglu_backward(dhidden, b.pre, b.slots, n, dpre)
        pf.moe_mm_dw(dpre, x, t, b.order, k, b.offsets, e, b.slots, 2 * n, d, grad["up"], dw_dtype="f32")
        pf.moe_mm_dx(dpre, self.w["up"], b.offsets, e, b.slots, 2 * n, d, dslots)
        pf.moe_combine(dslots, b.slot, None, t, k, d, dx)                  # a token's gradient is the sum of its slots'
        if self.scores == "sigmoid":
            pf.moe_route_scores_backward(b.logits, t, e, k, b.choice, b.weight, dweight, dlogits, dtype="bf16")
        else:
            pf.moe_route_backward(b.logits, t, e, k, b.choice, b.weight, dweight, dlogits, dtype="bf16")
        pf.moe_mm_dw(dlogits, x, t, None, 1, None, 1, t, e, d, grad["router"], dw_dtype="f32")
        pf.moe_mm_dx(dlogits, self.w["router"], None, 1, t, e, d, dx_router)
        return grad, dx + dx_router

    def balance(self, b, rate=1e-3):
        """The bias of experts with fewer slots than the mean goes up, of those with more down."""
        pf.moe_balance(b.offsets, self.experts, rate, self.bias, self.bias)

    def update(self, grad, optimiser):
        for name, v in self.master.items():
            v.grad = grad[name]
        optimiser.step()
        for name, v in self.master.items():
            self.w[name].copy_(v)


class Orthogonal(torch.optim.Adam):
    """The experts' weights, a batch of matrices each, go against their momentum made nearly orthogonal; `others` as with Adam."""

    def __init__(self, matrices, others, lr, keep=0.9):
        super().__init__(others, lr=lr)
        self.lr, self.keep, self.matrices = lr, keep, list(matrices)
        self.momentum = [torch.zeros_like(m) for m in self.matrices]
        self.out = [torch.empty_like(m, dtype=BF16) for m in self.matrices]
        self.work = empty(max(pf.orthogonalize_workspace(*m.shape) for m in self.matrices), dtype=U8)

    def step(self):
        super().step()
        for m, v, out in zip(self.matrices, self.momentum, self.out):
            v.mul_(self.keep).add_(m.grad)
            pf.orthogonalize(v, *m.shape, out, self.work)
            m.add_(out, alpha=-self.lr)


class FourBitLayer:
    """The layer with its experts' weights in 4-bit blocks; the router stays in 16 bits."""

    def __init__(self, layer):
        self.layer, self.blocks = layer, {}
        for name in ("up", "down"):
            w = layer.w[name]
            self.blocks[name] = blocks(w.view(-1, w.shape[-1]))

    def answer(self, x, b):
        L, t, k = self.layer, b.tokens, self.layer.top_k
        L.choose(x, b)
        codes, scales = blocks(x)
        pf.moe_mm_mx4(codes, scales, t, b.order, k, *self.blocks["up"], b.offsets, L.experts, b.slots, L.inner, L.width,
                      b.hidden, act="swiglu")
        codes, scales = blocks(b.hidden)
        pf.moe_mm_mx4(codes, scales, b.slots, None, 1, *self.blocks["down"], b.offsets, L.experts, b.slots, L.width, L.inner, b.y)
        pf.moe_combine(b.y, b.slot, b.weight, t, k, L.width, b.out)
        return b.out


class EightBitLayer:
    """The layer with its experts' weights in 8-bit integers; the router stays in 16 bits."""

    def __init__(self, layer):
        self.layer, self.integers = layer, {}
        for name in ("up", "down"):
            w = layer.w[name]
            self.integers[name] = integers(w.view(-1, w.shape[-1]))

    def answer(self, x, b):
        L, t, k = self.layer, b.tokens, self.layer.top_k
        L.choose(x, b)
        codes, scales = integers(x)
        pf.moe_mm_i8(codes, scales, t, b.order, k, *self.integers["up"], b.offsets, L.experts, b.slots, L.inner, L.width, b.hidden, act="swiglu")
        codes, scales = integers(b.hidden)
        pf.moe_mm_i8(codes, scales, b.slots, None, 1, *self.integers["down"], b.offsets, L.experts, b.slots, L.width, L.inner, b.y)
        pf.moe_combine(b.y, b.slot, b.weight, t, k, L.width, b.out)
        return b.out


def integers(x):
    codes, scales = empty(x.shape[0], pf.i8_row(x.shape[1]), dtype=I8), empty(x.shape[0], dtype=F32)
    pf.i8_quantize(x, x.shape[0], x.shape[1], codes, scales, dtype="bf16")
    return codes, scales


def blocks(x):
    codes, scales = empty(x.shape[0], x.shape[1] // 2, dtype=U8), empty(x.shape[0], x.shape[1] // 32, dtype=U8)
    pf.mx4_quantize(x, x.shape[0], x.shape[1], codes, scales, dtype="bf16")
    return codes, scales


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in (("tokens", 2048), ("width", 512), ("inner", 256), ("experts", 16), ("top-k", 2), ("steps", 40), ("served", 16)):
        ap.add_argument("--" + name, type=int, default=value)
    ap.add_argument("--rate", type=float, default=5e-3)
    ap.add_argument("--scores", choices=("softmax", "sigmoid"), default="softmax")
    ap.add_argument("--update", choices=("adam", "orthogonal"), default="adam")
    ap.add_argument("--bits", type=int, choices=(4, 8), default=4)
    o = ap.parse_args(argv)
    if o.bits == 4 and (o.width % 32 or o.inner % 32):
        ap.error("--width and --inner are multiples of 32, the length of a 4-bit block")
    teacher, layer = (ExpertLayer(o.width, o.inner, o.experts, o.top_k, seed=s, scores=o.scores) for s in (1, 2))
    for name in ("router", "up"):     # fitted: the second product
        layer.master[name].copy_(teacher.master[name])
        layer.w[name].copy_(teacher.w[name])
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    x = torch.randn(o.tokens, o.width, generator=g, device="cuda").to(BF16)
    b = Buffers(layer, o.tokens)
    if o.update == "orthogonal":
        optimiser = Orthogonal([layer.master["up"], layer.master["down"]], [layer.master["router"]], o.rate)
    else:
        optimiser = torch.optim.Adam(layer.master.values(), lr=o.rate)
    want = teacher.forward(x, b).float().clone()
    losses = []
    for step in range(o.steps):
        off = layer.forward(x, b).float() - want
        losses.append(float(off.square().mean() / want.square().mean()))
        if step % 10 == 0 or step == o.steps - 1:
            print(f"step {step:4d}  loss {losses[-1]:.4f}", flush=True)
        grad, _ = layer.backward(x, off.to(BF16), b)      # of half the sum of squares
        layer.update(grad, optimiser)
        if o.scores == "sigmoid":
            layer.balance(b)

    served, one = (FourBitLayer if o.bits == 4 else EightBitLayer)(layer), Buffers(layer, 1)
    whole = layer.forward(x, b)
    far = size = 0.0
    torch.cuda.synchronize()
    began = time.perf_counter()
    answers = [served.answer(x[i:i + 1], one).clone() for i in range(o.served)]
    torch.cuda.synchronize()
    took = (time.perf_counter() - began) / max(1, o.served)
    for i, y in enumerate(answers):
        far += float((y[0].float() - whole[i].float()).square().sum())
        size += float(whole[i].float().square().sum())
    off = (far / size) ** 0.5 if size else 0.0
    print(f"{o.bits}-bit answers: {off:.3f} off in the 2-norm, {took * 1e6:.0f} us a token")
    return losses, off


if __name__ == "__main__":
    main()
