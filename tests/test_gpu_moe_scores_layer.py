"""Routing by scores, the products with their gradients, the balance of the loads, orthogonal updates and the 8-bit form
(include/prefree_moe.h) as a layer runs them: step by step against 64-bit forms of what each reads, on another stream and
in replayed graphs."""
import pytest
import torch

import prefree_amd as pf
from moe_util import DEV, close, product, swiglu
from test_gpu_moe_i8 import integers
from test_gpu_moe_i8 import reference as product_i8
from test_gpu_moe_scores import reference as route_reference
from test_gpu_orthogonalize import near
from test_gpu_orthogonalize import reference as orthogonal

pytestmark = pytest.mark.gpu

OUTPUTS = ("choice", "weight", "offsets", "order", "slot", "out", "dw1", "dw2", "dx", "dz", "bias", "update1", "update2", "xq", "xs",
           "hq", "hs", "served")


class Layer:
    """`tokens` of width d, the top k of e experts of inner width n in `groups` groups, of which `kept` are looked at."""

    def __init__(self, tokens, e, k, groups, kept, d, n):
        self.sizes = tokens, e, k, d, n
        g = torch.Generator(device=DEV)
        g.manual_seed(tokens)
        randn = lambda *shape: torch.randn(*shape, generator=g, device=DEV)  # noqa: E731
        b = lambda *shape: torch.zeros(*shape, dtype=torch.bfloat16, device=DEV)  # noqa: E731
        i = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=DEV)  # noqa: E731
        f = lambda *shape: torch.zeros(*shape, device=DEV)  # noqa: E731
        u = lambda *shape: torch.zeros(*shape, dtype=torch.uint8, device=DEV)  # noqa: E731
        c = lambda rows, k: torch.zeros(rows, pf.i8_row(k), dtype=torch.int8, device=DEV)  # noqa: E731
        s = tokens * k
        self.how = dict(score="sigmoid", normalise=True, scale=2.5)
        self.z, self.x, self.dout, self.bias0 = randn(tokens, e).bfloat16(), randn(tokens, d).bfloat16(), randn(tokens, d).bfloat16(), randn(e) * 0.1
        self.z[3::16] = -float("inf")                 # tokens of the padding
        self.groups = dict(groups=groups, groups_kept=kept)
        self.w1, self.w2 = (randn(e, 2 * n, d) * d ** -0.5).bfloat16(), (randn(e, d, n) * n ** -0.5).bfloat16()
        self.choice, self.weight, self.offsets, self.order, self.slot = i(tokens, k), f(tokens, k), i(e + 1), i(s), i(s)
        self.work = u(pf.moe_route_workspace(tokens, e))
        self.h, self.pre, self.y, self.out, self.bias = b(s, n), b(s, 2 * n), b(s, d), b(tokens, d), f(e)
        self.dy, self.dweight, self.dh, self.dpre, self.dxs = b(s, d), f(tokens, k), b(s, n), b(s, 2 * n), b(s, d)
        self.dx, self.dz, self.dw1, self.dw2 = b(tokens, d), b(tokens, e), f(e, 2 * n, d), f(e, d, n)
        self.update1, self.update2 = b(e, 2 * n, d), b(e, d, n)
        self.orth = u(max(pf.orthogonalize_workspace(*w.shape) for w in (self.dw1, self.dw2)))
        self.w1q, self.w1s, self.w2q, self.w2s = c(e * 2 * n, d), f(e * 2 * n), c(e * d, n), f(e * d)
        self.xq, self.xs, self.hq, self.hs, self.h8, self.y8, self.served = c(tokens, d), f(tokens), c(s, n), f(s), b(s, n), b(s, d), b(tokens, d)
        pf.i8_quantize(self.w1, e * 2 * n, d, self.w1q, self.w1s)
        pf.i8_quantize(self.w2, e * d, n, self.w2q, self.w2s)
        torch.cuda.synchronize()

    def run(self, stream):
        t, e, k, d, n = self.sizes
        s, on = t * k, dict(stream=stream)
        pf.moe_route_scores(self.z, t, e, k, self.choice, self.weight, self.offsets, self.order, self.slot, self.work, dtype="bf16",
                            bias=self.bias0, **self.how, **self.groups, **on)
        pf.moe_mm(self.x, t, self.order, k, self.w1, self.offsets, e, s, n, d, self.h, act="swiglu", pre=self.pre, **on)
        pf.moe_mm(self.h, s, None, 1, self.w2, self.offsets, e, s, d, n, self.y, **on)
        pf.moe_combine(self.y, self.slot, self.weight, t, k, d, self.out, **on)
        pf.moe_combine_backward(self.dout, self.y, self.slot, self.weight, t, k, d, self.dy, self.dweight, **on)
        pf.moe_mm_dx(self.dy, self.w2, self.offsets, e, s, d, n, self.dh, **on)
        pf.moe_mm_dw(self.dy, self.h, s, None, 1, self.offsets, e, s, d, n, self.dw2, dw_dtype="f32", **on)
        pf.swiglu_backward(self.dh, self.pre, s, n, self.dpre, **on)
        pf.moe_mm_dx(self.dpre, self.w1, self.offsets, e, s, 2 * n, d, self.dxs, **on)
        pf.moe_mm_dw(self.dpre, self.x, t, self.order, k, self.offsets, e, s, 2 * n, d, self.dw1, dw_dtype="f32", **on)
        pf.moe_combine(self.dxs, self.slot, None, t, k, d, self.dx, **on)
        pf.moe_route_scores_backward(self.z, t, e, k, self.choice, self.weight, self.dweight, self.dz, dtype="bf16", **self.how, **on)
        pf.moe_balance(self.offsets, e, 1e-3, self.bias0, self.bias, **on)
        pf.orthogonalize(self.dw1, *self.dw1.shape, self.update1, self.orth, **on)
        pf.orthogonalize(self.dw2, *self.dw2.shape, self.update2, self.orth, **on)      # the same workspace, in order
        pf.i8_quantize(self.x, t, d, self.xq, self.xs, **on)
        pf.moe_mm_i8(self.xq, self.xs, t, self.order, k, self.w1q, self.w1s, self.offsets, e, s, n, d, self.h8, act="swiglu", **on)
        pf.i8_quantize(self.h8, s, n, self.hq, self.hs, **on)
        pf.moe_mm_i8(self.hq, self.hs, s, None, 1, self.w2q, self.w2s, self.offsets, e, s, d, n, self.y8, **on)
        pf.moe_combine(self.y8, self.slot, self.weight, t, k, d, self.served, **on)

    def outputs(self):
        return {name: getattr(self, name) for name in OUTPUTS}

    def wipe(self):
        # rows behind the last expert's are read by the quantisation and by nothing else: left as they are, zeros
        for v in self.outputs().values():
            v.fill_(3)
        self.work.fill_(0x5a)
        self.orth.fill_(0x7e)


def test_steps_of_a_layer():
    t, e, k, d, n = 150, 12, 3, 96, 40
    layer = Layer(t, e, k, 4, 2, d, n)
    layer.wipe()
    layer.run(None)
    torch.cuda.synchronize()
    want = route_reference(layer.z.double().cpu().numpy(), k, bias=layer.bias0.cpu().numpy(), groups=4, kept=2, **layer.how)
    got = [v.cpu().numpy() for v in (layer.choice, layer.weight, layer.offsets, layer.order, layer.slot)]
    assert all((g == w).all() for name, g, w in zip("cwosl", got, want) if name != "w")
    # In steps of 2^-24: a sigmoid's exponential |z| + 2, its sum 1, its quotient 2, at |z| < 5 ten; so ten for the sum of
    # three as well and two for its additions; the quotient three, the scale one: 26
    assert abs(layer.z[layer.z > -float("inf")]).max() < 5
    assert (abs(got[1] - want[1]) <= 26 * 2.0 ** -24 * abs(want[1])).all()
    at = layer.offsets.tolist()
    used = at[-1]
    token = layer.order[:used].long() // k
    weight = torch.from_numpy(want[1]).to(DEV)
    w1q, w2q, w1s, w2s = layer.w1q.view(e, 2 * n, -1), layer.w2q.view(e, d, -1), layer.w1s.view(e, -1), layer.w2s.view(e, -1)
    for i in range(e):
        a, b = at[i], at[i + 1]
        if a == b:
            continue
        pre, slack = product(layer.x[token[a:b]], layer.w1[i])
        close(layer.pre[a:b], pre, slack, "bf16", "pre")
        close(layer.h[a:b], *swiglu(pre[:, :n], pre[:, n:], slack[:, :n], slack[:, n:]), "bf16", "h")
        close(layer.y[a:b], *product(layer.h[a:b], layer.w2[i]), "bf16", "y")
        close(layer.dw2[i], *product(layer.dy[a:b].t(), layer.h[a:b].t()), "f32", "dw2")
        close(layer.dw1[i], *product(layer.dpre[a:b].t(), layer.x[token[a:b]].t()), "f32", "dw1")
        close(layer.h8[a:b], *product_i8(layer.xq[token[a:b]], layer.xs[token[a:b]], w1q[i], w1s[i], "swiglu", n), "bf16", "h8")
        close(layer.y8[a:b], *product_i8(layer.hq[a:b], layer.hs[a:b], w2q[i], w2s[i], "none", d), "bf16", "y8")
    for rows, codes, scales in ((layer.x, layer.xq, layer.xs), (layer.h8[:used], layer.hq[:used], layer.hs[:used])):
        ints, most = integers(rows)
        assert torch.equal(codes[:, :rows.shape[1]], ints) and torch.equal(scales, (most / 127).float())
    slot = layer.slot.view(t, k).long()
    for y, out in ((layer.y, layer.out), (layer.y8, layer.served)):
        terms = torch.where(slot[..., None] >= 0, y.double()[slot.clamp(min=0)], 0) * weight[..., None]
        # 26 steps of 2^-24 in a weight, one in its product and two in a sum of three
        close(out, terms.sum(1), 29 * 2.0 ** -24 * terms.abs().sum(1), "bf16", "out")
    # the gradient of the logits of sum(weight dweight), the choice held
    z = layer.z.double().clone().requires_grad_()
    s = torch.where(layer.choice >= 0, torch.sigmoid(torch.gather(z, 1, layer.choice.long().clamp(min=0))), 0)
    s = s * layer.how["scale"] / s.sum(1, keepdim=True).clamp(min=1e-300)
    dz, = torch.autograd.grad((s * layer.dweight.double()).sum(), z)
    # dz_i = (1 - s_i) w_i (d_i - sum_j w_j d_j / scale), terms of at most w_i |d_i| and sum_j w_j |d_j|; in steps of 2^-24: 26
    # for w_i, 26 + 4 for those of the sum, ten for s_i, a difference and three products
    size = (weight.abs() * layer.dweight.double().abs()).sum(1, keepdim=True)
    close(layer.dz, torch.nan_to_num(dz), 70 * 2.0 ** -24 * 2 * size, "bf16", "dz")
    loads = (layer.offsets[1:] - layer.offsets[:-1]).double()
    close(layer.bias, layer.bias0.double() + 1e-3 * torch.sign(loads.mean() - loads), 2.0 ** -24 * 1e-3, "f32", "bias")
    near(layer.update1, orthogonal(layer.dw1), "bf16")
    near(layer.update2, orthogonal(layer.dw2), "bf16")


# 66 blocks of tokens: two launches of the routing; narrow and square updates; and 1025 blocks: three launches
@pytest.mark.parametrize("sizes", [(4161, 8, 2, 4, 2, 384, 256), (65537, 32, 4, 8, 3, 64, 24)])
def test_on_another_stream_and_in_graphs(sizes):
    layer = Layer(*sizes)
    layer.wipe()
    layer.run(None)
    torch.cuda.synchronize()
    first = {k: v.clone() for k, v in layer.outputs().items()}
    used = int(first["offsets"][-1])
    assert used == (first["choice"] >= 0).sum()
    same = lambda: [k for k, v in layer.outputs().items() if not torch.equal(v, first[k])]  # noqa: E731
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        layer.wipe()
        layer.run(stream)
        stream.synchronize()
        assert not same(), "another stream"
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
        for graph in graphs:                                # two graphs of the same workspaces, replayed in turn
            with torch.cuda.graph(graph, stream=stream):
                layer.run(stream)
        for replay in range(4):
            layer.wipe()
            graphs[replay % 2].replay()
            graphs[1 - replay % 2].replay()
            stream.synchronize()
            assert not same(), f"replay {replay}"
            layer.wipe()
            layer.run(stream)                               # eager work between the replays
            stream.synchronize()
            assert not same(), f"after replay {replay}"
