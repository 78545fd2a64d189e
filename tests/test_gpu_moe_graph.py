"""A whole expert layer (include/prefree_moe.h) on another stream and in a replayed graph, at sizes whose routing takes
several launches and whose products take the kernel with a workgroup a CU."""
import pytest
import torch

import prefree_amd as pf
from moe_util import DEV

pytestmark = pytest.mark.gpu

OUTPUTS = ("choice", "weight", "offsets", "order", "slot", "out", "dw1", "dw2", "dx", "dz", "h4")


class Layer:
    """`tokens` of width d, the top k of e experts of inner width n; forward, backward and the 4-bit product."""

    def __init__(self, tokens, e, k, d, n):
        self.sizes = tokens, e, k, d, n
        g = torch.Generator(device=DEV)
        g.manual_seed(tokens)
        randn = lambda *shape: torch.randn(*shape, generator=g, device=DEV).bfloat16()  # noqa: E731
        b = lambda *shape: torch.zeros(*shape, dtype=torch.bfloat16, device=DEV)  # noqa: E731
        i = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=DEV)  # noqa: E731
        f = lambda *shape: torch.zeros(*shape, device=DEV)  # noqa: E731
        u = lambda *shape: torch.zeros(*shape, dtype=torch.uint8, device=DEV)  # noqa: E731
        s = tokens * k
        self.z, self.x, self.dout = randn(tokens, e), randn(tokens, d), randn(tokens, d)
        self.z[3::16] = -float("inf")
        self.w1, self.w2 = randn(e, 2 * n, d) * d ** -0.5, randn(e, d, n) * n ** -0.5
        self.choice, self.weight, self.offsets, self.order, self.slot = i(tokens, k), f(tokens, k), i(e + 1), i(s), i(s)
        self.work = u(pf.moe_route_workspace(tokens, e))
        self.h, self.pre, self.y, self.out = b(s, n), b(s, 2 * n), b(s, d), b(tokens, d)
        self.dy, self.dweight, self.dh, self.dpre, self.dxs = b(s, d), f(tokens, k), b(s, n), b(s, 2 * n), b(s, d)
        self.dx, self.dz, self.dw1, self.dw2, self.h4 = b(tokens, d), b(tokens, e), f(e, 2 * n, d), f(e, d, n), b(s, n)
        self.xq, self.xs, self.wq, self.ws = u(tokens, d // 2), u(tokens, d // 32), u(e * 2 * n, d // 2), u(e * 2 * n, d // 32)
        pf.mx4_quantize(self.w1, e * 2 * n, d, self.wq, self.ws)
        torch.cuda.synchronize()

    def run(self, stream):
        t, e, k, d, n = self.sizes
        s = t * k
        pf.moe_route(self.z, t, e, k, self.choice, self.weight, self.offsets, self.order, self.slot, self.work, dtype="bf16", stream=stream)
        pf.moe_mm(self.x, t, self.order, k, self.w1, self.offsets, e, s, n, d, self.h, act="swiglu", pre=self.pre, stream=stream)
        pf.moe_mm(self.h, s, None, 1, self.w2, self.offsets, e, s, d, n, self.y, stream=stream)
        pf.moe_combine(self.y, self.slot, self.weight, t, k, d, self.out, stream=stream)
        pf.moe_combine_backward(self.dout, self.y, self.slot, self.weight, t, k, d, self.dy, self.dweight, stream=stream)
        pf.moe_mm_dx(self.dy, self.w2, self.offsets, e, s, d, n, self.dh, stream=stream)
        pf.moe_mm_dw(self.dy, self.h, s, None, 1, self.offsets, e, s, d, n, self.dw2, dw_dtype="f32", stream=stream)
        pf.swiglu_backward(self.dh, self.pre, s, n, self.dpre, stream=stream)
        pf.moe_mm_dx(self.dpre, self.w1, self.offsets, e, s, 2 * n, d, self.dxs, stream=stream)
        pf.moe_mm_dw(self.dpre, self.x, t, self.order, k, self.offsets, e, s, 2 * n, d, self.dw1, dw_dtype="f32", stream=stream)
        pf.moe_combine(self.dxs, self.slot, None, t, k, d, self.dx, stream=stream)
        pf.moe_route_backward(self.z, t, e, k, self.choice, self.weight, self.dweight, self.dz, dtype="bf16", stream=stream)
        pf.mx4_quantize(self.x, t, d, self.xq, self.xs, stream=stream)
        pf.moe_mm_mx4(self.xq, self.xs, t, self.order, k, self.wq, self.ws, self.offsets, e, s, n, d, self.h4, act="swiglu", stream=stream)

    def outputs(self):
        return {name: getattr(self, name) for name in OUTPUTS}

    def wipe(self):
        for v in self.outputs().values():
            v.fill_(3)
        self.work.fill_(0x5a)


# 66 blocks of tokens: two launches of the routing, 256 x 256 tiles in every kind of product; and 1025 blocks: three launches
@pytest.mark.parametrize("sizes", [(4161, 8, 2, 1024, 1024), (65537, 5, 2, 64, 64)])
def test_layer_on_another_stream_and_in_a_graph(sizes):
    layer = Layer(*sizes)
    layer.wipe()
    layer.run(None)
    torch.cuda.synchronize()
    first = {k: v.clone() for k, v in layer.outputs().items()}
    assert int(first["offsets"][-1]) == (first["choice"] >= 0).sum()
    same = lambda: [k for k, v in layer.outputs().items() if not torch.equal(v, first[k])]  # noqa: E731
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        layer.wipe()
        layer.run(stream)
        stream.synchronize()
        assert not same(), "another stream"
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            layer.run(stream)
        for replay in range(4):
            layer.wipe()
            graph.replay()
            stream.synchronize()
            assert not same(), f"replay {replay}"
            layer.wipe()
            layer.run(stream)                      # eager work between the replays
            stream.synchronize()
            assert not same(), f"after replay {replay}"
