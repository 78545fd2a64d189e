"""examples/expert_layer.py with routing by scores, orthogonal updates and 8-bit integers: that it runs, and its gradient."""
import importlib.util
import math
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

spec = importlib.util.spec_from_file_location(
    "expert_layer_options", os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "expert_layer.py"))
example = importlib.util.module_from_spec(spec)
spec.loader.exec_module(example)


@pytest.mark.parametrize("options", [["--scores", "sigmoid", "--update", "orthogonal", "--bits", "8"], ["--scores", "sigmoid"],
                                     ["--update", "orthogonal", "--width", "136"], ["--bits", "8", "--inner", "40", "--width", "130"]])
def test_runs(options):
    if "136" in options:
        options = options + ["--bits", "8"]
    losses, off = example.main(["--tokens", "200", "--width", "128", "--inner", "64", "--experts", "8", "--steps", "3"] + options)
    assert len(losses) == 3 and all(math.isfinite(v) for v in losses) and math.isfinite(off)


def test_gradient_with_sigmoid_scores():
    """Each gradient against the 64-bit form's, the choice held fixed, and along a direction against differences."""
    t, d, n, e, k = 96, 64, 32, 6, 2
    layer = example.ExpertLayer(d, n, e, k, seed=4, scores="sigmoid")
    b = example.Buffers(layer, t)
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    layer.bias.copy_(torch.randn(e, generator=g, device="cuda") * 0.1)
    x = torch.randn(t, d, generator=g, device="cuda").bfloat16()
    dout = torch.randn(t, d, generator=g, device="cuda").bfloat16()
    out = layer.forward(x, b)
    grad, dx = layer.backward(x, dout, b)
    choice = b.choice.view(t, k).long().cpu()
    w64 = {name: v.double().cpu() for name, v in layer.w.items()}
    x64, d64 = x.double().cpu(), dout.double().cpu()

    def form(w, x):
        s = torch.gather(torch.sigmoid(x @ w["router"].t()), 1, choice)
        weight = s / s.sum(1, keepdim=True)
        y = torch.zeros(t, d, dtype=torch.float64)
        for j in range(k):
            pre = torch.matmul(w["up"][choice[:, j]], x[:, :, None])[..., 0]
            h = torch.nn.functional.silu(pre[:, :n]) * pre[:, n:]
            y = y + weight[:, j:j + 1] * torch.matmul(w["down"][choice[:, j]], h[:, :, None])[..., 0]
        return y

    leaves = {name: v.clone().requires_grad_() for name, v in w64.items()}
    xl = x64.clone().requires_grad_()
    ref = torch.autograd.grad((form(leaves, xl) * d64).sum(), list(leaves.values()) + [xl])

    # every intermediate row is rounded to bf16, by 2^-8 at most and half of that on average; at most seven of them lie on a
    # path, and sums of rounded terms are no further off than their terms in the 2-norm: 8 x 2^-8
    def near(got, want):
        got, want = got.double().cpu(), want.detach()
        return float((got - want).norm()) <= 8 * 2.0 ** -8 * float(want.norm())
    assert near(out, form(w64, x64))
    for (name, v), r in zip(list(grad.items()) + [("x", dx)], ref):
        assert near(v, r), name
    h = 1e-5
    for name in w64:
        way = torch.randn(w64[name].shape, generator=torch.Generator().manual_seed(6), dtype=torch.float64)
        slope = ((form({**w64, name: w64[name] + h * way}, x64) - form({**w64, name: w64[name] - h * way}, x64)) * d64).sum() / (2 * h)
        along = (grad[name].double().cpu() * way).sum()
        assert abs(slope - along) <= 8 * 2.0 ** -8 * ref[list(w64).index(name)].norm() * way.norm(), name
