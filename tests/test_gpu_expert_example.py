"""examples/expert_layer.py: a layer of experts that is trained and served from 4-bit weights."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

spec = importlib.util.spec_from_file_location(
    "expert_layer", os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "expert_layer.py"))
example = importlib.util.module_from_spec(spec)
spec.loader.exec_module(example)


def test_trains_and_serves():
    losses, off = example.main(["--tokens", "512", "--width", "128", "--inner", "64", "--experts", "8", "--steps", "30"])
    # two independent layers of equal size are sqrt(2) apart, squared 2; fitting the second product of the same routing
    # and activation is a least-squares problem that descends
    assert losses[-1] < 0.5 * losses[0]
    # 4-bit weights and activations: each value within 1/4 of itself at worst and about 1/8 on average, in three places
    assert off < 0.4


def test_gradient_of_the_whole_layer():
    """The layer's gradient along a direction against the difference of its 64-bit form, the choice held fixed."""
    t, d, n, e, k = 96, 64, 32, 6, 2
    layer = example.ExpertLayer(d, n, e, k, seed=4)
    b = example.Buffers(layer, t)
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    x = torch.randn(t, d, generator=g, device="cuda").bfloat16()
    dout = torch.randn(t, d, generator=g, device="cuda").bfloat16()
    out = layer.forward(x, b)
    grad, dx = layer.backward(x, dout, b)
    choice = b.choice.view(t, k).long().cpu()

    w64 = {name: v.double().cpu() for name, v in layer.w.items()}
    x64, d64 = x.double().cpu(), dout.double().cpu()

    def form(w, x):
        weight = torch.softmax(torch.gather(x @ w["router"].t(), 1, choice), 1)
        y = torch.zeros(t, d, dtype=torch.float64)
        for j in range(k):
            pre = torch.matmul(w["up"][choice[:, j]], x[:, :, None])[..., 0]
            h = torch.nn.functional.silu(pre[:, :n]) * pre[:, n:]
            y = y + weight[:, j:j + 1] * torch.matmul(w["down"][choice[:, j]], h[:, :, None])[..., 0]
        return y

    leaves = {name: v.clone().requires_grad_() for name, v in w64.items()}
    xl = x64.clone().requires_grad_()
    ref = torch.autograd.grad((form(leaves, xl) * d64).sum(), list(leaves.values()) + [xl])
    # Every intermediate row is rounded to bf16 (2^-9 of itself each time, half a unit in the last of 8 bits), at most
    # seven of them on a path, and sums of rounded terms are no further off than their terms in the 2-norm: 8 x 2^-8.
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
        # |<grad - ref, way>| <= ||grad - ref|| ||way||
        assert abs(slope - along) <= 8 * 2.0 ** -8 * ref[list(w64).index(name)].norm() * way.norm(), name
