"""How far orthogonal updates are from the same steps in 64 bits: the bounds that include/prefree_moe.h states.

More than 64 rows.  Two f16 pieces of X leave 2^-23 of an element, and what that puts where the matrix has nothing grows by
a = 3.4445 in each step: 485, 141, 41 and 12 times what the steps leave, under 10^-4 in all.  What one f16 piece of A, B and
the products' X leaves, 2^-12 / sqrt(3) in the root of the mean square, stays where the matrix has something.  These
roundings, emulated in 64 bits on matrices of 96 to 2048 rows, came to 0.1 to 0.28% after five steps, most for rank 1, where
the diagonal of B is all but a and rounds alike in all rows; 2^-8 is 0.39%.  The result's own rounding comes on top.  Elements
that are all of one magnitude round alike everywhere: what they come to is a recursion of one number, and after five steps at
most 1.04% off for any of 1376 sizes from 65 to 4096 rows; 2^-6 is 1.56%.

Up to 64 rows the second piece is a number of f16, off by 2^-25 / sqrt(3) at the most in the root of the mean square, of X held
times sqrt(n) / 2 and more: 2^-21.8 of its length, times 485 and 1.41 for all steps together, over the 0.7 that a singular
value of 1 becomes: 2^-11.9.  That is less than half a step of f16, 2^-11.
"""
import pytest
import torch

from moe_util import DEV, ROUND
from test_gpu_orthogonalize import FIVE, reference, run

pytestmark = pytest.mark.gpu


def matrices(kind, batch, rows, columns):
    g = torch.Generator(device=DEV)
    g.manual_seed(rows + 3 * columns)
    randn = lambda *shape: torch.randn(*shape, generator=g, device=DEV)  # noqa: E731
    few = lambda r: torch.matmul(randn(batch, rows, r), randn(batch, r, columns))  # noqa: E731
    if kind == "one magnitude":
        return randn(batch, rows, 1).sign() * randn(batch, 1, columns).sign() * 0.37
    if kind == "rank 1 and noise":
        return few(1) + 1e-3 * randn(batch, rows, columns)
    if kind == "all directions":
        return randn(batch, rows, columns)
    return few({"rank 1": 1, "rank 3": 3, "rank n / 8": max(1, min(rows, columns) // 8)}[kind])


def off(got, want):
    return max(float(torch.linalg.matrix_norm(x.double() - y) / torch.linalg.matrix_norm(y)) for x, y in zip(got, want))


@pytest.mark.parametrize("kind", ["rank 1", "rank 3", "rank n / 8", "rank 1 and noise", "one magnitude"])
@pytest.mark.parametrize("batch,rows,columns", [(3, 96, 96), (2, 130, 300), (2, 700, 90), (1, 512, 512), (1, 900, 700), (1, 1024, 1024), (4, 2048, 2048)])
def test_few_directions(kind, batch, rows, columns):
    got, held = run(matrices(kind, batch, rows, columns), "f32", "f16")
    assert off(got, reference(held)) <= (2.0 ** -6 if kind == "one magnitude" else 2.0 ** -8) + ROUND["f16"]


@pytest.mark.parametrize("kind", ["rank 1", "rank 3", "rank 1 and noise", "one magnitude"])
@pytest.mark.parametrize("batch,rows,columns", [(2, 64, 64), (1, 64, 2048), (3, 33, 33), (1, 300, 16)])
def test_few_directions_up_to_64_rows(kind, batch, rows, columns):
    got, held = run(matrices(kind, batch, rows, columns), "f32", "f16")
    assert off(got, reference(held)) <= 2.0 ** -11 + ROUND["f16"]


@pytest.mark.parametrize("n_steps", [6, 7, 8, 10])
@pytest.mark.parametrize("kind", ["rank 1", "rank n / 8", "one magnitude", "all directions"])
@pytest.mark.parametrize("batch,rows,columns", [(2, 70, 105), (1, 192, 128), (1, 512, 512), (2, 40, 64), (1, 300, 64)])
def test_more_steps(kind, batch, rows, columns, n_steps):
    steps = FIVE[:1] * n_steps
    got, held = run(matrices(kind, batch, rows, columns), "f32", "f16", steps=steps)
    bound = 2.0 ** -11 if min(rows, columns) <= 64 else 2.0 ** -6 if kind == "one magnitude" else 2.0 ** -8
    assert off(got, reference(held, steps)) <= bound * 3.5 ** (n_steps - 6) + ROUND["f16"]
