"""Orthogonal updates (include/prefree_moe.h) against the same steps in 64 bits.

Tolerance: a step rounds X, A and B to f16, by at most 2^-12 of an element and 2^-12 / sqrt(3) in the root of the mean
square.  In b A X and c A A X, b = -4.775 and c = 2.03, that is three and five factors, at singular values of 1: sqrt(3
b^2 + 5 c^2) = 9.4 of them, 1.3e-3 a step; a step's errors shrink by |a + 3 b + 5 c| = 0.72 in each later one, so that
all are 1.9e-3 in the 2-norm.  Four times that is 2^-7, with the result's rounding besides.
"""
import pytest
import torch

import prefree_amd as pf
from moe_util import DEV, NAN, ROUND, TORCH, strided

pytestmark = pytest.mark.gpu

FIVE = pf.ORTHOGONAL_STEPS


def reference(g, steps=FIVE):
    out = []
    for x in g.double():
        x = x / torch.linalg.matrix_norm(x).clamp(min=1e-300)
        for a, b, c in steps:
            q = x @ x.t() if x.shape[0] <= x.shape[1] else x.t() @ x
            x = a * x + (b * (q @ x) + c * (q @ (q @ x)) if x.shape[0] <= x.shape[1] else b * (x @ q) + c * ((x @ q) @ q))
        out.append(x)
    return torch.stack(out)


def run(g, dtype="f32", out_dtype="bf16", steps=FIVE, ld=0, shift=0, ld_out=0, shift_out=0, stream=None):
    batch, rows, columns = g.shape
    view, ld = strided(g.reshape(batch * rows, columns).to(TORCH[dtype]), ld, shift)
    out, lo = strided(torch.full((batch * rows, columns), NAN, dtype=TORCH[out_dtype], device=DEV), ld_out, shift_out, fill=7.0)
    need = pf.orthogonalize_workspace(batch, rows, columns)
    work = torch.full((need + 64,), 0x7e, dtype=torch.uint8, device=DEV)
    pf.orthogonalize(view, batch, rows, columns, out, work, dtype=dtype, out_dtype=out_dtype, steps=steps, workspace_bytes=need, ld_g=ld,
                     ld_out=lo, stream=stream)
    torch.cuda.synchronize()
    assert (work[need:] == 0x7e).all()
    if lo > columns:
        gaps = out.as_strided((batch * rows - 1, lo - columns), (lo, 1), out.storage_offset() + columns)
        assert (gaps == 7).all()
    return out.reshape(batch, rows, columns).clone(), view.reshape(batch, rows, columns)


def near(got, want, out_dtype, slack=2.0 ** -7):
    for i in range(got.shape[0]):
        off = torch.linalg.matrix_norm(got[i].double() - want[i])
        size = torch.linalg.matrix_norm(want[i])
        assert off <= (slack + ROUND[out_dtype]) * size, (i, float(off / size))


def momentum(batch, rows, columns, seed, few=None):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=g, device=DEV)  # noqa: E731
    if few is None:
        return randn(batch, rows, columns)
    return torch.matmul(randn(batch, rows, few), randn(batch, few, columns)) * few ** -0.5


@pytest.mark.parametrize("dtype,out_dtype", [("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("batch,rows,columns", [(1, 1, 1), (2, 1, 5), (1, 7, 1), (3, 33, 7), (1, 31, 65), (2, 64, 2048), (1, 100, 100),
                                                (1, 257, 513), (2, 300, 200), (3, 129, 128), (1, 640, 1100), (5, 96, 33)])
def test_orthogonalize(batch, rows, columns, dtype, out_dtype):
    g = momentum(batch, rows, columns, rows + columns)
    got, held = run(g, dtype, out_dtype)
    near(got, reference(held), out_dtype)


@pytest.mark.parametrize("batch,rows,columns,few", [(2, 64, 64, 1), (1, 256, 512, 16), (1, 512, 256, 3), (20, 700, 1030, 80), (1, 1024, 1024, 100)])
def test_few_directions(batch, rows, columns, few):
    """What rounding puts where the matrix has nothing is not carried along."""
    got, held = run(momentum(batch, rows, columns, few, few), "bf16")
    near(got, reference(held), "bf16")


@pytest.mark.parametrize("ld,shift,lo,so", [(70, 0, 0, 0), (67, 1, 69, 3), (0, 5, 72, 1)])
@pytest.mark.parametrize("rows", [40, 90])
def test_strides(rows, ld, shift, lo, so):
    for dtype, out in (("f32", "bf16"), ("bf16", "f16")):
        got, held = run(momentum(3, rows, 67, 1), dtype, out, ld=ld, shift=shift, ld_out=lo, shift_out=so)
        near(got, reference(held), out)


def test_sizes_of_elements():
    """Squares that fp32 does not hold."""
    g = momentum(4, 48, 80, 2)
    scaled = g * torch.tensor([1e-37, 1e-30, 1e25, 1e36], device=DEV)[:, None, None]
    got, held = run(scaled)
    near(got, reference(held), "bf16")


def test_zeros_and_matrices_without_an_answer():
    g = momentum(5, 70, 50, 3)
    g[1] = 0
    g[2, 69, 49] = float("inf")
    g[3, 0, 0] = NAN
    got, held = run(g)
    assert not got[1].any() and got[2].isnan().all() and got[3].isnan().all()
    near(got[[0, 4]], reference(held[[0, 4]]), "bf16")


def test_steps():
    g = momentum(2, 60, 90, 4)
    got, held = run(g, steps=[(1, 0, 0)])
    near(got, reference(held, [(1, 0, 0)]), "bf16", 2.0 ** -20)
    other = [(1.5, -0.5, 0.0), (1.875, -1.25, 0.375)] * 3      # the products of Newton and of the next order
    got, held = run(g, steps=other)
    near(got, reference(held, other), "bf16")
    # enough of them: orthogonal rows, within the result's rounding and the f16 products
    got, held = run(g, "f32", "f16", steps=[(1.875, -1.25, 0.375)] * 12)
    eye = torch.eye(60, device=DEV, dtype=torch.float64)
    for x in got.double():
        assert (x @ x.t() - eye).abs().max() < 2.0 ** -7


def test_same_bits_whatever_lay_in_the_workspace_and_beside():
    g = momentum(3, 200, 333, 5)
    first, _ = run(g)
    again, _ = run(g)
    alone, _ = run(g[1:2])
    assert torch.equal(first, again) and torch.equal(first[1:2], alone)


def test_stream_and_graph():
    batch, rows, columns = 2, 160, 96
    g = momentum(batch, rows, columns, 6)
    want, _ = run(g)
    out = torch.zeros(batch, rows, columns, dtype=torch.bfloat16, device=DEV)
    work = torch.zeros(pf.orthogonalize_workspace(batch, rows, columns), dtype=torch.uint8, device=DEV)
    stream = torch.cuda.Stream()
    call = lambda: pf.orthogonalize(g, batch, rows, columns, out, work, stream=stream)  # noqa: E731
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call()
        for _ in range(4):
            out.fill_(3)
            work.fill_(0xff)
            graph.replay()
            stream.synchronize()
            assert torch.equal(out, want)
            out.fill_(3)
            call()
            stream.synchronize()
            assert torch.equal(out, want)


def test_past_32_bits_of_workspace():
    """40 matrices of 2048 x 4096: their first pieces alone are more than 2^29 elements."""
    batch, rows, columns = 40, 2048, 4096
    g = momentum(1, rows, columns, 7).bfloat16()
    out = torch.zeros(batch, rows, columns, dtype=torch.bfloat16, device=DEV)
    work = torch.empty(pf.orthogonalize_workspace(batch, rows, columns), dtype=torch.uint8, device=DEV)
    pf.orthogonalize(g.repeat(batch, 1, 1), batch, rows, columns, out, work, dtype="bf16")
    torch.cuda.synchronize()
    near(out[-1:], reference(g), "bf16")
    assert all(torch.equal(out[i], out[-1]) for i in range(batch))


@pytest.mark.parametrize("shift", [0, 1, 3, 8])
@pytest.mark.parametrize("batch,rows,columns,ld", [(1, 1, 1, 0), (1, 3, 1, 0), (2, 5, 1, 0), (1, 9, 2, 3), (1, 1, 9, 0), (1, 1, 23, 0), (2, 2, 7, 8), (3, 17, 5, 0),
                                                   (1, 100, 3, 4), (2, 70, 129, 0), (1, 129, 70, 71), (1, 700, 65, 0), (2, 65, 66, 72)])
def test_length(batch, rows, columns, ld, shift):
    """One step that changes nothing, of matrices at any address: G / |G|.  Its roundings: the factor and two pieces, under 2^-14."""
    for dtype, out in (("bf16", "f16"), ("f32", "bf16")):
        got, held = run(momentum(batch, rows, columns, 5), dtype, out, steps=[(1.0, 0.0, 0.0)], ld=ld, shift=shift, ld_out=ld, shift_out=shift)
        near(got, reference(held, [(1.0, 0.0, 0.0)]), out, slack=2.0 ** -14)


# tiles of 64 rows with four, two and one tile of k in a step, of 128 with eight and with four waves, of 256
@pytest.mark.parametrize("batch,rows,columns", [(1, 66, 1500), (1, 70, 96), (2, 1100, 1100), (3, 800, 833), (16, 500, 520), (9, 860, 1000), (1, 65, 65), (4, 2048, 2050)])
def test_tiles(batch, rows, columns):
    for flip in (False, True):
        g = momentum(batch, rows, columns, 7)
        got, held = run(g.transpose(1, 2).contiguous() if flip else g, "bf16")
        near(got, reference(held), "bf16")


@pytest.mark.parametrize("batch,rows,columns", [(5, 64, 661), (1, 64, 2048), (7, 33, 33), (2, 300, 50), (1, 2, 9)])
def test_up_to_64_rows_as_exact_as_the_type(batch, rows, columns):
    """Two pieces hold 2^-22 of a number; 9.4 such roundings a step (see above) and as many of sums in fp32 are under 2^-17, and
    of five steps, where small singular values may keep all that earlier ones left, under 2^-14."""
    got, held = run(momentum(batch, rows, columns, 8), out_dtype="f16")
    near(got, reference(held), "f16", slack=2.0 ** -13)
