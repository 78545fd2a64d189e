"""Orthogonal updates (include/prefree_moe.h) — CPU only: refusals before any launch, the workspace's size."""
import pytest

import prefree_amd as pf
from test_moe_abi import ALIGN, INVALID, P, refused


def call(g=P, batch=2, rows=30, columns=40, out=P, work=P, dtype="f32", out_dtype="bf16", steps=pf.ORTHOGONAL_STEPS, work_bytes=1 << 20, **ld):
    pf.orthogonalize(g, batch, rows, columns, out, work, dtype=dtype, out_dtype=out_dtype, steps=steps, workspace_bytes=work_bytes, **ld)


@pytest.mark.parametrize("kw", [{"g": None}, {"out": None}, {"work": None}, {"batch": -1}, {"batch": 1025}, {"rows": -1}, {"columns": -1},
                                {"rows": (1 << 20) + 1}, {"columns": (1 << 20) + 1}, {"rows": 1 << 15, "columns": 1 << 15}, {"dtype": "f64"},
                                {"out_dtype": "f32"}, {"steps": ()}, {"steps": [(1, 2, 3)] * 65}, {"work_bytes": 100}, {"ld_g": 39},
                                {"ld_out": 39}, {"ld_g": -1}])
def test_refusals(kw):
    refused(INVALID, call, **kw)


def test_alignment_types_and_nothing_to_do():
    for kw in ({"g": P + 2}, {"g": P + 1, "dtype": "bf16"}, {"out": P + 1}, {"work": P + 8}):
        refused(ALIGN, call, **kw)
    with pytest.raises(ValueError):
        call(steps=[(1, 2)])
    torch = pytest.importorskip("torch")
    with pytest.raises(TypeError):
        call(g=torch.zeros(2, 30, 40))                 # not on the GPU
    with pytest.raises(TypeError):
        call(out=torch.zeros(2, 30, 40))
    for kw in ({"batch": 0}, {"rows": 0}, {"columns": 0}):
        call(**kw)


@pytest.mark.parametrize("batch,rows,columns", [(1, 1, 1), (3, 33, 7), (2, 64, 2048), (1, 300, 200)])
def test_workspace(batch, rows, columns):
    need = pf.orthogonalize_workspace(batch, rows, columns)
    assert need == pf.orthogonalize_workspace(batch, columns, rows)
    refused(INVALID, call, batch=batch, rows=rows, columns=columns, work_bytes=need - 1)
    assert pf.orthogonalize_workspace(0, 5, 5) == pf.orthogonalize_workspace(2, 0, 5) == 0
    # it may be relied on: no more than 16 bytes an element of matrices padded to multiples of 64, and 64 MiB
    up = lambda v: (v + 63) // 64 * 64  # noqa: E731
    assert need <= 16 * batch * up(rows) * up(columns) + (1 << 26)
