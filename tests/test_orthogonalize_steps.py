"""Steps of orthogonal updates are triples, each of them (moe.py); CPU only."""
import pytest

import prefree_amd as pf
from test_moe_abi import INVALID, P, refused


def call(steps):
    pf.orthogonalize(P, 2, 30, 40, P, P, steps=steps, workspace_bytes=100)


@pytest.mark.parametrize("steps", [[(1, 2), (3, 4, 5, 6)], [(1, 2, 3, 4, 5, 6), ()], [()], [(1, 2)], [(1, 2, 3), (1, 2, 3, 4), (1, 2)]])
def test_each_is_a_triple(steps):
    with pytest.raises(ValueError):
        call(steps)


@pytest.mark.parametrize("steps", [[(1, 2, 3)] * 2, ((1.0, 2.0, 3.0),), [[1, 2, 3]]])
def test_triples_get_as_far_as_the_workspace(steps):
    refused(INVALID, call, steps)


def test_triples_one_after_the_other():
    refused(INVALID, call, ((1, 2, 3) for _ in range(2)))
