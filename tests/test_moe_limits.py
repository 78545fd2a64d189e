"""Sizes at the ends of what the expert-layer operators (include/prefree_moe.h) take — CPU only."""
import pytest

import prefree_amd as pf

BLOCK, DIRECT, SUPER = 64, 1024, 64   # tokens a block of the routing; blocks without sums beforehand; blocks a sum


def routing_layout(tokens, experts):
    """Bytes that routing writes: a byte an expert and block, in rows of whole words, and above DIRECT blocks a word an
    expert and SUPER whole blocks."""
    blocks = -(-tokens // BLOCK)
    return blocks * 4 * -(-experts // 4) + (blocks // SUPER * 4 * experts if blocks > DIRECT else 0)


@pytest.mark.parametrize("tokens", [65, 128, 65472, 65473, 65536, 65537, 65600, 69632, 69633, 1 << 20, (1 << 24) + 1, 1 << 30])
def test_routing_workspace_holds_what_routing_writes(tokens):
    short = [e for e in range(1, 1025) if pf.moe_route_workspace(tokens, e) < routing_layout(tokens, e)]
    assert not short, short


@pytest.mark.parametrize("tokens", [65, 5000, 65536, 65537, 1 << 20])
def test_routing_workspace_stays_as_it_was_for_two_experts_and_more(tokens):
    for experts in (2, 3, 4, 5, 8, 33, 128, 1024):
        assert pf.moe_route_workspace(tokens, experts) == 4 * experts * -(-tokens // BLOCK)


def test_a_workspace_on_the_host_is_refused_in_python():
    torch = pytest.importorskip("torch")
    P = 4096   # a pointer that is never followed
    for dtype in (torch.uint8, torch.int32):
        work = torch.zeros(1 << 20, dtype=dtype)
        with pytest.raises(TypeError):
            pf.moe_route(P, 100, 8, 2, P, P, P, P, P, work)
        with pytest.raises(TypeError):
            pf.moe_route(P, 100, 8, 2, P, P, P, P, P, work, workspace_bytes=1 << 20)
