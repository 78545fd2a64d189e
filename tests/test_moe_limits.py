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


def test_arrays_of_words_that_do_not_lie_on_words_are_refused():
    """choice, weight, offsets, order, slot, rows and dweight hold 32-bit numbers.  (No call here is launched.)"""
    P = 4096
    odd = P + 2

    def each(call, names):
        for name in names:
            with pytest.raises(pf.PrefreeError) as e:
                call(**{name: odd})
            assert e.value.status == 2, name        # PF_ERR_ALIGN

    each(lambda choice=P, weight=P, offsets=P, order=P, slot=P: pf.moe_route(
        P, 100, 8, 2, choice, weight, offsets, order, slot, P, workspace_bytes=1 << 20), ("choice", "weight", "offsets", "order", "slot"))
    each(lambda choice=P, weight=P, dweight=P: pf.moe_route_backward(P, 4, 8, 2, choice, weight, dweight, P), ("choice", "weight", "dweight"))
    each(lambda slot=P, weight=P: pf.moe_combine(P, slot, weight, 4, 2, 64, P), ("slot", "weight"))
    each(lambda slot=P, weight=P, dweight=P: pf.moe_combine_backward(P, P, slot, weight, 4, 2, 64, P, dweight), ("slot", "weight", "dweight"))
    each(lambda rows=P, offsets=P: pf.moe_mm(P, 10, rows, 1, P, offsets, 4, 10, 64, 64, P), ("rows", "offsets"))
    each(lambda offsets=P: pf.moe_mm_dx(P, P, offsets, 4, 10, 64, 64, P), ("offsets",))
    each(lambda rows=P, offsets=P: pf.moe_mm_dw(P, P, 10, rows, 1, offsets, 4, 10, 64, 64, P), ("rows", "offsets"))
    each(lambda rows=P, offsets=P: pf.moe_mm_mx4(P, P, 10, rows, 1, P, P, offsets, 4, 10, 64, 64, P), ("rows", "offsets"))
