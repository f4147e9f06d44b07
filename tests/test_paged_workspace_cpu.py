"""What the workspace query of paged_attn answers, without a GPU."""

import pytest

from q4llm import ops


@pytest.mark.parametrize("L,shared", [(100, 0), (4000, 0), (4000, 2000), (512, 512), (1 << 30, 1 << 29)])
@pytest.mark.parametrize("batch", [1, 4, 1000])
def test_no_tokens_need_none(batch, L, shared):
    """(A prefix with ranges of its own divided by the number of tiles, which ended the process.)"""
    assert ops.paged_attn_workspace_bytes(0, 8, 2, 64, batch, L, shared) == 0


@pytest.mark.parametrize("T,n_q,n_kv,hd,batch,L,shared,most", [
    (64, 24, 8, 128, 64, 1000, 0, 0), (4, 8, 2, 64, 4, 100, 0, 0),        # one range a row, which writes the result itself
    (256, 32, 8, 128, 256, 8192, 2048, 40 << 20), (32, 32, 8, 128, 32, 2560, 2048, 20 << 20), (1, 24, 8, 128, 1, 700, 0, 1 << 20)])
def test_calls_without_cu_q_need_what_their_own_plan_does(T, n_q, n_kv, hd, batch, L, shared, most):
    even, ragged, both = (ops.paged_attn_workspace_bytes(T, n_q, n_kv, hd, batch, L, shared, r) for r in (False, True, None))
    assert even <= most and both == max(even, ragged) and (both > 0 or L == 100)  # (100 keys: one range with cu_q too)


def test_the_query_for_one_form_refuses_what_the_call_would():
    for bad in (dict(T=7), dict(n_kv=3), dict(L=0), dict(shared=101), dict(batch=0)):
        a = {**dict(T=4, n_q=8, n_kv=2, hd=64, batch=4, L=100, shared=0), **bad}
        with pytest.raises(Exception):
            ops.paged_attn_workspace_bytes(*a.values(), False)
    assert ops.paged_attn_workspace_bytes(7, 8, 2, 64, 4, 4000, 0, True) > 0  # 7 tokens of 4 sequences: with cu_q


def test_slots_with_cu_q_are_those_that_ranges_can_fill():
    """32 single tokens behind 2048 shared keys (8 KV heads of 128 dims): 264 tiles at most, which 256 places take one by one; a slot has
    128 rows, as the 128 of the batch may be one sequence's, and a row 130 floats; beside them the shared ranges' rows."""
    even, ragged = (ops.paged_attn_workspace_bytes(32, 32, 8, 128, 32, 2560, 2048, r) for r in (False, True))
    rows = 32 * 32
    assert ragged <= 264 * 128 * 130 * 4 + 32 * rows * 130 * 4 + rows * 8 + 64
