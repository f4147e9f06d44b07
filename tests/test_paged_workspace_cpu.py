"""What the workspace query of paged_attn answers, without a GPU."""

import pytest

from q4llm import ops


@pytest.mark.parametrize("L,shared", [(100, 0), (4000, 0), (4000, 2000), (512, 512), (1 << 30, 1 << 29)])
@pytest.mark.parametrize("batch", [1, 4, 1000])
def test_no_tokens_need_none(batch, L, shared):
    """(A prefix with ranges of its own divided by the number of tiles, which ended the process.)"""
    assert ops.paged_attn_workspace_bytes(0, 8, 2, 64, batch, L, shared) == 0
