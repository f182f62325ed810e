"""The decode state keeps what a captured step reads by its address: the plan of shared prefixes is written over, never let go. CPU
only: the calls that would launch are recorded instead."""

from __future__ import annotations

import pytest
import torch

from scratch_llm_amd.decode import DecodeState
from scratch_llm_amd.quant import kv_shared
from tests.test_block_decode_cpu import model


def ints(*x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.fixture
def shared(monkeypatch):
    """A state of two rows that share, and the leaders of every plan that was made, by plan."""
    made = []

    def plan(table, starts, leaders, *, block, tokens, heads, kv_heads, head_dim, out=None):
        assert table.dtype == leaders.dtype == torch.int32 and table.is_contiguous() and leaders.is_contiguous()
        sizes = (table.shape[0], tokens, heads, kv_heads, head_dim, block, table.shape[1])
        if out is None:
            out = kv_shared.SharedKV(torch.empty(16, dtype=torch.uint8), *sizes)
        assert (out.batch, out.tokens, out.heads, out.kv_heads, out.head_dim, out.block, out.width) == sizes
        made.append((out, leaders.tolist()))
        return out

    monkeypatch.setattr(kv_shared, "plan_shared_kv", plan)
    monkeypatch.setattr(DecodeState, "check_rows", lambda self, fn: None)
    st = DecodeState(model(), 2, 64, "int8_block", 16, kv_pages=5)
    st.share(ints(0, 0))
    return st, made


def test_a_plan_is_kept_and_taken_up_again(shared):
    st, made = shared
    first = st.shared
    assert made == [(first, [0, 0])]
    st.share(None)  # a step captured before goes on with every row for itself
    assert st.shared is None and st.leaders is None
    assert made[1][0] is first and made[1][1] == [-1, -1]
    st.share(None)
    assert len(made) == 2
    st.share(ints(1, 1))
    assert st.shared is first and made[2] == (first, [1, 1])
    st.set_lengths([3, 4])
    assert st.shared is first and made[3] == (first, [1, 1])


def test_a_table_of_another_width(shared):
    """The plan of the width before stays where it is, with every row for itself, and serves again."""
    st, made = shared
    first, table = st.shared, st.block_table
    st.block_table = torch.full((2, 7), -1, dtype=torch.int32)
    st.set_lengths([3, 4])
    assert st.shared is not first and st.shared.width == 7
    assert made[1][0] is first and made[1][1] == [-1, -1] and made[2] == (st.shared, [0, 0])
    second = st.shared
    st.block_table = table
    st.share(ints(0, 0))
    assert st.shared is first and made[3][0] is second and made[3][1] == [-1, -1] and made[4] == (first, [0, 0])
