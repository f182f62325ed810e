"""What the decode model refuses of a block-scaled state before anything reaches the GPU: CPU only."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from scratch_llm_amd.decode import DecodeConfig, DecodeState, Int4DecodeLM

CFG = DecodeConfig(vocab_size=64, d_model=256, n_layers=1, n_heads=2, n_kv_heads=1, d_ff=256, context_length=64)


def model():
    """As much of a model as a state and the checks of its calls read."""
    m = Int4DecodeLM.__new__(Int4DecodeLM)
    m.cfg, m.device, m.embed, m.layers = CFG, torch.device("cpu"), torch.zeros(64, 256, dtype=torch.bfloat16), []
    m.lm_head = SimpleNamespace(rows=64, cols=256)
    return m


def state(batch=2, block=16):
    return DecodeState(model(), batch, 64, "int8_block", block)


@pytest.mark.parametrize("block", [0, 48, -16, 256])
def test_block_sizes(block):
    with pytest.raises(ValueError, match="block must be one of"):
        state(block=block)


TABLES = {
    "int64": lambda t: t.long(), "fewer rows": lambda t: t[:1], "more rows": lambda t: torch.cat((t, t)), "one row": lambda t: t[0],
    "no blocks": lambda t: t[:, :0], "transposed": lambda t: t.t().contiguous().t(), "every other": lambda t: t[:, ::2],
}


@pytest.mark.parametrize("name", TABLES)
def test_a_table_that_is_none_is_refused(name):
    """The kernels read int32 [B, width], rows one after the other: another type would name other pages, fewer rows end before
    the last one's are read."""
    m, st = model(), state()
    st.block_table = TABLES[name](st.block_table)
    ids = torch.zeros(2, 3, dtype=torch.int32)
    for call in (lambda: m.step(st), lambda: m.extend(st, ids), lambda: m.verify(st, ids, None, None, temperature=0.0)):
        with pytest.raises(ValueError, match="block_table"):
            call()


def test_rows_of_another_type_are_refused():
    m, ids = model(), torch.zeros(2, 3, dtype=torch.int32)
    for bad in (torch.zeros(2, dtype=torch.int64), torch.zeros(1, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)[::2]):
        st = state()
        st.lengths = bad
        for call in (lambda: m.step(st), lambda: m.extend(st, ids)):
            with pytest.raises(ValueError, match="lengths"):
                call()


def test_tables_that_stay_allowed():
    """A server's own table, of any width, gets past the check (and is stopped by the CPU tensors)."""
    m, ids = model(), torch.zeros(2, 3, dtype=torch.int32)
    for width in (1, 4, 9):
        st = state()
        st.block_table = torch.zeros(2, width, dtype=torch.int32)
        for call in (lambda: m.step(st), lambda: m.extend(st, ids)):
            with pytest.raises(RuntimeError, match="device tensors"):
                call()
