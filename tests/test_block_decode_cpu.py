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


def test_a_pass_that_a_linear_cannot_take_is_refused():
    """Rows of 256 columns of bf16 below 2 GiB: 2^22 - 1 of them. More are refused before anything is written."""
    m, st = model(), state()
    assert CFG.d_model == CFG.d_ff == 256
    m._check_pass(2, (1 << 21) - 1, "f")
    for t in (1 << 21, 1 << 23):
        with pytest.raises(ValueError, match="smaller chunks"):
            m.extend(st, torch.zeros(1, dtype=torch.int32).expand(2, t))
    one = state(batch=1)
    m._check_pass(1, (1 << 22) - 1, "f")
    with pytest.raises(ValueError, match="smaller chunks"):
        m.extend(one, torch.zeros(1, dtype=torch.int32).expand(1, 1 << 22))


def test_open_blocks_refuse():
    """Every check of sqx_kvblock_open, before anything reaches the GPU (a non-null pointer is never followed)."""
    import ctypes

    from scratch_llm_amd import _lib

    lib, p = _lib.load(), ctypes.c_void_p(256)

    def call(**c):
        a = dict(kc=p, vc=p, ks=p, table=p, starts=p, L=2, B=3, Hkv=1, hd=64, block=16, pages=4, width=2, saved=p, nb=1 << 20)
        a.update(c)
        return lib.sqx_kvblock_open(0, a["kc"], a["vc"], a["ks"], p, a["table"], a["starts"], None, a["L"], a["B"], a["Hkv"], a["hd"],
                                    a["block"], a["pages"], a["width"], a["saved"], a["nb"], None)

    for bad in (dict(L=-1), dict(L=1 << 16), dict(B=1 << 16), dict(Hkv=0), dict(hd=96), dict(block=48), dict(pages=0), dict(width=0),
                dict(kc=None), dict(ks=None), dict(table=None), dict(starts=None), dict(saved=None), dict(vc=ctypes.c_void_p(8)),
                dict(saved=ctypes.c_void_p(24))):
        assert call(**bad) == -1, bad
        assert b"sqx_kvblock_open" in lib.sqx_last_error()
    assert lib.sqx_kvblock_open_bytes(2, 3, 1, 64, 16) == 2 * 3 * 2 * (16 * 64 + 4)
    assert call(nb=2 * 3 * 2 * (16 * 64 + 4) - 1) == -3
    assert call(L=0) == 0 and call(B=0) == 0
    for none in ((0, 3, 1, 64, 16), (2, 3, 1, 80, 16), (2, 3, 1, 64, 20), (2, 0, 1, 64, 16)):
        assert lib.sqx_kvblock_open_bytes(*none) == 0
