"""What the decode model's pool of pages, shared reading and sampling refuse: CPU only, no kernel launches."""

from __future__ import annotations

import pytest
import torch

from scratch_llm_amd.decode import DecodeState
from scratch_llm_amd.sampling import Sampling
from tests.test_block_decode_cpu import model


def ints(*x):
    return torch.tensor(x, dtype=torch.int32)


def test_a_pool_belongs_to_blocks():
    for dtype in ("bf16", "fp8"):
        with pytest.raises(ValueError, match="kv_pages"):
            DecodeState(model(), 2, 64, dtype, kv_pages=8)
    for pages in (0, -1):
        with pytest.raises(ValueError, match="kv_pages"):
            DecodeState(model(), 2, 64, "int8_block", 16, kv_pages=pages)
    st = DecodeState(model(), 2, 64, "int8_block", 16, kv_pages=5)
    assert st.k.shape[:2] == (1, 5) and st.refs.tolist() == [0] * 5 and st.block_table.tolist() == [[-1] * 4] * 2 and st.room.tolist() == [1]


def test_pool_calls_need_a_pool():
    st = DecodeState(model(), 2, 64, "int8_block", 16)
    for call in (lambda: st.reserve(ints(1, 1)), lambda: st.free(ints(0, 0)), lambda: st.fork(ints(0, 0)), st.compact):
        with pytest.raises(ValueError, match="no pool"):
            call()
    with pytest.raises(ValueError, match="block-scaled"):
        DecodeState(model(), 2, 64, "bf16").share(ints(0, 0))


def test_pool_calls_refuse_a_table_of_another_type():
    st = DecodeState(model(), 2, 64, "int8_block", 16, kv_pages=5)
    for call in (lambda: st.reserve(ints(1, 1)), lambda: st.fork(ints(0, 0)), lambda: st.share(ints(0, 0)), st.compact):
        with pytest.raises(RuntimeError, match="device tensors"):
            call()
    assert st.shared is None and st.leaders is None
    st.block_table = st.block_table.long()
    for call in (lambda: st.reserve(ints(1, 1)), lambda: st.fork(ints(0, 0)), lambda: st.share(ints(0, 0)), st.compact):
        with pytest.raises(ValueError, match="block_table"):
            call()


def test_sampling_is_checked_when_it_is_set():
    st = DecodeState(model(), 2, 64)
    for bad, what in ((Sampling(temperature=-1.0), "temperature"), (Sampling(top_k=torch.ones(3, dtype=torch.int32)), "top_k"),
                      (Sampling(top_p=0.0), "top_p"), (Sampling(min_p=2.0), "min_p")):
        with pytest.raises(ValueError, match=what):
            st.set_sampling(bad)
        assert st.sampling is None
    with pytest.raises(RuntimeError, match="device tensors"):
        st.set_sampling(Sampling(temperature=torch.ones(2)))
    assert st.sampling is None
    st.set_sampling(Sampling(top_k=3))
    st.u = torch.zeros(3)
    with pytest.raises(ValueError, match="u must"):
        model().step(st)


@pytest.mark.parametrize("ok", [1, 0])
def test_tokens_of_a_fork(monkeypatch, ok):
    """A row takes its parent's next token; one that a parent outside the batch empties keeps its own, as do all where pages lack."""
    from scratch_llm_amd.quant import kv_pages

    monkeypatch.setattr(kv_pages, "fork_kv_rows", lambda *a: ints(ok))
    monkeypatch.setattr(DecodeState, "check_rows", lambda self, fn: None)
    st = DecodeState(model(), 5, 64, "int8_block", 16, kv_pages=5)
    st.tokens.copy_(ints(10, 11, 12, 13, 14))
    st.fork(ints(2, -1, 2, 5, 0))
    assert st.tokens.tolist() == ([12, 11, 12, 13, 10] if ok else [10, 11, 12, 13, 14])
    assert st.room.tolist() == [ok]
