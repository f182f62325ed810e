"""A captured step outlives what it was captured with: after ``share(None)`` it reads every row for itself, after another
``set_sampling`` it draws with the settings that it has, and their memory is nobody else's. Equal to eager steps bit for bit."""

from __future__ import annotations

import gc
import weakref

import pytest
import torch

from tests.test_gpu_block_decode import small  # noqa: F401
from tests.test_gpu_pool_decode import DEV, books, i32, prefilled

pytestmark = pytest.mark.gpu
ROWS, N = 4, 110


def state(model):
    st, _ = prefilled(model, ROWS, N, "int8_block", pages=40)
    st.fork(i32([0] * ROWS))
    st.share(i32([0] * ROWS))
    set_sampling(st)
    return st


def set_sampling(st):
    from scratch_llm_amd.sampling import Sampling

    st.set_sampling(Sampling(temperature=torch.full((ROWS,), 1.2, device=DEV), top_k=i32([40, 0, 5, 300]),
                             top_p=torch.full((ROWS,), 0.9, device=DEV)))


def test_a_replay_after_the_state_went_on_to_something_else(small):
    model, _ = small
    model.step(state(model))  # loads all code
    a, b = state(model), state(model)
    graph = model.capture(a)
    g = torch.Generator().manual_seed(3)

    def steps(n, what):
        for step in range(n):
            u = torch.rand(ROWS, generator=g)
            for s in (a, b):
                s.u.copy_(u)
            graph.replay()
            model.step(b)
            torch.cuda.synchronize()
            for x, y in ((a.logits, b.logits), (a.tokens, b.tokens), (a.lengths, b.lengths), (a.block_table, b.block_table), (a.refs, b.refs)):
                assert torch.equal(x, y), (what, step)
            books(a)

    steps(3, "shared")
    settings = [weakref.ref(x) for x in a.sampling.tensors() if x is not None]
    assert len(settings) == 3
    plan = a.shared.plan.data_ptr()
    a.share(None)
    a.set_sampling(None)
    gc.collect()
    assert all(x() is not None for x in settings)
    # memory of the sizes that were let go, if any was, is written over
    others = [torch.full((n,), 0x7F, dtype=torch.uint8, device=DEV) for n in (16, 512, a.plans[a.block_table.shape[1]].plan.numel()) for _ in range(16)]
    held = {x().data_ptr() for x in settings} | {plan}
    assert not held & {x.data_ptr() for x in others}
    b.share(i32([-1] * ROWS))
    steps(3, "every row for itself")
    for s in (a, b):
        s.share(i32([2, 2, 1, 1]))
    steps(3, "in other groups")
    for s in (a, b):
        assert int(s.fork(i32([1, 1, 1, 2]))) == 1
        s.free(i32([1 << 20, 70, 1 << 20, 1 << 20]))
    steps(3, "forked and cut")
    # a step captured anew has what the state has now: greedy picks
    again = model.capture(a)
    b.set_sampling(None)
    for _ in range(3):
        again.replay()
        model.step(b)
        torch.cuda.synchronize()
        assert torch.equal(a.logits, b.logits) and torch.equal(a.tokens, b.tokens)


def test_a_graph_keeps_its_state(small):
    """The state and its tensors live as long as the graph does."""
    model, _ = small
    st = state(model)
    model.step(st)
    graph = model.capture(st)
    alive = [weakref.ref(x) for x in (st.k, st.block_table, st.lengths, st.u, st.shared.plan, st.sampling.top_k)]
    logits = st.logits
    st.u = torch.rand(ROWS, device=DEV)
    st.lengths = st.lengths.clone()
    del st
    gc.collect()
    assert all(x() is not None for x in alive)
    graph.replay()
    torch.cuda.synchronize()
    assert bool(logits.isfinite().all()) and alive[2]().tolist() == [N + 2] * ROWS
    del graph
    gc.collect()
    assert all(x() is None for x in alive)
