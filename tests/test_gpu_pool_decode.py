"""The decode model on a pool of pages, as a server draws several answers to a prompt: a chunk, a fork, shared reading, sampled steps,
drafts, cuts, a pool that is too small. Against the same model on pages of its own, bit for bit where the arithmetic is the same,
and against oracle/decode_ref.py where shared reading adds in another order."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import sample_ref as S
from tests.conftest import print_case
from tests.test_gpu_block_decode import CTX, FMT, BlockRefCache, check, ref_chunk, ref_steps, small  # noqa: F401

pytestmark = pytest.mark.gpu
DEV = "cuda"
BLOCK = 16


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def own_copies(model, st, rows):
    """A plain state whose rows hold what rows `rows` of `st` hold, on pages of their own."""
    to = model.new_state(len(rows), CTX, kv_dtype=st.kv_dtype, kv_block_size=BLOCK)
    for b, r in enumerate(rows):
        n = -(-int(st.lengths[r]) // BLOCK)
        src, dst = st.block_table[r, :n].long(), to.block_table[b, :n].long()
        for x, y in ((st.k, to.k), (st.v, to.v), (st.k_scale, to.k_scale), (st.v_scale, to.v_scale)):
            x, y = (t.view(torch.uint8) if t.element_size() == 1 else t for t in (x, y))
            y[:, dst] = x[:, src]
    to.lengths.copy_(st.lengths[rows])
    to.tokens.copy_(st.tokens[rows])
    return to


def prefilled(model, rows, n, kv_dtype, pages=64, seed=1):
    st = model.new_state(rows, CTX, kv_dtype=kv_dtype, kv_block_size=BLOCK, kv_pages=pages)
    prompt = torch.randint(0, 1000, (rows, n), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)
    logits = model.extend(st, prompt.to(DEV), i32([n] + [0] * (rows - 1)), last_only=True)
    assert st.lengths.tolist() == [n] + [0] * (rows - 1) and int(st.room) == 1
    st.tokens.copy_(logits.float().argmax(-1))
    return st, prompt


def books(st):
    table, refs = st.block_table.cpu().numpy(), st.refs.cpu().numpy()
    assert np.array_equal(refs, np.bincount(table[table >= 0].ravel(), minlength=len(refs)))


@pytest.mark.parametrize("kv_dtype", ["int8_block", "fp8_block"])
@pytest.mark.parametrize("n", [37, 48])
def test_forked_rows_decode_as_rows_of_their_own(small, kv_dtype, n):
    """A prompt in row 0, four answers: sampled steps over two blocks, then beams and more steps, equal to plain states."""
    from scratch_llm_amd.sampling import Sampling

    model, _ = small
    print_case("fork", kv_dtype, n)
    st, _ = prefilled(model, 4, n, kv_dtype)
    assert int(st.fork(i32([0, 0, 0, 0]))) == 1 and st.lengths.tolist() == [n] * 4
    books(st)
    plain = own_copies(model, st, [0, 1, 2, 3])
    settings = Sampling(temperature=1.5, top_k=50, top_p=0.95, min_p=0.01)
    g = torch.Generator().manual_seed(n)
    for s in (st, plain):
        s.set_sampling(settings)
    for step in range(24):
        if step == 14:  # beams: rows 0 and 2 go on twice
            assert int(st.fork(i32([0, 2, 2, 0]))) == 1
            books(st)
            plain = own_copies(model, plain, [0, 2, 2, 0])
            plain.set_sampling(settings)
        u = torch.rand(4, generator=g)
        for s in (st, plain):
            s.u.copy_(u)
            model.step(s)
        assert int(st.room) == 1
        assert torch.equal(st.logits, plain.logits) and torch.equal(st.tokens, plain.tokens) and torch.equal(st.lengths, plain.lengths)
        want = [S.sample(row, float(x), 1.5, 50, 0.95, 0.01) for row, x in zip(st.logits.float().cpu().numpy(), u)]
        assert st.tokens.tolist() == want
    assert len(set(st.tokens.tolist())) > 1  # the answers have parted
    books(st)
    before = int((st.refs > 0).sum())
    st.free(i32([n + 3, 0, 1 << 20, 16]))
    books(st)
    assert int((st.refs > 0).sum()) < before and st.lengths.tolist() == [n + 3, 0, n + 24, 16]
    assert int(st.compact()) == int((st.refs > 0).sum()) and int((st.refs > 0).nonzero().max()) == int((st.refs > 0).sum()) - 1
    books(st)
    kept = own_copies(model, st, [0, 1, 2, 3])
    st.set_sampling(None)
    for step in range(3):
        for s in (st, kept):
            s.tokens.copy_(i32([1, 2, 3, 4]) + step)
            model.step(s)
        assert torch.equal(st.logits, kept.logits)


@pytest.mark.parametrize("kv_dtype", ["int8_block", "fp8_block"])
@pytest.mark.parametrize("rows,n", [(3, 40), (5, 67)])
def test_shared_reading_matches_reference(small, kv_dtype, rows, n):
    model, refs = small
    print_case("shared reading", kv_dtype, rows, n)
    st, prompt = prefilled(model, rows, n, kv_dtype)
    st.fork(i32([0] * rows))
    st.share(i32([0] * rows))
    caches = {dt: BlockRefCache.make(r, rows, dt, FMT[kv_dtype], BLOCK) for dt, r in refs.items()}
    ref_chunk(refs, caches, prompt[:1].expand(rows, n), [n] * rows)
    g = torch.Generator().manual_seed(rows)
    for step in range(20):
        tok = torch.randint(0, 1000, (rows,), generator=g)
        model.step(st, tok)
        l16, l32 = ref_steps(refs, caches, tok[:, None])
        check(st.logits, l16[:, 0], l32[:, 0], f"step {step}")
    st.share(None)
    tok = torch.randint(0, 1000, (rows,), generator=g)
    model.step(st, tok)
    l16, l32 = ref_steps(refs, caches, tok[:, None])
    check(st.logits, l16[:, 0], l32[:, 0], "on their own again")


def test_a_cut_into_the_shared_part_is_planned_anew(small):
    """A row cut back into the shared pages goes on with a copy of the page it writes to; the others' stays."""
    model, _ = small
    st, _ = prefilled(model, 3, 60, "int8_block")
    st.fork(i32([0, 0, 0]))
    st.share(i32([0, 0, 0]))
    st.free(i32([1 << 20, 21, 1 << 20]))
    assert st.lengths.tolist() == [60, 21, 60]
    books(st)
    alone = own_copies(model, st, [0, 1, 2])
    for step in range(15):
        for s in (st, alone):
            s.tokens.copy_(i32([7, 8, 9]) + step)
            model.step(s)
        scale = float(alone.logits.float().abs().max())
        # the same numbers added in another order: attention outputs that may differ by a rounding, through two layers
        assert float((st.logits.float() - alone.logits.float()).abs().max()) <= 2.0**-5 * scale
        books(st)
    st.share(None)
    other = own_copies(model, st, [0, 1, 2])
    for s in (st, other):
        s.tokens.copy_(i32([1, 2, 3]))
        model.step(s)
    assert torch.equal(st.logits, other.logits)


def test_lengths_set_back_into_the_shared_part(small):
    """The row through which the group reads is cut and writes on: to a page of its own, which the others do not see."""
    model, _ = small
    st, _ = prefilled(model, 3, 70, "int8_block")
    st.fork(i32([0, 0, 0]))
    st.share(i32([0, 0, 0]))
    st.set_lengths([21, 70, 70])
    alone = own_copies(model, st, [0, 1, 2])
    for step in range(4):
        for s in (st, alone):
            s.tokens.copy_(i32([7, 8, 9]) + step)
            model.step(s)
        scale = float(alone.logits.float().abs().max())
        # as above
        assert float((st.logits.float() - alone.logits.float()).abs().max()) <= 2.0**-5 * scale
    assert st.block_table[0, 1] != st.block_table[1, 1] and torch.equal(st.block_table[1, :4], st.block_table[2, :4])


@pytest.mark.parametrize("kv_dtype", ["int8_block", "fp8_block"])
def test_a_pool_that_is_too_small_changes_nothing(small, kv_dtype):
    model, _ = small
    st, _ = prefilled(model, 3, 30, kv_dtype, pages=4)
    assert int(st.fork(i32([0, 0, 0]))) == 1  # one full page, three open ones: all four
    books(st)
    tokens = i32([3, 4, 5])
    for step in range(4):  # two tokens fit the open pages
        st.tokens.copy_(tokens)
        held = [x.clone() for x in (st.k.view(torch.uint8), st.v.view(torch.uint8), st.k_scale, st.v_scale, st.block_table, st.refs, st.lengths)]
        model.step(st)
        if step < 2:
            assert int(st.room) == 1 and st.lengths.tolist() == [31 + step] * 3
            continue
        assert int(st.room) == 0 and torch.equal(st.tokens, tokens)
        for x, y in zip(held, (st.k.view(torch.uint8), st.v.view(torch.uint8), st.k_scale, st.v_scale, st.block_table, st.refs, st.lengths)):
            assert torch.equal(x, y)
    assert int(st.fork(i32([2, 2, 1]))) == 1 and st.lengths.tolist() == [32, 32, 32]
    model.extend(st, torch.zeros(3, 2, dtype=torch.int32, device=DEV))
    assert int(st.room) == 0 and st.lengths.tolist() == [32] * 3
    st.tokens.copy_(tokens)
    model.verify(st, torch.zeros(3, 2, dtype=torch.int32, device=DEV), None, None, temperature=0.0)
    assert int(st.room) == 0 and st.lengths.tolist() == [32] * 3 and torch.equal(st.tokens, tokens)
    st.free(i32([100, 0, 0]))
    books(st)
    st.active.copy_(torch.tensor([1, 0, 0], dtype=torch.uint8))
    model.step(st)
    assert int(st.room) == 1 and st.lengths.tolist() == [33, 0, 0]


@pytest.mark.parametrize("kv_dtype", ["int8_block", "fp8_block"])
def test_drafts_on_a_pool_equal_drafts_on_own_pages(small, kv_dtype):
    model, _ = small
    st, _ = prefilled(model, 3, 41, kv_dtype)
    st.fork(i32([0, 0, 0]))
    plain = own_copies(model, st, [0, 1, 2])
    g = torch.Generator().manual_seed(5)
    for step in range(5):
        draft = torch.randint(0, 1000, (3, 6), generator=g, dtype=torch.int32)
        draft[0, 0] = int(st.logits[0].float().argmax()) if step else 0
        u, r = torch.rand(3, 6, generator=g), torch.rand(3, generator=g)
        got = [model.verify(s, draft.to(DEV), u.to(DEV), r.to(DEV), counts=i32([6, 3, 0])) for s in (st, plain)]
        for x, y in zip(*got):
            assert torch.equal(x, y)
        assert torch.equal(st.lengths, plain.lengths) and torch.equal(st.tokens, plain.tokens) and int(st.room) == 1
        books(st)
        for s in (st, plain):
            model.step(s)
        assert torch.equal(st.logits, plain.logits)


@pytest.mark.parametrize("n", [50, 110])
def test_captured_steps_take_pages_share_and_sample(small, n):
    """One captured step, replayed while rows are forked, cut and freed eagerly between the replays, equal to eager steps."""
    from scratch_llm_amd.sampling import Sampling

    model, _ = small
    states = []
    for _ in range(2):
        st, _ = prefilled(model, 4, n, "int8_block", pages=40)
        st.fork(i32([0, 0, 0, -1]))
        st.active.copy_(torch.tensor([1, 1, 1, 0], dtype=torch.uint8))
        st.share(i32([0, 0, 0, 0]))
        st.set_sampling(Sampling(temperature=torch.full((4,), 1.2, device=DEV), top_k=i32([40, 0, 5, 0]), top_p=0.9))
        states.append(st)
    a, b = states
    model.step(a)  # loads all code
    a, _ = prefilled(model, 4, n, "int8_block", pages=40)
    a.fork(i32([0, 0, 0, -1]))
    a.active.copy_(torch.tensor([1, 1, 1, 0], dtype=torch.uint8))
    a.share(i32([0, 0, 0, 0]))
    a.set_sampling(Sampling(temperature=torch.full((4,), 1.2, device=DEV), top_k=i32([40, 0, 5, 0]), top_p=0.9))
    graph = model.capture(a)
    g = torch.Generator().manual_seed(9)
    for step in range(30):
        u = torch.rand(4, generator=g)
        for s in (a, b):
            s.u.copy_(u)
            if step == 7:
                s.fork(i32([0, 0, 2, 2]))
                s.active.fill_(1)
            if step == 13:
                s.free(i32([1 << 20, 30, 1 << 20, 0]))
                s.active.copy_(torch.tensor([1, 1, 1, 0], dtype=torch.uint8))
            if step == 19:
                s.compact()
        graph.replay()
        model.step(b)
        torch.cuda.synchronize()
        for x, y in ((a.logits[:3], b.logits[:3]), (a.tokens[:3], b.tokens[:3]), (a.lengths, b.lengths), (a.block_table, b.block_table), (a.refs, b.refs)):
            assert torch.equal(x, y), step
        assert int(a.room) == int(b.room) == 1
        books(a)


def test_sampled_steps_of_every_cache_and_rows_without_a_distribution(small):
    """Sampling needs no pool; a row whose logits are NaN keeps its token and stays."""
    from scratch_llm_amd.sampling import Sampling

    model, _ = small
    for kv_dtype in ("bf16", "fp8", "int8_block"):
        st = model.new_state(3, CTX, kv_dtype=kv_dtype)
        st.set_sampling(Sampling(temperature=0.9, top_p=0.8))
        g = torch.Generator().manual_seed(2)
        for step in range(4):
            u = torch.rand(3, generator=g)
            st.u.copy_(u)
            model.step(st)
            assert st.tokens.tolist() == [S.sample(x, float(y), 0.9, 0, 0.8) for x, y in zip(st.logits.float().cpu().numpy(), u)]
        st.set_sampling(None)
        model.step(st)
        assert torch.equal(st.tokens.long(), st.logits.float().argmax(-1)) and st.lengths.tolist() == [5] * 3
    st.set_sampling(Sampling())
    st.block_table[1, 0] = 1 << 20  # names no page: whoever attends it gets NaN
    before = st.tokens.clone()
    model.step(st)
    assert bool(st.logits[1].isnan().any()) and int(st.tokens[1]) == int(before[1]) and st.lengths.tolist() == [6, 5, 6]


def test_an_emptied_row_keeps_its_token(small):
    model, _ = small
    st, _ = prefilled(model, 4, 37, "int8_block")
    st.tokens.copy_(i32([10, 11, 12, 13]))
    assert int(st.fork(i32([0, -1, 0, 4]))) == 1
    assert st.lengths.tolist() == [37, 0, 37, 0] and st.tokens.tolist() == [10, 11, 10, 13]
    books(st)
