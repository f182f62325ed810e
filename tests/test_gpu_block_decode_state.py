"""What the decode model's passes over several tokens a row leave of a state on the block-scaled cache."""

from __future__ import annotations

import pytest
import torch

from oracle import decode_ref as D
from tests.conftest import print_case

pytestmark = pytest.mark.gpu
DEV = "cuda"
SMALL = dict(vocab=512, d_model=512, n_layers=2, n_heads=4, n_kv_heads=2, d_ff=1024)
CTX = 96
LOUD, NAN = 500, 501  # a token whose keys and values are many times the others', and one that has none
KV = ["int8_block", "fp8_block"]


def build(p):
    from scratch_llm_amd.decode import DecodeConfig, Int4DecodeLM

    cfg = DecodeConfig(vocab_size=SMALL["vocab"], d_model=SMALL["d_model"], n_layers=SMALL["n_layers"], n_heads=SMALL["n_heads"],
                       n_kv_heads=SMALL["n_kv_heads"], d_ff=SMALL["d_ff"], context_length=CTX)
    return Int4DecodeLM.from_state_dict(cfg, lambda n: p[n], DEV)


@pytest.fixture(scope="module")
def model():
    """Layer 0's keys and values depend on the embeddings alone, so its cache can be compared bit for bit. LOUD's embedding
    points along one key row and one value row of each kv head."""
    p = D.random_params(**SMALL, seed=21, std=0.05)
    k, v = p["blocks.0.attn.k_proj.weight"], p["blocks.0.attn.v_proj.weight"]
    e = sum(x / x.norm() for w in (k, v) for x in (w[5], w[128 + 9]))
    p["token_emb.weight"][LOUD] = e * (SMALL["d_model"] ** 0.5 / e.norm())
    p["token_emb.weight"][NAN] = float("nan")
    return build(p)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def ids(shape, seed):
    return torch.randint(0, LOUD, shape, generator=torch.Generator().manual_seed(seed), dtype=torch.int32).to(DEV)


def raw(st):
    return [x.view(torch.uint8).clone() if x.element_size() == 1 else x.clone() for x in (st.k, st.v, st.k_scale, st.v_scale)]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def layer0(st, row, n):
    """Values of a row's first n positions in layer 0, and the scales of their blocks."""
    from scratch_llm_amd.quant import kv_block

    block = st.k.shape[3]
    k, v = kv_block.read_kv_blocks(*st.kv_layer(0), st.block_table[row:row + 1], i32([0]), n)
    page = st.block_table[row, :-(-n // block)].long()
    return k, v, st.k_scale[0, page], st.v_scale[0, page]


# prompt lengths (blocks of 16), drafts that are kept, drafts a row has
ROWS = [(10, 7, 8),   # kept tokens reach into a block that the pass begins; the loud rejected one lies behind them in it
        (13, 8, 8),   # all kept, the loud one too
        (10, 3, 8),   # not active; its table names row 0's pages
        (16, 0, 8),   # at a block's first slot: nothing older is in the block
        (9, 2, 8),    # the loud rejected one lies in the block that holds older tokens
        (7, 0, 5),    # the same, nothing kept but the current token
        (12, 1, 1),   # one draft, kept
        (15, 0, 0)]   # none


def test_any_flag_but_zero_is_active(model):
    """`active` is read as the step's `advance` reads it: a row is active where its flag is not zero."""
    B = 2
    one, two = (model.new_state(B, CTX, kv_dtype="int8_block") for _ in range(2))
    two.active.copy_(torch.tensor([2, 255], dtype=torch.uint8))
    prompt, draft = ids((B, 9), 9), ids((B, 3), 10)
    u, r = torch.full((B, 3), 0.5, device=DEV), torch.full((B,), 0.5, device=DEV)
    for s in (one, two):
        model.extend(s, prompt, i32([9, 4]))
        s.tokens.copy_(i32([1, 2]))
        model.step(s)
        model.verify(s, draft, u, r)
    assert torch.equal(one.lengths, two.lengths) and torch.equal(one.tokens, two.tokens)
    assert torch.equal(one.k, two.k) and torch.equal(one.v_scale, two.v_scale)


def test_a_refused_verification_changes_nothing(model):
    """Every argument that the verification refuses is refused before the pass writes into the cache."""
    B, T = 2, 3
    st = model.new_state(B, CTX, kv_dtype="int8_block")
    model.extend(st, ids((B, 9), 11))
    st.tokens.copy_(i32([1, 2]))
    draft, u, r = ids((B, T), 12), torch.rand(B, T, device=DEV), torch.rand(B, device=DEV)
    probs = torch.full((B, T, SMALL["vocab"]), 1.0 / SMALL["vocab"], device=DEV)
    held = raw(st) + [st.lengths.clone(), st.tokens.clone()]
    for change in (dict(temperature=-1.0), dict(u=None), dict(r=None), dict(u=u.double()), dict(u=u[:, :2]), dict(r=r[:1]),
                   dict(draft_probs=probs[:, :2]), dict(draft_probs=probs.double()), dict(counts=i32([1])),
                   dict(counts=torch.ones(B, device=DEV)), dict(u=u.cpu()), dict(draft_probs=probs.cpu()), dict(draft=draft.cpu())):
        a = {**dict(draft=draft, u=u, r=r), **change}
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            model.verify(st, a.pop("draft"), a.pop("u"), a.pop("r"), **a)
        torch.cuda.synchronize()
        assert same(raw(st) + [st.lengths, st.tokens], held), f"{list(change)}: the state has changed"


@pytest.mark.parametrize("temperature", [0.9, 1.0])
def test_a_row_without_a_next_token_stays_before_it(model, temperature):
    """Behind a token of NaN every row of logits is no distribution: there is no next token (-1), the row's state stays at the
    last kept token, which the next pass scores anew, and the other rows go on."""
    B, T = 3, 3
    st = model.new_state(B, CTX, kv_dtype="int8_block", kv_block_size=16)
    model.extend(st, ids((B, 12), 7))
    st.tokens.copy_(i32([5, NAN, 6]))
    draft = ids((B, T), 8)
    draft[0, 1] = NAN
    n, tok = model.verify(st, draft, torch.zeros(B, T, device=DEV), torch.full((B,), 0.5, device=DEV), temperature=temperature)
    assert n.tolist() == [2, 0, 3]
    assert tok[0].tolist() == [int(draft[0, 0]), NAN, -1, -1] and tok[1].tolist() == [-1] * 4
    assert st.lengths.tolist() == [14, 12, 16]
    assert st.tokens.tolist() == [NAN, NAN, int(tok[2, 3])] and int(st.tokens[2]) >= 0


@pytest.mark.parametrize("hkv,d,block", [(1, 64, 16), (3, 64, 32), (2, 256, 16), (8, 128, 64), (5, 128, 128)])
def test_open_blocks_are_put_back(hkv, d, block):
    """What sqx_kvblock_open saves of three layers it puts back whole, for the rows that are asked for and are in the middle of
    a block on a page, and nothing else."""
    from scratch_llm_amd import _lib

    print_case("open blocks", hkv, d, block)
    L, pages, width = 3, 9, 2
    starts = [1, block - 1, block, 0, block + 3, 2 * block - 1, 2 * block + 1, -5, 3, 7]
    rows = [1, 1, 1, 1, 5, 1, 1, 1, 0, 1]
    B = len(starts)
    table = torch.tensor([[0, 1], [2, 1], [1, 3], [3, 1], [1, 4], [1, 5], [6, 6], [6, 6], [7, 1], [9, 1]], dtype=torch.int32)
    open_pages = [0, 2, 4, 5]
    g = torch.Generator().manual_seed(block + d)
    codes = [torch.randint(0, 256, (L, pages, hkv, block * d), generator=g, dtype=torch.uint8).to(DEV) for _ in range(2)]
    scales = [torch.rand(L, pages, hkv, generator=g).to(DEV) for _ in range(2)]
    held = [x.clone() for x in codes + scales]
    lib = _lib.load()
    nb = lib.sqx_kvblock_open_bytes(L, B, hkv, d, block)
    saved = torch.zeros(nb + 64, dtype=torch.uint8, device=DEV)
    table, st, rw = table.to(DEV), i32(starts), i32(rows)

    def go(back):
        _lib.check(lib.sqx_kvblock_open(back, *(x.data_ptr() for x in codes + scales), table.data_ptr(), st.data_ptr(), rw.data_ptr(), L,
                                        B, hkv, d, block, pages, width, saved.data_ptr(), nb,
                                        torch.cuda.current_stream().cuda_stream), "open")

    go(0)
    assert all(torch.equal(x, y) for x, y in zip(codes + scales, held)) and int(saved[nb:].max()) == 0
    other = [torch.randint(0, 256, x.shape, generator=g, dtype=torch.uint8).to(DEV) for x in codes]
    other += [torch.rand(x.shape, generator=g).to(DEV) for x in scales]
    for x, y in zip(codes + scales, other):
        x.copy_(y)
    go(1)
    torch.cuda.synchronize()
    for x, y, z in zip(codes + scales, held, other):
        want = z.clone()
        want[:, open_pages] = y[:, open_pages]
        assert torch.equal(x, want)


@pytest.mark.parametrize("replay", [False, True])
@pytest.mark.parametrize("kv_dtype", KV)
def test_rejected_drafts_leave_no_trace(model, kv_dtype, replay):
    """After a verification the cache's first layer is, bit for bit, that of a pass over the kept tokens alone: neither the
    older tokens' codes nor the scales nor the kept tokens' codes show what a rejected draft of many times their size did
    to their blocks in between. Eager and as the second replay of a graph."""
    print_case("verify leaves no trace", kv_dtype, replay)
    B, T = len(ROWS), 8
    start, kept, count = (list(x) for x in zip(*ROWS))
    prompt = ids((B, 16), 1)
    st, ref = (model.new_state(B, CTX, kv_dtype=kv_dtype, kv_block_size=16) for _ in range(2))
    draft = ids((B, T), 2)
    for b in range(B):
        draft[b, min(kept[b], T - 1)] = LOUD
    u = torch.full((B, T), 0.9999, device=DEV)
    for b in range(B):
        u[b, :kept[b]] = 0.0
    r, counts = torch.full((B,), 0.3, device=DEV), i32(count)

    def fill(s):
        s.lengths.zero_()
        s.active.fill_(1)
        s.block_table.copy_(torch.arange(s.block_table.numel(), dtype=torch.int32, device=DEV).view_as(s.block_table))
        for x in (s.k, s.v):
            x.view(torch.uint8).zero_()
        s.k_scale.zero_()
        s.v_scale.zero_()
        model.extend(s, prompt, i32(start))
        s.tokens.copy_(ids((B,), 3))
        s.active[2] = 0
        s.block_table[2] = s.block_table[0]

    go = lambda: model.verify(st, draft, u, r, counts=counts)
    fill(st)
    n, tok = go()
    if replay:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            n, tok = go()
        for _ in range(2):
            fill(st)
            graph.replay()
    fill(ref)
    before = ref.lengths.cpu().tolist()
    tokens = torch.cat((ref.tokens[:, None], draft), 1)
    model.extend(ref, tokens, i32([k + 1 for k in kept]))
    live = [b for b in range(B) if b != 2]
    assert [int(n[b]) for b in live] == [kept[b] for b in live]
    assert [int(st.lengths[b]) for b in live] == [before[b] + kept[b] + 1 for b in live] and int(st.lengths[2]) == before[2]
    for b in live:
        for x, y, name in zip(layer0(st, b, int(st.lengths[b])), layer0(ref, b, int(ref.lengths[b])), ("keys", "values", "key scales", "value scales")):
            assert torch.equal(x, y), f"row {b}: {name}"
        assert int(st.tokens[b]) == int(tok[b, kept[b]])
    # that the rejected drafts would have shown: written together with them, scales are larger
    loud = model.new_state(B, CTX, kv_dtype=kv_dtype, kv_block_size=16)
    fill(loud)
    model.extend(loud, tokens, i32([c + 1 for c in count]), advance=False)
    for b in (0, 4, 5):
        page = int(st.block_table[b, (int(st.lengths[b]) - 1) // 16])
        assert bool((loud.k_scale[0, page] > ref.k_scale[0, page]).all()) and bool((loud.v_scale[0, page] > ref.v_scale[0, page]).all())


@pytest.mark.parametrize("most", [5, 9, 14])
def test_the_kept_tokens_layers_in_several_writes(most, monkeypatch):
    """Where all layers' rows are more than a write takes, they go layer by layer or a few at a time, the last ones fewer: the
    cache is the same. Three layers of 5 rows."""
    from scratch_llm_amd import decode

    p = D.random_params(**{**SMALL, "n_layers": 3}, seed=22, std=0.05)
    cfg = decode.DecodeConfig(vocab_size=SMALL["vocab"], d_model=SMALL["d_model"], n_layers=3, n_heads=SMALL["n_heads"],
                              n_kv_heads=SMALL["n_kv_heads"], d_ff=SMALL["d_ff"], context_length=CTX)
    model = decode.Int4DecodeLM.from_state_dict(cfg, lambda n: p[n], DEV)
    B, T = 5, 4
    draft, u = ids((B, T), 61), torch.full((B, T), 0.9999, device=DEV)
    u[0], u[2, :2] = 0.0, 0.0
    states = []
    for limit in (1 << 16, most):
        st = model.new_state(B, CTX, kv_dtype="int8_block", kv_block_size=16)
        model.extend(st, ids((B, 13), 62), i32([13, 12, 9, 11, 0]))
        monkeypatch.setattr(decode, "_WRITE_ROWS", limit)
        n, _ = model.verify(st, draft, u, torch.full((B,), 0.3, device=DEV))
        assert n.tolist() == [4, 0, 2, 0, 0]
        states.append(raw(st))
    assert same(*states)


@pytest.mark.parametrize("kv_dtype", KV)
def test_rejected_drafts_at_the_table(model, kv_dtype):
    """Rows whose open block is on no page, past the table's end and at a negative length beside an ordinary one: nothing of
    the other rows' pages changes but what the ordinary row's kept tokens change."""
    print_case("verify at the table", kv_dtype)
    B, T = 4, 5
    st, ref = (model.new_state(B, 64, kv_dtype=kv_dtype, kv_block_size=32) for _ in range(2))
    prompt, draft, cur = ids((B, 40), 4), ids((B, T), 5), ids((B,), 6)
    draft[:, 2] = LOUD
    u = torch.full((B, T), 0.9999, device=DEV)
    u[:, :2] = 0.0
    for s in (st, ref):
        model.extend(s, prompt)
        s.tokens.copy_(cur)
        s.block_table[1, 1] = 1 << 20
        s.lengths[2] = 70  # the table ends at 64
        s.lengths[3] = -3
    held = raw(st)
    n, tok = model.verify(st, draft, u, torch.full((B,), 0.3, device=DEV))
    model.extend(ref, torch.cat((cur[:, None], draft), 1), i32([3, 0, 0, 0]))
    assert int(n[0]) == 2
    for x, y in zip(layer0(st, 0, 43), layer0(ref, 0, 43)):
        assert torch.equal(x, y)
    mine = st.block_table[0].long()
    for x, y in zip(raw(st), held):
        keep = torch.ones(x.shape[1], dtype=torch.bool, device=DEV)
        keep[mine] = False
        assert torch.equal(x[:, keep], y[:, keep])


def test_scores_are_those_of_the_whole_chunk():
    """A chunk is attended over a cache that holds all of it, so a loud token scales its block for the tokens before it in the
    chunk as well: the scores are those of the reference over a cache written so, loud token or not."""
    from tests.test_gpu_block_decode import BlockRefCache, check, ref_chunk
    from tests.test_gpu_block_decode import CTX as REF_CTX

    p = D.random_params(**SMALL, seed=21, std=0.05)
    k, v = p["blocks.0.attn.k_proj.weight"], p["blocks.0.attn.v_proj.weight"]
    e = sum(x / x.norm() for w in (k, v) for x in (w[5], w[128 + 9]))
    p["token_emb.weight"][LOUD] = e * (SMALL["d_model"] ** 0.5 / e.norm())
    model = build(p)
    refs = {dt: D.int4_model(p, n_layers=SMALL["n_layers"], n_heads=SMALL["n_heads"], n_kv_heads=SMALL["n_kv_heads"],
                             context_length=REF_CTX, dtype=dt) for dt in (torch.bfloat16, torch.float32)}
    B = 2
    st = model.new_state(B, CTX, kv_dtype="int8_block", kv_block_size=16)
    caches = {dt: BlockRefCache.make(r, B, dt, "int8", 16) for dt, r in refs.items()}
    prompt, chunk = ids((B, 10), 41).cpu(), ids((B, 4), 42).cpu()
    chunk[0, 2] = LOUD
    for x in (prompt, chunk):
        got = model.extend(st, x.to(DEV))
        l16, l32 = ref_chunk(refs, caches, x, [x.shape[1]] * B)
        check(got, l16, l32, f"chunk of {x.shape[1]}")


@pytest.mark.parametrize("kv_dtype", KV)
def test_speculation_follows_a_clear_continuation(kv_dtype):
    """A head whose row of the token that follows t is t's embedding, behind layers that add little: every pick is far ahead of
    the next best, so counts and continuation hold without conditions. Rows: all kept; a wrong second draft; an id
    outside the vocabulary first; fewer drafts than the others."""
    p = D.random_params(**SMALL, seed=31, std=0.02)
    follows = torch.randperm(SMALL["vocab"], generator=torch.Generator().manual_seed(32))
    p["lm_head.weight"] = torch.zeros_like(p["lm_head.weight"])
    p["lm_head.weight"][follows] = 0.05 * p["token_emb.weight"]
    model = build(p)
    B, T = 4, 4
    plain, spec = (model.new_state(B, CTX, kv_dtype=kv_dtype, kv_block_size=16) for _ in range(2))
    prompt = ids((B, 13), 33)
    for s in (plain, spec):
        s.tokens.copy_(model.extend(s, prompt, last_only=True).argmax(-1).to(torch.int32))
    want = [spec.tokens.cpu()]
    assert want[0].tolist() == follows[prompt[:, -1].long().cpu()].tolist()
    for _ in range(20):
        model.step(plain)
        top = plain.logits.float().topk(2, -1).values
        assert bool((top[:, 0] - top[:, 1] > 2.0**-3 * top[:, 0]).all())
        want.append(plain.tokens.cpu().clone())
        assert want[-1].tolist() == follows[want[-2].long()].tolist()
    want = torch.stack(want, 1)
    have = [[int(want[b, 0])] for b in range(B)]
    for step in range(3):
        draft = torch.zeros(B, T, dtype=torch.int32)
        for b in range(B):
            draft[b] = want[b, len(have[b]):len(have[b]) + T]
        draft[1, 1] = (draft[1, 1] + 1) % SMALL["vocab"]
        draft[2, 0] = SMALL["vocab"]
        n, tok = model.verify(spec, draft.to(DEV), None, None, temperature=0.0, counts=i32([T, T, T, 2]))
        assert n.tolist() == [T, 1, 0, 2], f"step {step}"
        for b in range(B):
            have[b] += tok[b, :int(n[b]) + 1].tolist()
            assert have[b] == want[b, :len(have[b])].tolist(), f"row {b} step {step}"
            assert int(spec.lengths[b]) == 13 + len(have[b]) - 1 and int(spec.tokens[b]) == have[b][-1]


@pytest.mark.parametrize("kv_dtype", KV)
def test_steps_of_a_wide_batch(kv_dtype):
    """70 rows: the step's linears are the prompt GEMM."""
    from tests.test_gpu_block_decode import CTX as REF_CTX
    from tests.test_gpu_block_decode import FMT, BlockRefCache, check, ref_steps

    print_case("block kv step of 70 rows", kv_dtype)
    p = D.random_params(**SMALL, seed=51, std=0.05)
    model = build(p)
    refs = {dt: D.int4_model(p, n_layers=SMALL["n_layers"], n_heads=SMALL["n_heads"], n_kv_heads=SMALL["n_kv_heads"],
                             context_length=REF_CTX, dtype=dt) for dt in (torch.bfloat16, torch.float32)}
    B = 70
    st = model.new_state(B, CTX, kv_dtype=kv_dtype, kv_block_size=32)
    caches = {dt: BlockRefCache.make(r, B, dt, FMT[kv_dtype], 32) for dt, r in refs.items()}
    for t in range(3):
        tok = ids((B,), 52 + t).cpu()
        model.step(st, tok)
        l16, l32 = ref_steps(refs, caches, tok[:, None])
        check(st.logits, l16[:, 0], l32[:, 0], f"step {t}")


def test_two_states_on_two_streams(model):
    """Verifications of two states issued beside each other on streams of their own: each as alone."""
    B, T = 3, 4
    draft, u = ids((B, T), 71), torch.full((B, T), 0.9999, device=DEV)
    u[0], u[1, :2] = 0.0, 0.0
    r = torch.full((B,), 0.4, device=DEV)

    def fresh(seed):
        s = model.new_state(B, CTX, kv_dtype="int8_block", kv_block_size=16)
        model.extend(s, ids((B, 11), seed))
        s.tokens.copy_(i32([3, 4, 5]))
        return s

    alone, beside = [fresh(72 + i) for i in range(2)], [fresh(72 + i) for i in range(2)]
    for s in alone:
        for _ in range(3):
            model.verify(s, draft, u, r)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for s, stream in zip(beside, streams):
            with torch.cuda.stream(stream):
                model.verify(s, draft, u, r)
    torch.cuda.synchronize()
    for a, b in zip(alone, beside):
        assert same(raw(a) + [a.lengths, a.tokens], raw(b) + [b.lengths, b.tokens])
