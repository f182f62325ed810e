"""The decode model on the block-scaled 8-bit cache: the step, chunks of a prompt, drafted tokens and their verification,
together as a server runs them, against oracle/decode_ref.py over oracle/kv_block_ref.py's cache.

Logits are compared as the other caches' are (tests/test_gpu_decode.py): against the fp32 reference over the same kind of
cache, within twice what the bf16 reference is off plus 2^-9 of the largest logit."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import decode_ref as D
from oracle import kv_block_ref as R
from tests.conftest import print_case

pytestmark = pytest.mark.gpu
DEV = "cuda"
SMALL = dict(vocab=1000, d_model=1024, n_layers=2, n_heads=8, n_kv_heads=2, d_ff=2048)
CTX = 192
FMT = {"int8_block": "int8", "fp8_block": "e4m3"}


@pytest.fixture(scope="module")
def small():
    from scratch_llm_amd.decode import DecodeConfig, Int4DecodeLM

    p = D.random_params(**SMALL, seed=11, std=0.05)
    cfg = DecodeConfig(vocab_size=SMALL["vocab"], d_model=SMALL["d_model"], n_layers=SMALL["n_layers"], n_heads=SMALL["n_heads"],
                       n_kv_heads=SMALL["n_kv_heads"], d_ff=SMALL["d_ff"], context_length=CTX)
    model = Int4DecodeLM.from_state_dict(cfg, lambda n: p[n], DEV)
    refs = {dt: D.int4_model(p, n_layers=cfg.n_layers, n_heads=cfg.n_heads, n_kv_heads=cfg.n_kv_heads, context_length=CTX,
                             dtype=dt) for dt in (torch.bfloat16, torch.float32)}
    return model, refs


class BlockRefCache(D.RefCache):
    """A RefCache whose keys and values are what a block-scaled cache gives back."""

    @classmethod
    def make(cls, m, batch, dtype, fmt, block):
        c = cls.empty(m, batch, CTX, dtype)
        c.fmt, c.block = fmt, block
        w = CTX // block
        c.table = np.arange(batch * w).reshape(batch, w)
        c.store = [(np.zeros((batch * w, m.n_kv_heads, block, m.head_dim), np.uint8),
                    np.zeros((batch * w, m.n_kv_heads, m.head_dim, block), np.uint8),
                    np.zeros((batch * w, m.n_kv_heads), np.float32), np.zeros((batch * w, m.n_kv_heads), np.float32))
                   for _ in range(m.n_layers)]
        return c

    def write_chunk(self, layer, k_new, v_new, counts):
        """k_new, v_new [B, Hkv, s, hd]: a block's scale goes by all of its tokens that one write brings."""
        st, n = self.store[layer], self.lengths.numpy()
        R.write(k_new.float().transpose(1, 2).numpy(), v_new.float().transpose(1, 2).numpy(), *st, self.table, n, counts, self.fmt)
        k, v = R.read(*st, self.table, np.zeros_like(n), n + counts, CTX, self.fmt)
        # fp32(code) * scale in the reference's own type, as attention takes it
        self.k[layer], self.v[layer] = (torch.from_numpy(x).transpose(1, 2).to(k_new.dtype) for x in (k, v))

    def write_decode(self, layer, k_new, v_new):
        self.write_chunk(layer, k_new, v_new, self.active.long().numpy())


def check(got, l16, l32, what):
    scale = float(l32.abs().max())
    e_hip, e_ref = float((got.float().cpu() - l32).abs().max()), float((l16.float() - l32).abs().max())
    assert e_hip <= 2 * e_ref + 2.0**-9 * scale, f"{what}: {e_hip:.4g} off, the bf16 reference {e_ref:.4g}"


def ref_steps(refs, caches, tokens):
    """Reference logits [B, n, V] of n tokens a row, one after the other."""
    out = {}
    for dt in refs:
        out[dt] = torch.stack([D.decode_step(refs[dt], caches[dt], tokens[:, i], dt).float() for i in range(tokens.shape[1])], 1)
    return out[torch.bfloat16], out[torch.float32]


@torch.no_grad()
def ref_chunk(refs, caches, tokens, counts):
    """Reference logits [B, n, V] of a chunk of tokens written at once (model.py:439-505 over several tokens a row)."""
    out = []
    for dt in (torch.bfloat16, torch.float32):
        m, cache = refs[dt], caches[dt]
        b, n = tokens.shape
        cos, sin = D.rope_tables(m.head_dim, m.context_length, m.rope_theta)
        pos = cache.lengths[:, None] + torch.arange(n)
        seen = (torch.arange(CTX) <= pos[..., None])[:, None]
        x = m.embed.to(dt)[tokens.long()]
        for i in range(m.n_layers):
            h = D.rmsnorm(x, m.norms[f"blocks.{i}.attn_norm"].to(dt), m.eps)
            q, k, v = (D.linear(h, m.linears[f"blocks.{i}.attn.{c}_proj"]).view(b, n, -1, m.head_dim).transpose(1, 2) for c in "qkv")
            q, k = (D.rope(y, pos.clamp(max=m.context_length - 1), cos, sin) for y in (q, k))
            cache.write_chunk(i, k, v, np.array(counts))
            kk, vv = (y.repeat_interleave(m.n_heads // m.n_kv_heads, 1) for y in (cache.k[i], cache.v[i]))
            o = D.attention(q, kk, vv, seen).transpose(1, 2).reshape(b, n, -1)
            x = x + D.linear(o, m.linears[f"blocks.{i}.attn.o_proj"])
            x = x + D._ffn(m, i, D.rmsnorm(x, m.norms[f"blocks.{i}.ffn_norm"].to(dt), m.eps))
        out.append(D.linear(D.rmsnorm(x, m.final_norm.to(dt), m.eps), m.linears["lm_head"]).float())
        cache.lengths += torch.tensor(counts)
    return out


@pytest.mark.parametrize("kv_dtype", ["int8_block", "fp8_block"])
@pytest.mark.parametrize("B,block", [(1, 16), (3, 64), (5, 32)])
def test_step_matches_reference(small, B, block, kv_dtype):
    model, refs = small
    print_case("block kv step", B, block, kv_dtype)
    st = model.new_state(B, CTX, kv_dtype=kv_dtype, kv_block_size=block)
    caches = {dt: BlockRefCache.make(r, B, dt, FMT[kv_dtype], block) for dt, r in refs.items()}
    tok = torch.randint(0, model.cfg.vocab_size, (B,), generator=torch.Generator().manual_seed(B))
    for t in range(20 if block == 16 else 6):
        nxt = model.step(st, tok)
        l16, l32 = ref_steps(refs, caches, tok[:, None])
        check(st.logits, l16[:, 0], l32[:, 0], f"step {t}")
        assert st.lengths.cpu().tolist() == [t + 1] * B
        tok = nxt.cpu().long()
        assert torch.equal(tok, st.logits.float().argmax(-1).cpu())


@pytest.mark.parametrize("kv_dtype", ["int8_block", "fp8_block"])
def test_chunks_of_a_prompt_then_steps(small, kv_dtype):
    """Ragged chunks (row counts 7, 3 and 0 of 7; then 20 of each: 60 rows; then 30: 90 rows, the prompt GEMM and its
    SiLU kernel), then steps."""
    model, refs = small
    print_case("block kv extend", kv_dtype)
    B = 3
    st = model.new_state(B, CTX, kv_dtype=kv_dtype)
    caches = {dt: BlockRefCache.make(r, B, dt, FMT[kv_dtype], 64) for dt, r in refs.items()}
    g = torch.Generator().manual_seed(3)
    first = torch.randint(0, 1000, (B, 7), generator=g, dtype=torch.int32)
    counts = [7, 3, 0]
    got = model.extend(st, first.to(DEV), torch.tensor(counts, dtype=torch.int32, device=DEV))
    assert got.shape == (B, 7, 1000) and st.lengths.cpu().tolist() == counts
    l16, l32 = ref_chunk(refs, caches, first, counts)
    for b, n in enumerate(counts):
        if n:
            check(got[b, :n], l16[b, :n], l32[b, :n], f"first chunk, row {b}")
    for n in (20, 30):
        chunk = torch.randint(0, 1000, (B, n), generator=g, dtype=torch.int32)
        last = n == 30
        got = model.extend(st, chunk.to(DEV), last_only=last)
        l16, l32 = ref_chunk(refs, caches, chunk, [n] * B)
        check(got, l16[:, -1] if last else l16, l32[:, -1] if last else l32, f"chunk of {n}")
    tok = torch.tensor([5, 6, 7])
    for t in range(3):
        nxt = model.step(st, tok)
        l16, l32 = ref_steps(refs, caches, tok[:, None])
        check(st.logits, l16[:, 0], l32[:, 0], f"step {t}")
        tok = nxt.cpu().long()
    assert st.lengths.cpu().tolist() == [n + 53 for n in counts]


def test_write_kv_equals_the_cache_write(small):
    """A prefill's keys and values stored by write_kv read back as write_kv_blocks leaves them."""
    from scratch_llm_amd.quant import kv_block

    model, _ = small
    st = model.new_state(2, 100, kv_dtype="int8_block", kv_block_size=32)
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(2, 2, 70, 128, generator=g).bfloat16().to(DEV) for _ in range(2))
    st.write_kv(1, k, v)
    k2, v2 = kv_block.read_kv_blocks(*st.kv_layer(1), st.block_table, torch.zeros(2, dtype=torch.int32, device=DEV), 70)
    for x, y in ((k, k2), (v, v2)):
        for i in range(0, 70, 32):
            a, b = x[:, :, i:i + 32].float(), y.transpose(1, 2)[:, :, i:i + 32]
            step = a.abs().amax((-1, -2), keepdim=True) / 127
            assert bool(((a - b).abs() <= step * 0.5001).all())
    assert int(st.k[0].abs().max()) == 0
    with pytest.raises(ValueError):
        st.write_kv(1, k, v, start=40)


@pytest.mark.parametrize("kv_dtype", ["int8_block", "fp8_block"])
def test_graph_replays_equal_eager_and_inactive_rows_stay(small, kv_dtype):
    """A captured step replayed with eager steps, a chunk and changing flags between the replays; a row that is not active
    keeps its cache, bit for bit, and its length."""
    model, _ = small
    print_case("block kv graph", kv_dtype)
    a, b = (model.new_state(4, CTX, kv_dtype=kv_dtype, kv_block_size=16) for _ in range(2))
    prompt = torch.randint(0, 1000, (4, 37), generator=torch.Generator().manual_seed(2), dtype=torch.int32).to(DEV)
    for s in (a, b):
        model.extend(s, prompt)
        s.set_tokens(torch.tensor([5, 17, 300, 999]), 1000)
    graph = model.capture(b)
    for t in range(6):
        if t == 2:
            a.active[1] = b.active[1] = 0
            held = [x[:, b.block_table[1].long()].clone() for x in (b.k.view(torch.uint8), b.v.view(torch.uint8), b.k_scale, b.v_scale)]
        model.step(a)
        graph.replay()
        torch.cuda.synchronize()
        live = [0, 2, 3] if t >= 2 else [0, 1, 2, 3]
        assert torch.equal(a.logits[live], b.logits[live]), f"replay {t}"
        a.tokens[1] = b.tokens[1] = 17
    for x, y in zip(held, (b.k.view(torch.uint8), b.v.view(torch.uint8), b.k_scale, b.v_scale)):
        assert torch.equal(x, y[:, b.block_table[1].long()])
    assert torch.equal(a.k.view(torch.uint8), b.k.view(torch.uint8)) and torch.equal(a.v_scale, b.v_scale)
    assert b.lengths.cpu().tolist() == [43, 39, 43, 43]


@pytest.mark.parametrize("kv_dtype", ["int8_block", "fp8_block"])
def test_speculative_steps(small, kv_dtype):
    """Drafts taken from the model's own greedy continuation (kept), with wrong tokens put in (rejected there): the tokens
    kept are the greedy continuation, whatever was drafted. Scores that differ between one token and several a row by
    their rounding may turn a near tie, so the continuation is followed where its top two are apart."""
    model, refs = small
    print_case("speculative", kv_dtype)
    B, T = 4, 4
    prompt = torch.randint(0, 1000, (B, 25), generator=torch.Generator().manual_seed(4), dtype=torch.int32).to(DEV)
    plain, spec = (model.new_state(B, CTX, kv_dtype=kv_dtype) for _ in range(2))
    for s in (plain, spec):
        lg = model.extend(s, prompt, last_only=True)
        s.tokens.copy_(lg.argmax(-1).to(torch.int32))
    first = plain.tokens.clone()
    want, sure = [first.cpu()], []
    for _ in range(16):
        model.step(plain)
        want.append(plain.tokens.cpu().clone())
        top = plain.logits.float().topk(2, -1).values.cpu()
        sure.append((top[:, 0] - top[:, 1]) > 2.0**-5 * plain.logits.float().abs().max().cpu())
    want, sure = torch.stack(want, 1), torch.stack(sure, 1)  # want[:, i + 1] is sure where sure[:, i]
    have = [[int(first[b])] for b in range(B)]
    for step in range(3):
        draft = torch.zeros(B, T, dtype=torch.int32)
        for b in range(B):
            at = len(have[b])
            draft[b] = want[b, at:at + T]
            if b == 1:
                draft[b, 1] = (draft[b, 1] + 1) % 1000
            if b == 2:
                draft[b, 0] = 1000  # no such token
        before = spec.lengths.cpu().tolist()
        n, tok = model.verify(spec, draft.to(DEV), None, None, temperature=0.0,
                              counts=torch.tensor([T, T, T, 2], dtype=torch.int32, device=DEV))
        n, tok = n.cpu().tolist(), tok.cpu()
        for b in range(B):
            ok = bool(sure[b, :len(have[b]) + T].all())
            if ok:
                assert n[b] == {0: T, 1: 1, 2: 0, 3: 2}[b], f"row {b} step {step}: {n[b]} accepted"
            have[b] += tok[b, :n[b] + 1].tolist()
            if ok:
                assert have[b] == want[b, :len(have[b])].tolist()
            assert tok[b, n[b] + 1:].tolist() == [-1] * (T - n[b])
            assert spec.lengths.cpu()[b] == before[b] + n[b] + 1 and int(spec.tokens[b]) == have[b][-1]
    assert bool(sure.float().mean() > 0.5), "too few clear picks to say anything"


def test_verify_samples_with_given_numbers_and_skips_inactive_rows(small):
    model, _ = small
    B, T = 3, 3
    prompt = torch.randint(0, 1000, (B, 10), generator=torch.Generator().manual_seed(4), dtype=torch.int32).to(DEV)
    g = torch.Generator().manual_seed(5)
    draft = torch.randint(0, 1000, (B, T), generator=g, dtype=torch.int32).to(DEV)
    probs = torch.softmax(torch.randn(B, T, 1000, generator=g), -1).to(DEV)
    u, r = torch.rand(B, T, generator=g).to(DEV), torch.rand(B, generator=g).to(DEV)
    st, other = (model.new_state(B, CTX, kv_dtype="int8_block") for _ in range(2))
    for s in (st, other):
        model.extend(s, prompt)
        s.tokens.fill_(7)
        s.active[2] = 0
    lg = model.extend(other, torch.cat((other.tokens[:, None], draft), 1), advance=False)
    n, tok = model.verify(st, draft, u, r, draft_probs=probs, temperature=0.9)
    wn, wt = R.verify(lg.double().cpu().numpy(), draft.cpu().numpy(), [T] * B, probs.double().cpu().numpy(), u.cpu().numpy(),
                      r.cpu().numpy(), 0.9)
    assert n.cpu().tolist() == wn.tolist() and tok.cpu().tolist() == wt.tolist()
    assert st.lengths.cpu().tolist() == [10 + int(wn[0]) + 1, 10 + int(wn[1]) + 1, 10]
    assert int(st.tokens[2]) == 7 and int(st.tokens[0]) == int(wt[0, wn[0]])


@pytest.mark.parametrize("temperature", [0.0, 0.9])
def test_a_captured_chunk_and_verification_replay_as_eager(small, temperature):
    """A chunk and a speculative step recorded in one graph and replayed with other tokens, drafts, numbers and counts: the
    same logits, tokens and cache as the calls themselves, which run between the replays."""
    model, _ = small
    B, T = 3, 3
    g = torch.Generator().manual_seed(8)
    ids, draft = (torch.zeros(B, n, dtype=torch.int32, device=DEV) for n in (5, T))
    counts = torch.zeros(B, dtype=torch.int32, device=DEV)
    u, r, probs = torch.zeros(B, T, device=DEV), torch.zeros(B, device=DEV), torch.zeros(B, T, 1000, device=DEV)

    def fresh():
        for x in (ids, draft):
            x.copy_(torch.randint(0, 1000, x.shape, generator=g, dtype=torch.int32))
        counts.copy_(torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32))
        u.copy_(torch.rand(B, T, generator=g))
        r.copy_(torch.rand(B, generator=g))
        probs.copy_(torch.softmax(2 * torch.randn(B, T, 1000, generator=g), -1))

    def go(s):
        return (model.extend(s, ids, last_only=True), *model.verify(s, draft, u, r, draft_probs=probs, counts=counts, temperature=temperature))

    fresh()
    st, eager = (model.new_state(B, CTX, kv_dtype="int8_block", kv_block_size=32) for _ in range(2))
    go(model.new_state(B, CTX, kv_dtype="int8_block", kv_block_size=32))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = go(st)
    for i in range(4):
        fresh()
        want = go(eager)
        graph.replay()
        torch.cuda.synchronize()
        for x, y, name in zip(got, want, ("logits", "accepted", "tokens")):
            assert torch.equal(x, y), f"replay {i}: {name}"
        for name in ("k", "v", "k_scale", "v_scale", "lengths", "tokens"):
            assert torch.equal(getattr(st, name), getattr(eager, name)), f"replay {i}: state's {name}"


def test_refusals(small):
    model, _ = small
    st = model.new_state(2, 64, kv_dtype="int8_block")
    ids = torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="block-scaled"):
        model.extend(model.new_state(2, 64), ids)
    with pytest.raises(ValueError, match="no blocks"):
        model.new_state(2, 64).kv_layer(0)
    for bad in (ids[:1], ids.long(), ids[:, :0], ids[0]):
        with pytest.raises(ValueError, match="tokens"):
            model.extend(st, bad)
    with pytest.raises(ValueError, match="counts"):
        model.extend(st, ids, torch.zeros(2, device=DEV))
    with pytest.raises(RuntimeError, match="device tensors"):
        model.extend(st, ids.cpu())
    with pytest.raises(ValueError, match="draft"):
        model.verify(st, ids.long(), None, None, temperature=0.0)
    with pytest.raises(ValueError, match="at most"):
        model.verify(st, torch.zeros(2, 64, dtype=torch.int32, device=DEV), None, None, temperature=0.0)
    with pytest.raises(ValueError, match="per-head scales"):
        st.set_kv_scales(0, torch.ones(2), torch.ones(2))
    with pytest.raises(ValueError, match="kv_dtype"):
        model.new_state(2, 64, kv_dtype="int8")
    with pytest.raises(ValueError, match="block must be"):
        model.new_state(2, 64, kv_dtype="int8_block", kv_block_size=48)


def test_past_the_end_of_the_table(small):
    """Steps and chunks past a row's last page store nothing, attend what is there and touch no other row."""
    model, _ = small
    st = model.new_state(2, 32, kv_dtype="int8_block", kv_block_size=32)
    ids = torch.randint(0, 1000, (2, 30), generator=torch.Generator().manual_seed(4), dtype=torch.int32).to(DEV)
    model.extend(st, ids)
    st.lengths[1] = 20
    for _ in range(2):
        model.step(st)
    held = st.k[:, 0].clone()
    lg = model.extend(st, ids[:, :5])
    model.step(st)
    assert torch.equal(held, st.k[:, 0]) and bool(torch.isfinite(lg.float()).all())
    assert st.lengths.cpu().tolist() == [38, 28]
