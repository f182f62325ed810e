"""Several continuations of one prompt over the paged 8-bit key/value cache, as timed cases.

Three operators in the order in which a serving loop calls them when it draws several answers to a prompt, searches with
beams, or serves many users behind one system prompt:

* `pages`: the pages of the cache are handed out, shared, copied, released and moved together. A page that a row goes on
  writing to is copied, full pages are shared and counted (`fork`); rows give their pages back and new tokens get theirs
  (`turn`); named pages are copied (`copy`); what is in use moves to the front of the pool (`compact`);
* `attend`: attention of one or a few new tokens per row where rows share the first part of their context, which is read
  once for all of them;
* `sample`: the next token from a row of logits, with temperature, top-k, top-p and min-p, from given random numbers.

Caches are those of `perf/operators.py`, with all layers of a model in one tensor: codes of the keys
[layers, pages, Hkv, block, D] and of the values [layers, pages, Hkv, D, block] (int8 or E4M3), fp32 scales
[layers, pages, Hkv] of each. A row's block table names the page of every `block` tokens, -1 where there is none;
`refs` counts the table entries that name a page. Heads are those of Llama-3-8B (32 query, 8 key/value, 128 wide) and of
generic models; the vocabularies are its 128256 and generic ones.

Pages move bit by bit: their codes come back as the whole numbers that are stored, to be equal, beside their scales.

`own` is set by what imports this file: with it false `run` computes plain torch operations, with it true it calls
this package.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def listed():
    return [
        # one prompt, eight answers: the open page is copied for seven rows of a small model, latency counts
        {"name": "fork_samples", "kind": "fork", "b": 8, "n": 8, "beam": False, "layers": 4, "hkv": 2, "d": 64, "block": 16,
         "fmt": "int8", "ctx": 777},
        # beams of sixteen prompts take up the better half's, all layers of an 8B model
        {"name": "fork_beams", "kind": "fork", "b": 64, "n": 4, "beam": True, "layers": 32, "hkv": 8, "d": 128, "block": 64,
         "fmt": "e4m3", "ctx": 1500},
        # a quarter of a full batch is done and makes room for new prompts, the others need room for their next token
        {"name": "turn_batch", "kind": "turn", "b": 96, "layers": 8, "hkv": 8, "d": 128, "block": 32, "fmt": "int8",
         "ctx": 3001, "new": 700},
        # a prompt's pages copied out of a pool
        {"name": "copy_prompt", "kind": "copy", "n": 125, "layers": 16, "hkv": 8, "d": 128, "block": 64, "fmt": "int8",
         "pages": 320},
        # a pool of which sixty in a hundred pages are in use, anywhere, over 2^31 bytes of keys
        {"name": "compact_pool", "kind": "compact", "b": 24, "layers": 32, "hkv": 8, "d": 128, "block": 64, "fmt": "int8",
         "pages": 1100, "ctx": 1760},
        # eight answers to one prompt, a token each
        {"name": "attend_samples", "kind": "attend", "layers": 4, "b": 8, "n": 8, "t": 1, "h": 32, "hkv": 8, "d": 128,
         "block": 64, "fmt": "int8", "dtype": "bf16", "shared": 2000, "ctx": 150},
        # a full batch behind one long system prompt
        {"name": "attend_system", "kind": "attend", "layers": 4, "b": 64, "n": 64, "t": 1, "h": 32, "hkv": 8, "d": 128,
         "block": 64, "fmt": "int8", "dtype": "bf16", "shared": 8192, "ctx": 700},
        # many prompts with several answers each, uneven and long
        {"name": "attend_groups", "kind": "attend", "layers": 2, "b": 96, "n": 16, "t": 1, "h": 32, "hkv": 8, "d": 128,
         "block": 32, "fmt": "e4m3", "dtype": "bf16", "shared": 15000, "ctx": 900},
        # drafted tokens of a few answers to each prompt, a model with as many key heads as query heads
        {"name": "attend_drafts", "kind": "attend", "layers": 4, "b": 12, "n": 4, "t": 5, "h": 12, "hkv": 12, "d": 64,
         "block": 16, "fmt": "e4m3", "dtype": "fp16", "shared": 3333, "ctx": 400},
        # one stream's next token
        {"name": "sample_token", "kind": "sample", "b": 1, "v": 32000, "dtype": "fp32", "temp": 0.8, "k": 40, "p": 0.95,
         "minp": 0.0, "each": False},
        # a batch's, nucleus only
        {"name": "sample_batch", "kind": "sample", "b": 64, "v": 128256, "dtype": "bf16", "temp": 1.0, "k": 0, "p": 0.95,
         "minp": 0.0, "each": False},
        # a large batch whose rows each have settings of their own, an odd vocabulary
        {"name": "sample_rows", "kind": "sample", "b": 201, "v": 50257, "dtype": "fp32", "temp": 0.9, "k": 100, "p": 0.9,
         "minp": 0.05, "each": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["fork", "turn", "copy", "compact", "attend", "attend", "attend", "attend", "sample", "sample", "sample"])
    d = rng.choice([64, 128, 128, 256])
    fmt = rng.choice(["int8", "e4m3"])
    block = rng.choice([16, 32, 64, 128])
    hkv = rng.choice([1, 2, 4, 8, 12])
    if kind == "sample":
        b = _log_int(rng, 1, 200)
        return {"kind": kind, "b": b, "v": _log_int(rng, 500, min(128256, 8000000 // b)), "dtype": rng.choice(["bf16", "fp32", "fp16"]),
                "temp": rng.choice([0.0, 0.6, 1.0, 1.5]), "k": rng.choice([0, 0, 1, 20, 100, 5000]),
                "p": rng.choice([1.0, 0.95, 0.9, 0.5]), "minp": rng.choice([0.0, 0.0, 0.02, 0.1]), "each": rng.random() < 0.4}
    if kind == "attend":
        t = rng.choice([1, 1, 1, _log_int(rng, 2, 8)])
        n = _log_int(rng, 2, 48)
        shared = _log_int(rng, 40, 20000)
        groups = _log_int(rng, 1, max(1, min(48 // n, 200000 // (n * shared))))
        group = rng.choice([1, 2, 3, 4, 8]) if hkv < 12 else rng.choice([1, 2])
        layers = rng.choice([1, 2, 4])
        shared = max(40, min(shared, int(8e9) // (layers * n * groups * t * hkv * group * d)))
        return {"kind": kind, "layers": layers, "b": n * groups, "n": n, "t": t, "h": hkv * group, "hkv": hkv,
                "d": d, "block": block, "fmt": fmt, "dtype": rng.choice(["bf16", "bf16", "fp16"]), "shared": shared,
                "ctx": t + _log_int(rng, 1, 1000)}
    page = hkv * block * d  # bytes of a page's keys
    layers = max(1, min(_log_int(rng, 1, 32), (1 << 23) // page))
    if kind == "copy":
        n = _log_int(rng, 1, max(1, min(500, (1 << 28) // (page * layers))))
        return {"kind": kind, "n": n, "layers": layers, "hkv": hkv, "d": d, "block": block, "fmt": fmt, "pages": 2 * n + rng.randrange(1, 40)}
    ctx = _log_int(rng, 2, max(3, min(4000, (1 << 29) // (page * layers) * block)))
    if kind == "compact":
        b = _log_int(rng, 1, max(1, min(64, (1 << 30) // (page * layers * (ctx // block + 1)))))
        return {"kind": kind, "b": b, "layers": layers, "hkv": hkv, "d": d, "block": block, "fmt": fmt,
                "pages": int(b * (ctx // block + 1) * rng.uniform(1.1, 3.0)) + 2, "ctx": ctx}
    rows = max(1, min(64, (1 << 30) // (page * layers * (ctx // block + 2))))
    if kind == "turn":
        return {"kind": kind, "b": _log_int(rng, 1, rows), "layers": layers, "hkv": hkv, "d": d, "block": block, "fmt": fmt,
                "ctx": ctx, "new": _log_int(rng, 1, ctx)}
    n = _log_int(rng, 2, max(2, rows))
    return {"kind": kind, "b": n * max(1, rng.randrange(1, rows // n + 1) if rows > n else 1), "n": n, "beam": rng.random() < 0.5,
            "layers": layers, "hkv": hkv, "d": d, "block": block, "fmt": fmt, "ctx": ctx}


# ---------------------------------------------------------------------------------------------- sizes of a case
def _spread(b, most, part):
    """Lengths of b rows: the first the longest, the others down to 1 - part of it, unevenly."""
    return [most - (i * 7919) % (int(most * part) + 1) for i in range(b)]


def _groups(case):
    """(shared tokens of each group, own tokens of each row) of an `attend` case; the last t of a row's own are the new ones.
    The shared part ends where the group's prompt does, inside a page or not: the rows share the pages before."""
    shared = _spread(case["b"] // case["n"], case["shared"], 0.4)
    rest = [max(case["t"], x) for x in _spread(case["b"], case["ctx"], 0.7)]
    return shared, rest


def _parents(case):
    """The row that each row of a `fork` case goes on from."""
    b, n = case["b"], case["n"]
    return [i - i % n + (i % n) // 2 if case["beam"] else i - i % n for i in range(b)]


def _page_bytes(case):
    """Bytes of one page in all layers, keys and values and their scales."""
    return 2 * case["layers"] * case["hkv"] * (case["block"] * case["d"] + 4)


def work(case):
    kind = case["kind"]
    if kind == "sample":
        es = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": case["b"] * (case["v"] * es + 8), "flops": 4 * case["b"] * case["v"]}
    if kind == "attend":
        shared, rest = _groups(case)
        h, hkv, d, block, t = (case[x] for x in ("h", "hkv", "d", "block", "t"))
        full = [s - s % block for s in shared]
        keys = sum(full) + sum(shared[i // case["n"]] % block + r for i, r in enumerate(rest))
        pairs = sum(t * (shared[i // case["n"]] + r) - t * (t - 1) // 2 for i, r in enumerate(rest))
        return {"bytes": case["layers"] * (4 * case["b"] * t * h * d + keys * 2 * hkv * d + 8 * hkv * (keys // block + case["b"])),
                "flops": case["layers"] * 4 * h * d * pairs}
    if kind == "copy":
        return {"bytes": 2 * case["n"] * _page_bytes(case), "flops": 0}
    block = case["block"]
    if kind == "fork":
        parents, lengths = _parents(case), _spread(case["b"], case["ctx"], 0.3)
        moved = sum(lengths[p] % block != 0 for p in parents) - sum(lengths[p] % block != 0 for p in set(parents))
        entries = 2 * sum(-(-lengths[p] // block) for i, p in enumerate(parents) if i != p)
    elif kind == "turn":
        starts, counts = _turn(case)
        moved = sum(_shares(i) and starts[i] > 0 and starts[i] % block != 0 and starts[i - i % 4 + 2] == starts[i] for i in range(case["b"]))
        entries = sum(-(-(s + c) // block) - s // block for s, c in zip(starts, counts))
    else:
        live = sum(-(-x // block) for x in _spread(case["b"], case["ctx"], 0.5))
        moved = live - live * live // case["pages"]  # of pages in use anywhere, those behind the first `live`
        entries = live
    return {"bytes": 2 * moved * _page_bytes(case) + 16 * entries, "flops": 0}


def _shares(i):
    """Rows 2 and 3 of every four of a `turn` case are one sequence that has not parted yet, open page included."""
    return i % 4 in (2, 3)


def _turn(case):
    """(tokens that each row of a `turn` case keeps, tokens it gets room for): every fourth row is done, a prompt takes its place."""
    lengths = _spread(case["b"], case["ctx"], 0.5)
    lengths = [lengths[i - 1] if i % 4 == 3 else x for i, x in enumerate(lengths)]
    fresh = _spread(case["b"], case["new"], 0.5)
    return [0 if i % 4 == 1 else x for i, x in enumerate(lengths)], [fresh[i] if i % 4 == 1 else 1 for i in range(case["b"])]


# ---------------------------------------------------------------------------------------------- inputs
def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cache(gen, case, pages):
    """A filled cache: codes as a quantizer leaves them, scales that vary from page to page."""
    layers, hkv, block, d = (case[x] for x in ("layers", "hkv", "block", "d"))
    lim = 126 if case["fmt"] == "int8" else 120  # of E4M3 codes: magnitudes below 256, no NaN
    codes = []
    for shape in ((layers, pages, hkv, block, d), (layers, pages, hkv, d, block)):
        out = torch.empty(shape, dtype=torch.int8, device="cuda")
        for layer in out:
            # the sum of two uniform numbers: most codes are small, as those of normal values are
            x = torch.randint(-lim // 2, lim // 2 + 1, layer.shape, generator=gen, device="cuda", dtype=torch.int8)
            layer.copy_(x).add_(torch.randint(-lim // 2, lim // 2 + 1, layer.shape, generator=gen, device="cuda", dtype=torch.int8))
            if case["fmt"] == "e4m3":
                layer.copy_((layer.to(torch.float32) * (1.0 / 32.0)).to(torch.float8_e4m3fn).view(torch.int8))
        codes.append(out.view(CODES[case["fmt"]]))
    spread = 40.0 if case["fmt"] == "int8" else 1.4
    scales = [torch.exp(0.3 * torch.randn(layers, pages, hkv, generator=gen, device="cuda")) / spread for _ in range(2)]
    return codes[0], codes[1], scales[0], scales[1]


def _scattered(gen, pages, lengths, block, width):
    """A table of rows that own their pages, anywhere in the pool, as a server's allocator leaves them."""
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    used = _int32([-(-x // block) for x in lengths])[:, None]
    at = torch.arange(width, device="cuda")
    first = torch.cumsum(used, 0) - used
    return torch.where(at < used, order[(first + at).clamp(max=pages - 1).long()], -1).to(torch.int32)


def _refs(table, pages):
    return torch.bincount(table[table >= 0], minlength=pages).to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind = case["kind"]
    st = {"case": case}
    if kind == "sample":
        b, v = case["b"], case["v"]
        # a broad bulk and a few likely tokens, rows of different sharpness; some rows may use half of the vocabulary only
        x = 2.0 * torch.randn(b, v, generator=gen, device="cuda")
        x += 9.0 * (torch.rand(b, v, generator=gen, device="cuda") < 60.0 / v)
        x *= 0.7 + 0.8 * torch.rand(b, 1, generator=gen, device="cuda")
        allowed = (torch.rand(b, v, generator=gen, device="cuda") < 0.5) | (torch.arange(b, device="cuda") % 4 != 3)[:, None]
        allowed[:, 0] = True
        st["logits"] = x.masked_fill_(~allowed, -math.inf).to(DTYPES[case["dtype"]])
        st["u"] = torch.rand(b, generator=gen, device="cuda")
        st["temp"], st["k"], st["p"], st["minp"] = case["temp"], case["k"], case["p"], case["minp"]
        if case["each"]:  # settings row by row: some greedy, some without one of the limits
            r = torch.rand(4, b, generator=gen, device="cuda")
            st["temp"] = torch.where(r[0] < 0.1, 0.0, case["temp"] + r[0])
            st["k"] = torch.where(r[1] < 0.3, 0, (r[1] * (2 * case["k"] + 4)).to(torch.int32))
            st["p"] = torch.where(r[2] < 0.3, 1.0, r[2])
            st["minp"] = torch.where(r[3] < 0.5, 0.0, case["minp"] * r[3])
        return st
    block = case["block"]
    if kind == "attend":
        shared, rest = _groups(case)
        b, n, t, h = case["b"], case["n"], case["t"], case["h"]
        own_pages = [-(-(shared[i // n] % block + r) // block) for i, r in enumerate(rest)]
        full = [s // block for s in shared]
        width = max(full[i // n] + own_pages[i] for i in range(b))
        pages = sum(full) + sum(own_pages) + 1
        st["cache"] = _cache(gen, case, pages)
        order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
        common = _int32(full)
        at = torch.arange(width, device="cuda")
        group = torch.arange(b, device="cuda") // n
        mine = _int32(own_pages)
        lead = (torch.cumsum(common, 0) - common)[group][:, None] + at
        tail = sum(full) + (torch.cumsum(mine, 0) - mine)[:, None] + at - common[group][:, None]
        where = torch.where(at < common[group][:, None], lead, tail.clamp(max=pages - 1))
        st["table"] = torch.where(at < (common[group] + mine)[:, None], order[where.long()], -1).to(torch.int32).contiguous()
        st["starts"] = _int32([shared[i // n] + r - t for i, r in enumerate(rest)])
        st["leaders"] = (group * n).to(torch.int32)
        st["q"] = [torch.randn(b, t, h, case["d"], generator=gen, device="cuda").to(DTYPES[case["dtype"]]) for _ in range(case["layers"])]
        return st
    if kind == "copy":
        st["cache"] = _cache(gen, case, case["pages"])
        order = torch.randperm(case["pages"], generator=gen, device="cuda").to(torch.int32)
        st["src"], st["dst"] = order[:case["n"]].contiguous(), order[case["n"]:2 * case["n"]].contiguous()
        return st
    b = case["b"]
    if kind == "compact":
        lengths = _spread(b, case["ctx"], 0.5)
        pages = case["pages"]
        st["table"] = _scattered(gen, pages, lengths, block, -(-max(lengths) // block))
    elif kind == "fork":
        lengths = _spread(b, case["ctx"], 0.3)
        pages = 2 * sum(-(-x // block) for x in lengths) + b
        st["table"] = _scattered(gen, pages, lengths, block, -(-max(lengths) // block) + 1)
        st["parents"] = _int32(_parents(case))
    else:
        lengths = _spread(b, case["ctx"], 0.5)
        lengths = [lengths[i - 1] if i % 4 == 3 else x for i, x in enumerate(lengths)]
        starts, counts = _turn(case)
        width = max(-(-max(x, s + c) // block) for x, s, c in zip(lengths, starts, counts))
        pages = sum(-(-max(x, s + c) // block) for x, s, c in zip(lengths, starts, counts)) + b
        st["table"] = _scattered(gen, pages, lengths, block, width)
        twin = torch.arange(b, device="cuda")
        st["table"] = st["table"][torch.where(twin % 4 == 3, twin - 1, twin)].contiguous()
        st["keep"], st["counts"] = _int32(starts), _int32(counts)
    st["cache"] = _cache(gen, case, pages)
    st["refs"] = _refs(st["table"], pages)
    st["lengths"] = _int32(lengths)
    # what a server's tables hold when the pass begins; `fork` may go on from its own result
    st["begin"] = {x: st[x].clone() for x in ("table", "refs", "lengths")} if kind != "fork" else {}
    return st


# ---------------------------------------------------------------------------------------------- one pass
def run(st):
    kind = st["case"]["kind"]
    for x in st.get("begin", ()):
        st[x].copy_(st["begin"][x])
    if own:
        return _own(st, kind)
    return {"fork": _plain_fork, "turn": _plain_turn, "copy": _plain_copy, "compact": _plain_compact, "attend": _plain_attend,
            "sample": _plain_sample}[kind](st)


def _own(st, kind):
    from scratch_llm_amd import sampling
    from scratch_llm_amd.quant import kv_pages, kv_shared

    case = st["case"]
    if kind == "sample":
        return sampling.sample_tokens(st["logits"], st["u"], temperature=st["temp"], top_k=st["k"], top_p=st["p"], min_p=st["minp"])
    cache = st["cache"]
    if kind == "attend":
        shared = kv_shared.plan_shared_kv(st["table"], st["starts"], st["leaders"], block=case["block"], tokens=case["t"],
                                          heads=case["h"], kv_heads=case["hkv"], head_dim=case["d"])
        return [kv_shared.attend_shared_kv(q, *layer, st["table"], st["starts"], shared=shared) for q, layer in zip(st["q"], zip(*cache))]
    if kind == "copy":
        kv_pages.copy_kv_pages(st["src"], st["dst"], *cache)
        return _pool(cache)
    if kind == "compact":
        live, moved = kv_pages.compact_kv_pages(*cache, st["table"], st["refs"])
        return {"live": live, "moved": moved, **_tables(st), **_pool(cache)}
    if kind == "fork":
        ok = kv_pages.fork_kv_rows(st["parents"], *cache, st["table"], st["lengths"], st["refs"])
    else:
        kv_pages.free_kv_rows(st["keep"], st["table"], st["lengths"], st["refs"], block=case["block"])
        ok = kv_pages.reserve_kv_pages(*cache, st["table"], st["lengths"], st["counts"], st["refs"])
    return {"ok": ok, **_tables(st), **_pool(cache)}


def _tables(st):
    return {"table": st["table"], "refs": st["refs"], "lengths": st["lengths"]}


def _pool(cache):
    return {"k_codes": cache[0].view(torch.int8), "v_codes": cache[1].view(torch.int8), "k_scale": cache[2], "v_scale": cache[3]}


# ---------------------------------------------------------------------------------------------- plain forms
def _move(cache, src, dst):
    for x in cache:
        x = x.view(torch.int8) if x.element_size() == 1 else x
        x[:, dst.long()] = x[:, src.long()]


def _count(refs, entries, by):
    """refs plus `by` for every page among the entries."""
    some = entries[entries >= 0].long()
    return refs.index_add_(0, some, torch.full_like(some, by, dtype=torch.int32))


def _plain_copy(st):
    _move(st["cache"], st["src"], st["dst"])
    return _pool(st["cache"])


def _plain_fork(st):
    """A row that goes on from its parent shares its full pages. The open one stays with the parent's row if that goes on from
    itself, else with the first of those that go on from it, and is copied for the others to the lowest free pages."""
    table, lengths, refs, block = st["table"], st["lengths"], st["refs"], st["case"]["block"]
    parents = st["parents"].long()
    b, width = table.shape
    rows = torch.arange(b, device=table.device)
    first = torch.full((b,), b, device=table.device).scatter_reduce_(0, parents, rows, "amin")
    keeper = torch.where(parents[parents] == parents, parents, first[parents])
    n = lengths[parents]
    at = torch.arange(width, device=table.device)
    new = torch.where(at < -(-n // block)[:, None], table[parents], -1)
    open_at = (n // block).long().clamp(max=width - 1)[:, None]
    source = new.gather(1, open_at)[:, 0]
    copied = (keeper != rows) & (n % block != 0) & (source >= 0)
    new = torch.where((at == open_at) & copied[:, None], -1, new)
    stays = (parents == rows)[:, None]
    new = torch.where(stays, table, new)
    after = _count(_count(refs.clone(), table, -1), new, 1)
    free = (after == 0).nonzero()[:, 0]
    need = copied.cumsum(0)
    ok = need[-1] <= free.numel()
    page = free[(need - 1).clamp(0, free.numel() - 1)].to(torch.int32)
    new = torch.where((at == open_at) & copied[:, None], page[:, None], new)
    src, dst = source[copied & ok], page[copied & ok]
    _move(st["cache"], src, dst)
    after = _count(after, dst, 1)
    table.copy_(torch.where(ok, new, table))
    lengths.copy_(torch.where(ok, n, lengths))
    refs.copy_(torch.where(ok, after, refs))
    return {"ok": ok.to(torch.int32).view(1), **_tables(st), **_pool(st["cache"])}


def _plain_turn(st):
    """Pages behind the tokens that a row keeps go back; the blocks of a row's next tokens get the lowest free pages where they
    have none, and copies where others hold their page too."""
    table, lengths, refs, block = st["table"], st["lengths"], st["refs"], st["case"]["block"]
    keep, counts = st["keep"], st["counts"]
    at = torch.arange(table.shape[1], device=table.device)
    lengths.copy_(torch.minimum(lengths, keep))
    gone = at >= -(-keep // block)[:, None]
    _count(refs, torch.where(gone, table, -1), -1)
    table.masked_fill_(gone, -1)
    touched = (at >= (lengths // block)[:, None]) & (at < -(-(lengths + counts) // block)[:, None]) & (counts > 0)[:, None]
    need = touched & ((table < 0) | (refs[table.clamp_min(0).long()] > 1))
    free = (refs == 0).nonzero()[:, 0]
    rank = need.flatten().cumsum(0).view_as(need)
    ok = rank[-1, -1] <= free.numel()
    page = free[(rank - 1).clamp(0, free.numel() - 1)].to(torch.int32)
    need &= ok
    had = need & (table >= 0)
    _move(st["cache"], table[had], page[had])
    _count(_count(refs, table[had], -1), page[need], 1)
    table.copy_(torch.where(need, page, table))
    return {"ok": ok.to(torch.int32).view(1), **_tables(st), **_pool(st["cache"])}


def _plain_compact(st):
    """The pages in use behind the first `live` ones move into the free ones among those, in order."""
    table, refs = st["table"], st["refs"]
    used = refs > 0
    live = used.sum()
    ids = torch.arange(refs.numel(), device=refs.device)
    src, dst = (used & (ids >= live)).nonzero()[:, 0], (~used & (ids < live)).nonzero()[:, 0]
    moved = torch.where(used, ids, -1)
    moved[src] = dst
    _move(st["cache"], src, dst)
    refs[dst] = refs[src]
    refs[src] = 0
    table.copy_(torch.where(table >= 0, moved[table.clamp_min(0).long()].to(torch.int32), -1))
    return {"live": live.to(torch.int32).view(1), "moved": moved.to(torch.int32), **_tables(st), **_pool(st["cache"])}


def _plain_values(codes, scale, table, flip):
    """[b, hkv, tokens, d] fp32 values of the pages of a table."""
    at = table.clamp_min(0).long()
    c = codes.view(torch.int8)[at].view(codes.dtype).float() * scale[at][..., None, None]
    c = (c.transpose(-1, -2) if flip else c).transpose(1, 2)
    return c.reshape(c.shape[0], c.shape[1], -1, c.shape[-1])


def _plain_layer(q, layer, table, starts):
    b, t, h, d = q.shape
    hkv = layer[0].shape[1]
    k = _plain_values(layer[0], layer[2], table, False)
    v = _plain_values(layer[1], layer[3], table, True)
    qf = q.float().view(b, t, hkv, h // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d) / math.sqrt(d)
    s = (qf @ k.transpose(-1, -2).contiguous()).view(b, hkv, h // hkv, t, -1)
    seen = torch.arange(k.shape[2], device=q.device) <= (starts[:, None] + torch.arange(t, device=q.device))[..., None]
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    s -= s.amax(-1, keepdim=True)
    p = s.exp_()
    p /= p.sum(-1, keepdim=True)
    o = (p.view(b, hkv, -1, k.shape[2]) @ v).view(b, hkv, h // hkv, t, d)
    return o.permute(0, 3, 1, 2, 4).reshape(b, t, h, d).to(q.dtype)


def _plain_attend(st):
    return [_plain_layer(q, layer, st["table"], st["starts"]) for q, layer in zip(st["q"], zip(*st["cache"]))]


def _column(x, like):
    """A setting as a column of 64-bit numbers, one for each row."""
    x = x if isinstance(x, torch.Tensor) else torch.full((like.shape[0],), x, dtype=torch.float64, device=like.device)
    return x.double()[:, None]


def _plain_sample(st):
    """Tokens in the order of their logits, equal ones by their id: the first k, of these the shortest run that holds p of
    their weight, of these those with min_p of the first one's weight. The draw is the least id whose cumulative weight
    exceeds u times the total."""
    logits = st["logits"].float()
    b, v = logits.shape
    temp, k, p, minp = (_column(st[x], logits) for x in ("temp", "k", "p", "minp"))
    order = logits.sort(dim=-1, descending=True, stable=True)
    x, ids = order.values.double(), order.indices
    w = ((x - x[:, :1]) / torch.where(temp > 0, temp, 1.0)).exp()
    rank = torch.arange(v, device=w.device)
    w = torch.where((k < 1) | (rank < k), w, 0.0)
    c = w.cumsum(-1)
    kept = ((p >= 1) | (c - w < p * c[:, -1:])) & (w >= minp)
    w = torch.zeros_like(w).scatter_(1, ids, torch.where(kept, w, 0.0))
    c = w.cumsum(-1)
    over = c > _column(st["u"], logits) * c[:, -1:]
    last = v - 1 - (w > 0).flip(-1).int().argmax(-1)
    pick = torch.where(over.any(-1), over.int().argmax(-1), last)
    return torch.where(temp[:, 0] > 0, pick, ids[:, 0]).to(torch.int32)


# ---------------------------------------------------------------------------------------------- in 64 bits
def _exact_attend(case, st):
    """Row by row and head by head over the row's own keys."""
    h, hkv, d, block, t = (case[x] for x in ("h", "hkv", "d", "block", "t"))
    starts = st["starts"].tolist()
    outs = []
    for q, (kc, vc, ks, vs) in zip(st["q"], zip(*st["cache"])):
        out = torch.zeros(case["b"], t, h, d, dtype=torch.float64, device="cuda")
        for i, s0 in enumerate(starts):
            n = s0 + t
            pages = st["table"][i, :(n + block - 1) // block].long()
            late = torch.arange(n, device="cuda") > s0 + torch.arange(t, device="cuda")[:, None]
            for g in range(hkv):
                k = kc.view(torch.int8)[pages, g].view(kc.dtype).double() * ks[pages, g].double()[:, None, None]
                v = vc.view(torch.int8)[pages, g].view(vc.dtype).double().transpose(1, 2) * vs[pages, g].double()[:, None, None]
                heads = slice(g * (h // hkv), (g + 1) * (h // hkv))
                x = q[i, :, heads].double().transpose(0, 1).reshape(-1, d)
                s = torch.matmul(x, k.flatten(0, 1)[:n].t().contiguous()).view(-1, t, n) * d ** -0.5
                p = torch.softmax(s.masked_fill(late, -math.inf), -1)
                out[i, :, heads] = torch.matmul(p.view(-1, n), v.flatten(0, 1)[:n]).view(-1, t, d).transpose(0, 1)
        outs.append(out)
    return outs


def _exact_pages(case, st):
    """The scales after the pass, by lists on the host: pages are numbers in them, and every free page is looked for anew."""
    block = case["block"]
    scales = [x.double().cpu() for x in st["cache"][2:]]

    def put(src, dst):
        for x in scales:
            x[:, dst] = x[:, src].clone()

    if case["kind"] == "copy":
        for s, t in zip(st["src"].tolist(), st["dst"].tolist()):
            put(s, t)
        return scales
    table, lengths = st["table"].tolist(), st["lengths"].tolist()
    pages = st["refs"].numel()

    def held():
        return {p for row in table for p in row if p >= 0}

    if case["kind"] == "compact":
        live = sorted(held())
        holes = sorted(set(range(len(live))) - set(live))
        for s, t in zip([p for p in live if p >= len(live)], holes):
            put(s, t)
    elif case["kind"] == "fork":
        parents = st["parents"].tolist()
        old = [list(row) for row in table]
        waiting, taken = [], set()
        for i, p in enumerate(parents):
            n = lengths[p]
            table[i] = [x if j * block < n else -1 for j, x in enumerate(old[p])]
            if n % block and (i != p if parents[p] == p else p in taken):
                waiting.append((i, n // block, table[i][n // block]))
                table[i][n // block] = -1
            taken.add(p)
        free = sorted(set(range(pages)) - held())
        for (i, j, s), t in zip(waiting, free):
            put(s, t)
    else:
        keep, counts = st["keep"].tolist(), st["counts"].tolist()
        for row, n in zip(table, keep):
            row[:] = [x if j * block < n else -1 for j, x in enumerate(row)]
        many = {}
        for row in table:
            for p in row:
                many[p] = many.get(p, 0) + 1
        free = iter(sorted(set(range(pages)) - held()))
        for row, n, c in zip(table, keep, counts):
            for j in range(n // block, (n + c + block - 1) // block):
                if row[j] < 0 or many[row[j]] > 1:
                    to = next(free)
                    if row[j] >= 0:
                        put(row[j], to)
    return scales


def exact(case, seed):
    kind = case["kind"]
    if kind == "sample":
        return None
    st = prepare(case, seed)
    if kind == "attend":
        return _exact_attend(case, st)
    k_scale, v_scale = _exact_pages(case, st)
    return {"k_scale": k_scale, "v_scale": v_scale}
