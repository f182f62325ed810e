"""Serving over an 8-bit key/value cache with one scale per block of tokens and head, as timed cases.

Four operators in the order in which a serving step calls them: rotary positions (`rope`), the cache write with its
quantizer and the read back (`write`), attention of one or more new tokens per row over the cache (`attend`), and
the verification of drafted tokens (`verify`).

The cache of a layer is four tensors: codes of the keys [pages, Hkv, block, D] and of the values [pages, Hkv, D, block]
(int8, or E4M3), and fp32 scales [pages, Hkv] of each. A row's block table names the page of every `block` tokens;
pages lie in any order. Heads are those of Llama-3-8B (32 query, 8 key/value, 128 wide) and of generic models with
narrower and wider heads; the vocabularies are its 128256 and a generic 32000.

`own` is set by what imports this file: with it false `run` computes plain torch operations, with it true it calls
this package.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
QMAX = {"int8": 127.0, "e4m3": 448.0}
MIN_SCALE = 1e-12


def listed():
    return [
        # one decoded token's query and key heads: launch latency and host cost
        {"name": "rope_token", "kind": "rope", "n": 1, "heads": 40, "d": 128, "rot": 128, "interleaved": True, "far": 0,
         "dtype": "bf16"},
        # a chunk of long-context prompt, half of each head rotated, positions past a hundred thousand
        {"name": "rope_prompt", "kind": "rope", "n": 8191, "heads": 40, "d": 128, "rot": 64, "interleaved": False,
         "far": 120000, "dtype": "fp16"},
        # eight streams append the token that they decoded, rotary included
        {"name": "write_token", "kind": "write", "b": 8, "t": 1, "h": 32, "hkv": 8, "d": 128, "block": 64, "fmt": "int8",
         "dtype": "bf16", "start": 1021, "rot": 128, "interleaved": True},
        # ragged prompt chunks of a model with 64-wide heads, appended in the middle of a block
        {"name": "write_chunk", "kind": "write", "b": 5, "t": 300, "h": 12, "hkv": 12, "d": 64, "block": 16, "fmt": "e4m3",
         "dtype": "fp16", "start": 700, "rot": 32, "interleaved": False},
        # a batch of prompts enters the cache
        {"name": "write_prompt", "kind": "write", "b": 8, "t": 2048, "h": 32, "hkv": 8, "d": 128, "block": 64, "fmt": "int8",
         "dtype": "bf16", "start": 0, "rot": 128, "interleaved": True},
        # one stream decodes at the context of the benchmark's decode step
        {"name": "attend_token", "kind": "attend", "b": 1, "t": 1, "h": 32, "hkv": 8, "d": 128, "block": 64, "fmt": "int8",
         "dtype": "bf16", "ctx": 2048},
        # a full batch decodes, contexts of uneven lengths
        {"name": "attend_batch", "kind": "attend", "b": 64, "t": 1, "h": 32, "hkv": 8, "d": 128, "block": 64, "fmt": "int8",
         "dtype": "bf16", "ctx": 8192},
        # drafted tokens of sixteen streams checked in one pass
        {"name": "attend_draft", "kind": "attend", "b": 16, "t": 5, "h": 32, "hkv": 8, "d": 128, "block": 32, "fmt": "e4m3",
         "dtype": "bf16", "ctx": 16000},
        # decoding far into very long contexts: the largest cache (over 2^31 bytes of keys)
        {"name": "attend_long", "kind": "attend", "b": 3, "t": 1, "h": 32, "hkv": 8, "d": 128, "block": 128, "fmt": "int8",
         "dtype": "bf16", "ctx": 800001},
        # a chunk of prompt attends what came before it and itself
        {"name": "attend_prompt", "kind": "attend", "b": 2, "t": 2048, "h": 32, "hkv": 8, "d": 128, "block": 64,
         "fmt": "int8", "dtype": "bf16", "ctx": 6000},
        # one stream's drafted tokens against a small vocabulary, proposed without probabilities (prompt lookup)
        {"name": "verify_lookup", "kind": "verify", "b": 1, "t": 4, "v": 32000, "dtype": "fp32", "probs": False, "temp": 0.8},
        # a batch's drafted tokens with the draft model's probabilities
        {"name": "verify_batch", "kind": "verify", "b": 64, "t": 5, "v": 128256, "dtype": "bf16", "probs": True, "temp": 1.0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["rope", "write", "write", "attend", "attend", "attend", "verify"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    d = rng.choice([64, 128, 128, 256])
    fmt = rng.choice(["int8", "e4m3"])
    block = rng.choice([16, 32, 64, 128])
    hkv = rng.choice([1, 2, 4, 8, 12])
    group = rng.choice([1, 2, 3, 4, 6, 8, 16])
    if kind == "rope":
        return {"kind": kind, "n": _log_int(rng, 1, 8000), "heads": _log_int(rng, 1, 48), "d": d,
                "rot": rng.choice([d, d // 2, d // 4]), "interleaved": rng.random() < 0.5, "far": rng.choice([0, 4000, 100000]),
                "dtype": dtype}
    if kind == "write":
        t = _log_int(rng, 1, 1500)
        return {"kind": kind, "b": _log_int(rng, 1, max(1, min(64, 12000 // t))), "t": t, "h": hkv * rng.choice([1, 2, 4]),
                "hkv": hkv, "d": min(d, 128), "block": block, "fmt": fmt, "dtype": dtype, "start": rng.randrange(0, 3000),
                "rot": rng.choice([min(d, 128), 32]), "interleaved": rng.random() < 0.5}
    if kind == "attend":
        t = rng.choice([1, 1, 1, _log_int(rng, 2, 8), _log_int(rng, 9, 1024)])
        ctx = t + _log_int(rng, 1, 4000 if t > 8 else 60000)
        b = _log_int(rng, 1, max(1, min(48, 2000 // t, 400000 // ctx)))
        if t > 8:  # prompts of wide models would cost more than any listed case
            group = min(group, max(1, 32 // hkv))
        return {"kind": kind, "b": b, "t": t, "h": hkv * group, "hkv": hkv, "d": d, "block": block, "fmt": fmt,
                "dtype": dtype, "ctx": ctx}
    return {"kind": kind, "b": _log_int(rng, 1, 48), "t": rng.randrange(1, 8), "v": _log_int(rng, 500, 128256),
            "dtype": rng.choice(["bf16", "fp32", "fp16"]), "probs": rng.random() < 0.7, "temp": rng.choice([0.0, 0.6, 1.0, 1.3])}


# ---------------------------------------------------------------------------------------------- sizes of a case
def _spread(b, most, part):
    """Lengths of b rows: the first the longest, the others down to 1 - part of it, unevenly."""
    return [most - (i * 7919) % (int(most * part) + 1) for i in range(b)]


def _rows(case):
    """(starts, counts) of a `write` or `attend` case: tokens before the row's new ones, and how many are new."""
    b, t = case["b"], case["t"]
    counts = _spread(b, t, 0.5 if t > 16 else 0.0)
    if case["kind"] == "write":
        return [case["start"] + (i * 13 if case["start"] else 0) for i in range(b)], counts
    return [max(0, n - t) for n in _spread(b, case["ctx"], 0.5)], counts


def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "rope":
        n, heads, d, rot = case["n"], case["heads"], case["d"], case["rot"]
        return {"bytes": n * (2 * heads * d * es + rot * 4), "flops": 3 * n * heads * rot}
    if case["kind"] == "verify":
        b, t, v = case["b"], case["t"], case["v"]
        return {"bytes": b * v * ((t + 1) * es + (4 if case["probs"] else 0)), "flops": 4 * b * (t + 1) * v}
    starts, counts = _rows(case)
    h, hkv, d = case["h"], case["hkv"], case["d"]
    if case["kind"] == "write":
        n = sum(counts)
        back = sum(s % case["block"] + c for s, c in zip(starts, counts))
        return {"bytes": n * ((2 * h + 2 * hkv) * d * es + 2 * hkv * d) + back * 2 * hkv * d * 3,
                "flops": n * (3 * (h + hkv) * case["rot"] + 4 * hkv * d)}
    keys = sum(s + c for s, c in zip(starts, counts))
    pairs = sum(c * s + c * (c + 1) // 2 for s, c in zip(starts, counts))
    return {"bytes": 2 * sum(counts) * h * d * es + keys * 2 * hkv * d + 8 * hkv * (keys // case["block"] + case["b"]),
            "flops": 4 * h * d * pairs}


# ---------------------------------------------------------------------------------------------- inputs
def _tables(rot, rows, device):
    """cos and sin [rows, rot/2] of the angles position * 10000^(-2i/rot), in 64 bits, rounded once to 32."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    ang = torch.outer(torch.arange(rows, dtype=torch.float64, device=device), inv)
    return ang.cos().float(), ang.sin().float()


def _to_codes(y, fmt):
    """Values in units of their scale as 8-bit codes, in pieces (a long cache does not fit in 32 bits twice)."""
    lim = QMAX[fmt]
    y = y.clamp_(-lim, lim)
    return y.round_().to(torch.int8) if fmt == "int8" else y.to(torch.float8_e4m3fn)


def _cache(gen, pages, hkv, block, d, fmt, dev):
    """A filled cache: codes as a quantizer leaves them for normal keys and values, scales that vary from page to page."""
    spread = QMAX[fmt] / 3.6  # the largest of a block lies near 3.6 standard deviations
    codes = []
    for shape in ((pages, hkv, block, d), (pages, hkv, d, block)):
        out = torch.empty(shape, dtype=CODES[fmt], device=dev)
        step = max(1, (1 << 28) // (hkv * block * d))
        for i in range(0, pages, step):
            y = torch.randn(out[i:i + step].shape, generator=gen, device=dev) * spread
            out[i:i + step] = _to_codes(y, fmt)
        codes.append(out)
    scales = [torch.exp(0.4 * torch.randn(pages, hkv, generator=gen, device=dev)) / spread for _ in range(2)]
    return codes[0], codes[1], scales[0], scales[1]


def _table(gen, b, blocks, dev):
    """Each row's pages, scattered over the cache as a server's allocator leaves them."""
    order = torch.randperm(b * blocks, generator=gen, device=dev)
    return order.to(torch.int32).view(b, blocks).contiguous()


def _int32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    st = {"case": case}
    if case["kind"] == "rope":
        n, rot = case["n"], case["rot"]
        st["x"] = torch.randn(n, case["heads"], case["d"], generator=gen, device=dev).to(dt)
        st["cos"], st["sin"] = _tables(rot, n + case["far"] + 64, dev)
        st["pos"] = (torch.arange(n, device=dev) + case["far"] + seed % 61).to(torch.int32)
        return st
    if case["kind"] == "verify":
        b, t, v = case["b"], case["t"], case["v"]
        base = 3.0 * torch.randn(b, t + 1, v, generator=gen, device=dev)
        st["logits"] = base.to(dt)
        # the draft model: near the target, so that most of its tokens are accepted
        q = torch.softmax(base[:, :t] + 0.4 * torch.randn(b, t, v, generator=gen, device=dev), -1)
        draft = torch.multinomial(q.view(b * t, v), 1, generator=gen).view(b, t).to(torch.int32)
        likely = st["logits"][:, :t].argmax(-1).to(torch.int32)
        st["draft"] = torch.where(torch.rand(b, t, generator=gen, device=dev) < (0.3 if case["probs"] else 0.7), likely, draft)
        st["probs"] = q if case["probs"] else None
        st["u"] = torch.rand(b, t, generator=gen, device=dev)
        st["r"] = torch.rand(b, generator=gen, device=dev)
        return st
    starts, counts = _rows(case)
    b, t, h, hkv, d, block = (case[x] for x in ("b", "t", "h", "hkv", "d", "block"))
    blocks = max((s + c + block - 1) // block for s, c in zip(starts, counts))
    st["k_codes"], st["v_codes"], st["k_scale"], st["v_scale"] = _cache(gen, b * blocks, hkv, block, d, case["fmt"], dev)
    st["table"] = _table(gen, b, blocks, dev)
    st["starts"], st["counts"] = _int32(starts, dev), _int32(counts, dev)
    if case["kind"] == "write":
        # the fused projection's rows [q | k | v], keys with a few loud channels
        qkv = torch.randn(b, t, h + 2 * hkv, d, generator=gen, device=dev)
        qkv[:, :, h:h + hkv, 5::d // 2] *= 6.0
        qkv = qkv.to(dt)
        st["q"], st["k"], st["v"] = qkv[:, :, :h], qkv[:, :, h:h + hkv], qkv[:, :, h + hkv:]
        st["cos"], st["sin"] = _tables(case["rot"], max(starts) + t + 8, dev)
        # what is read back: the row's first open block and everything written after it
        st["back"] = _int32([s - s % block for s in starts], dev)
        st["n_back"] = _int32([s % block + c for s, c in zip(starts, counts)], dev)
        st["most_back"] = max(s % block + c for s, c in zip(starts, counts))
        return st
    st["q"] = torch.randn(b, t, h, d, generator=gen, device=dev).to(dt)
    st["out"] = torch.zeros(b, t, h, d, dtype=dt, device=dev)
    return st


# ---------------------------------------------------------------------------------------------- one pass
def run(st):
    kind = st["case"]["kind"]
    if own:
        return _own(st, kind)
    return {"rope": _plain_rope, "write": _plain_write, "attend": _plain_attend, "verify": _plain_verify}[kind](st)


def _own(st, kind):
    from scratch_llm_amd import rope, speculative
    from scratch_llm_amd.quant import kv_block

    case = st["case"]
    if kind == "rope":
        return rope.apply_rope(st["x"], st["pos"], st["cos"], st["sin"], interleaved=case["interleaved"])
    if kind == "verify":
        return speculative.verify_draft(st["logits"], st["draft"], st["u"], st["r"], draft_probs=st["probs"],
                                        temperature=case["temp"])
    cache = (st["k_codes"], st["v_codes"], st["k_scale"], st["v_scale"])
    if kind == "write":
        q = kv_block.write_kv_blocks(st["k"], st["v"], *cache, st["table"], st["starts"], st["counts"], q=st["q"],
                                     rope=(st["cos"], st["sin"]), interleaved=case["interleaved"])
        k, v = kv_block.read_kv_blocks(*cache, st["table"], st["back"], st["most_back"], st["n_back"],
                                       dtype=DTYPES[case["dtype"]])
        return q, k, v
    return kv_block.attend_kv_blocks(st["q"], *cache, st["table"], st["starts"], st["counts"], out=st["out"])


# ---------------------------------------------------------------------------------------------- plain forms
def _plain_rotate(x, cos, sin, interleaved):
    """x [..., heads, d] with cos, sin [..., 1, rot/2]: fp32 products and sums, rounded once to x's type."""
    half = cos.shape[-1]
    f = x.float()
    rot, rest = f[..., :2 * half], f[..., 2 * half:]
    a, b = (rot[..., 0::2], rot[..., 1::2]) if interleaved else (rot[..., :half], rot[..., half:])
    ra, rb = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((ra, rb), -1).flatten(-2) if interleaved else torch.cat((ra, rb), -1)
    return torch.cat((turned, rest), -1).to(x.dtype)


def _plain_rope(st):
    pos = st["pos"].long()
    return _plain_rotate(st["x"], st["cos"][pos][:, None], st["sin"][pos][:, None], st["case"]["interleaved"])


def _plain_blocks(x, codes, scale, pages, off, fresh, keep, fmt):
    """Codes and scales of the touched blocks. x [b, j, block, hkv, d] new values (0 where none), `keep` [b, j, block]
    where they are; codes [b, j, hkv, block, d] what the pages hold, of which the first `off` tokens of a row's first
    block stay; fresh [b, j] blocks that hold no earlier token."""
    x = x.float().permute(0, 1, 3, 2, 4)
    old = codes.float()
    most = torch.where(x.isfinite(), x.abs(), 0.0).amax((-1, -2))
    need = (most / QMAX[fmt]).clamp_min(MIN_SCALE)
    has = scale[pages.long()]
    mn, en = torch.frexp(need)
    mh, eh = torch.frexp(has)
    grow = (en - eh + (mn > mh).int()).clamp_min(0)
    s = torch.where(fresh[..., None], need, torch.ldexp(has, grow))
    down = torch.ldexp(torch.ones_like(s), -grow)[..., None, None]
    lim = QMAX[fmt]
    moved, new = old * down, (x / s[..., None, None]).clamp(-lim, lim)
    if fmt == "int8":
        moved, new = moved.round(), new.round()
    else:
        moved, new = (y.to(torch.float8_e4m3fn).float() for y in (moved, new))
    stay = (torch.arange(keep.shape[2], device=x.device) < off[:, None, None]) & ~fresh[..., None]
    kept, put = stay[:, :, None, :, None], keep[:, :, None, :, None]
    return torch.where(put, new, torch.where(kept, moved, old)), s


def _plain_write(st):
    case, block = st["case"], st["case"]["block"]
    starts, counts = st["starts"].long(), st["counts"].long()
    b, t, hkv, d = st["k"].shape
    dev = starts.device
    pos = starts[:, None] + torch.arange(t, device=dev)
    cos, sin = (st[x][pos.clamp(max=st[x].shape[0] - 1)][:, :, None] for x in ("cos", "sin"))
    q = _plain_rotate(st["q"], cos, sin, case["interleaved"])
    k = _plain_rotate(st["k"], cos, sin, case["interleaved"])
    off = starts % block
    nj = (t + 2 * block - 2) // block  # most blocks that t tokens can touch
    live = torch.arange(t, device=dev) < counts[:, None]
    slot = (off[:, None] + torch.arange(t, device=dev)).clamp(max=nj * block - 1)
    keep = torch.zeros(b, nj * block + 1, dtype=torch.bool, device=dev)
    keep.scatter_(1, torch.where(live, slot, nj * block), True)
    keep = keep[:, :-1].view(b, nj, block)
    touched = keep.any(-1)
    first = (starts // block)[:, None] + torch.arange(nj, device=dev)
    pages = st["table"].gather(1, first.clamp(max=st["table"].shape[1] - 1))
    fresh = (torch.arange(nj, device=dev) > 0) | (off[:, None] == 0)
    for x, codes, scale, flip in ((k, st["k_codes"], st["k_scale"], False), (st["v"], st["v_codes"], st["v_scale"], True)):
        wide = torch.zeros(b, nj * block + 1, hkv, d, dtype=x.dtype, device=dev)
        at = torch.where(live, slot, nj * block)[:, :, None, None].expand(b, t, hkv, d)
        wide.scatter_(1, at, x)
        wide = wide[:, :-1].view(b, nj, block, hkv, d)
        held = codes.view(torch.uint8)[pages.long()].view(codes.dtype)
        held = held.transpose(-1, -2) if flip else held
        new, s = _plain_blocks(wide, held, scale, pages, off, fresh, keep, case["fmt"])
        new = new.transpose(-1, -2) if flip else new
        where = pages.long()[touched]
        codes.view(torch.uint8)[where] = new.to(codes.dtype).view(torch.uint8)[touched]
        scale[where] = s[touched]
    back, n = st["back"].long(), st["n_back"].long()
    steps = torch.arange(st["most_back"], device=dev)
    at = back[:, None] + steps
    page = st["table"].gather(1, (at // block).clamp(max=st["table"].shape[1] - 1)).long()
    some = (steps < n[:, None])[:, :, None, None]
    outs = [q]
    for codes, scale, flip in ((st["k_codes"], st["k_scale"], False), (st["v_codes"], st["v_scale"], True)):
        flat = codes.view(torch.uint8).transpose(-1, -2) if flip else codes.view(torch.uint8)
        c = flat[page, :, at % block].contiguous().view(codes.dtype).float()
        outs.append(torch.where(some, c * scale[page][..., None], 0.0).to(q.dtype))
    return tuple(outs)


def _plain_cache(codes, scale, table, flip):
    """[b, hkv, tokens, d] fp32 values of the pages of a table."""
    c = codes.view(torch.uint8)[table.long()].view(codes.dtype).float() * scale[table.long()][..., None, None]
    c = (c.transpose(-1, -2) if flip else c).transpose(1, 2)
    return c.reshape(c.shape[0], c.shape[1], -1, c.shape[-1])


def _plain_attend(st):
    q = st["q"]
    b, t, h, d = q.shape
    hkv = st["k_codes"].shape[1]
    k = _plain_cache(st["k_codes"], st["k_scale"], st["table"], False)
    v = _plain_cache(st["v_codes"], st["v_scale"], st["table"], True)
    qf = q.float().view(b, t, hkv, h // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d) / math.sqrt(d)
    s = (qf @ k.transpose(-1, -2).contiguous()).view(b, hkv, h // hkv, t, -1)
    pos = st["starts"].long()[:, None] + torch.arange(t, device=q.device)
    seen = torch.arange(k.shape[2], device=q.device) <= pos[..., None]
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    s -= s.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p = s.exp_()
    p /= p.sum(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).tiny)
    o = (p.view(b, hkv, -1, k.shape[2]) @ v).view(b, hkv, h // hkv, t, d).permute(0, 3, 1, 2, 4).reshape(b, t, h, d)
    live = (torch.arange(t, device=q.device) < st["counts"][:, None])[..., None, None]
    st["out"].copy_(torch.where(live, o.to(q.dtype), st["out"]))
    return st["out"]


def _plain_verify(st):
    logits, draft, q = st["logits"], st["draft"].long(), st["probs"]
    b, t = draft.shape
    v = logits.shape[2]
    temp = st["case"]["temp"]
    if temp == 0.0:
        best = logits.argmax(-1)
        good = draft == best[:, :t]
        n = good.int().cumprod(1).sum(1)
        pick = best.gather(1, n[:, None])[:, 0]
    else:
        z = logits.double() / temp
        p = (z - z.amax(-1, keepdim=True)).exp_()
        p /= p.sum(-1, keepdim=True)
        px = p[:, :t].gather(2, draft[..., None])[..., 0]
        qx = torch.ones_like(px) if q is None else q.gather(2, draft[..., None])[..., 0].double()
        good = st["u"].double() * qx < px
        n = good.int().cumprod(1).sum(1)
        w = p[torch.arange(b, device=p.device), n]
        row = n.clamp(max=t - 1)
        if q is None:
            spot = draft.gather(1, row[:, None])
            prop = torch.zeros_like(w).scatter_(1, spot, 1.0)
        else:
            prop = q[torch.arange(b, device=p.device), row].double()
        rest = torch.where(w > prop, w - prop, 0.0)
        use = (n < t)[:, None] & (rest.sum(-1, keepdim=True) > 0)
        w = torch.where(use, rest, w)
        c = w.cumsum(-1)
        over = c > st["r"].double()[:, None] * c[:, -1:]
        last = v - 1 - (w > 0).flip(-1).int().argmax(-1)
        pick = torch.where(over.any(-1), over.int().argmax(-1), last)
    step = torch.arange(t + 1, device=draft.device)
    wide = torch.cat((draft, draft[:, :1]), 1)
    tokens = torch.where(step < n[:, None], wide, torch.where(step == n[:, None], pick[:, None], -1))
    return n.to(torch.int32), tokens.to(torch.int32)


# ---------------------------------------------------------------------------------------------- in 64 bits
def _turn64(x, cos, sin, interleaved):
    """The rotation as a complex product, in 64 bits."""
    x64 = x.double()
    r = cos.shape[-1]
    pairs = x64[..., :2 * r].unflatten(-1, (r, 2)) if interleaved else x64[..., :2 * r].unflatten(-1, (2, r)).transpose(-1, -2)
    z = torch.view_as_complex(pairs.contiguous()) * torch.complex(cos.double(), sin.double())
    y = torch.view_as_real(z)
    y = (y if interleaved else y.transpose(-1, -2)).flatten(-2)
    return torch.cat((y, x64[..., 2 * r:]), -1)


def _exact_write(case, st):
    """Row by row and block by block: what the pages hold after the write, as values."""
    block, fmt, lim = case["block"], case["fmt"], QMAX[case["fmt"]]
    dt = DTYPES[case["dtype"]]
    starts, counts = _rows(case)
    most = st["most_back"]
    hkv, d = case["hkv"], case["d"]
    pos = (torch.tensor(starts, device="cuda")[:, None] + torch.arange(case["t"], device="cuda")).clamp(max=st["cos"].shape[0] - 1)
    cos, sin = st["cos"][pos][:, :, None], st["sin"][pos][:, :, None]
    q = _turn64(st["q"], cos, sin, case["interleaved"])
    k = _turn64(st["k"], cos, sin, case["interleaved"]).to(dt)
    result = [q]

    def to_code(y):
        y = y.clamp(-lim, lim)
        return y.round() if fmt == "int8" else y.float().to(torch.float8_e4m3fn).double()

    for x, codes, scale, flip in ((k, st["k_codes"], st["k_scale"], False), (st["v"], st["v_codes"], st["v_scale"], True)):
        out = torch.zeros(case["b"], most, hkv, d, dtype=torch.float64, device="cuda")
        for i, (s0, c) in enumerate(zip(starts, counts)):
            done = 0
            while done < c:
                at, j = (s0 + done) % block, (s0 + done) // block
                n = min(block - at, c - done)
                new = x[i, done:done + n].double()  # [n, hkv, d]
                need = (new.abs().amax((0, 2)).float() / lim).clamp_min(MIN_SCALE).double()
                lo = (s0 + done) - (s0 - s0 % block)
                if at:
                    page = int(st["table"][i, j])
                    had = codes[page].transpose(-1, -2) if flip else codes[page]
                    before = scale[page].double()
                    up = torch.exp2(torch.ceil(torch.log2(need / before)).clamp_min(0))
                    s = before * up
                    old = to_code(had[:, :at].double() / up[:, None, None]) * s[:, None, None]
                    out[i, lo - at:lo] = old.transpose(0, 1)
                else:
                    s = need
                out[i, lo:lo + n] = to_code((new / s[:, None]).float().double()) * s[:, None]
                done += n
        result.append(out)
    return tuple(result)


def _exact_attend(case, st):
    """Row by row and head by head over the row's own keys."""
    starts, counts = _rows(case)
    h, hkv, d, block = case["h"], case["hkv"], case["d"], case["block"]
    out = torch.zeros(case["b"], case["t"], h, d, dtype=torch.float64, device="cuda")
    for i, (s0, c) in enumerate(zip(starts, counts)):
        n = s0 + c
        pages = st["table"][i, :(n + block - 1) // block].long()
        for g in range(hkv):
            k = st["k_codes"].view(torch.uint8)[pages, g].view(st["k_codes"].dtype).double()
            k = (k * st["k_scale"][pages, g].double()[:, None, None]).flatten(0, 1)[:n]
            v = st["v_codes"].view(torch.uint8)[pages, g].view(st["v_codes"].dtype).double().transpose(1, 2)
            v = (v * st["v_scale"][pages, g].double()[:, None, None]).flatten(0, 1)[:n]
            heads = slice(g * (h // hkv), (g + 1) * (h // hkv))
            q = st["q"][i, :c, heads].double().transpose(0, 1)  # [group, c, d]
            s = torch.matmul(q.reshape(-1, d), k.t().contiguous()).view(-1, c, n) * d ** -0.5
            late = torch.arange(n, device="cuda") > s0 + torch.arange(c, device="cuda")[:, None]
            p = torch.softmax(s.masked_fill(late, -math.inf), -1)
            out[i, :c, heads] = torch.matmul(p.view(-1, n), v).view(-1, c, d).transpose(0, 1)
    return out


def exact(case, seed):
    if case["kind"] == "verify":
        return None
    st = prepare(case, seed)
    if case["kind"] == "rope":
        pos = st["pos"].long()
        return _turn64(st["x"], st["cos"][pos][:, None], st["sin"][pos][:, None], case["interleaved"])
    return _exact_write(case, st) if case["kind"] == "write" else _exact_attend(case, st)
