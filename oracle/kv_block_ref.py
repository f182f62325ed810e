"""numpy statement of the block-scaled 8-bit KV cache, rotary positions and draft verification — TEST INFRASTRUCTURE ONLY.

Written from the operators' definitions (include/sqx.h), token by token and block by block, in float64 except where the
definition itself rounds to fp32 (scales, quotients). The reference has no counterpart; parity unpinned.
"""

from __future__ import annotations

import numpy as np

from oracle import fp8_ref

F32 = np.float32
MIN_SCALE = F32(1e-12)
QMAX = {"int8": F32(127.0), "e4m3": F32(448.0)}


def rope(x, positions, cos, sin, interleaved: bool) -> np.ndarray:
    """x [N, H, d] float64; positions [N]; cos, sin [P, rot / 2]. In float64, unrounded."""
    x = np.asarray(x, np.float64).copy()
    n, _, _ = x.shape
    half = cos.shape[1]
    for i in range(n):
        p = min(max(int(positions[i]), 0), cos.shape[0] - 1)
        c, s = cos[p].astype(np.float64), sin[p].astype(np.float64)
        ia = 2 * np.arange(half) if interleaved else np.arange(half)
        ib = ia + (1 if interleaved else half)
        a, b = x[i][:, ia].copy(), x[i][:, ib].copy()
        x[i][:, ia] = a * c - b * s
        x[i][:, ib] = a * s + b * c
    return x


def encode(x, s, fmt: str) -> np.ndarray:
    """fp32 values and their fp32 scale -> code bytes."""
    with np.errstate(all="ignore"):
        y = (np.asarray(x, F32) / F32(s)).astype(F32)
        if fmt == "e4m3":
            return fp8_ref.e4m3_encode_sat(y)
        r = np.clip(np.rint(y), -127, 127)
        return np.where(np.isnan(y), 0, r).astype(np.int8).view(np.uint8)


def decode(codes, fmt: str) -> np.ndarray:
    c = np.asarray(codes, np.uint8)
    return (fp8_ref.e4m3_decode(c) if fmt == "e4m3" else c.view(np.int8)).astype(np.float64)


def shrink(codes, k: int, fmt: str) -> np.ndarray:
    """Codes of values 2^k smaller."""
    c = np.asarray(codes, np.uint8)
    v = decode(c, fmt) * 2.0 ** -k
    if fmt == "int8":
        return np.rint(v).astype(np.int8).view(np.uint8)
    with np.errstate(invalid="ignore"):
        return np.where((c & 0x7F) == 0x7F, c, fp8_ref.e4m3_encode_sat(v.astype(F32)))


def write(k, v, kc, vc, ks, vs, table, starts, counts, fmt: str) -> None:
    """k, v [B, T, Hkv, D] fp32 values; kc [P, Hkv, block, D], vc [P, Hkv, D, block] uint8 and ks, vs [P, Hkv] fp32,
    updated in place."""
    pages, hkv, block, _ = kc.shape
    for b in range(k.shape[0]):
        if starts[b] < 0:
            continue
        n = min(max(int(counts[b]), 0), k.shape[1])
        t = 0
        while t < n:
            pos = int(starts[b]) + t
            lo, m = pos % block, min(block - pos % block, n - t)
            blk = pos // block
            page = int(table[b, blk]) if blk < table.shape[1] else -1
            if 0 <= page < pages:
                for h in range(hkv):
                    for x, codes, scale in ((k, kc[page, h], ks), (v, vc[page, h].T, vs)):
                        new = x[b, t:t + m, h].astype(F32)
                        a = np.abs(new[np.isfinite(new)])
                        most = a.max() if a.size else F32(0)
                        s = max(F32(most * (F32(1) / QMAX[fmt])), MIN_SCALE)
                        if lo:
                            had = max(scale[page, h], MIN_SCALE)
                            e = 0
                            while float(s) > float(had) * 2.0**e:
                                e += 1
                            s = F32(float(had) * 2.0**e)
                            if e:
                                codes[:lo] = shrink(codes[:lo], e, fmt)
                        scale[page, h] = s
                        codes[lo:lo + m] = encode(new, s, fmt)
            t += m


def read(kc, vc, ks, vs, table, starts, counts, tokens: int, fmt: str):
    """(k, v) [B, tokens, Hkv, D] as fp32(code) * scale in fp32."""
    pages, hkv, block, d = kc.shape
    out = np.zeros((2, table.shape[0], tokens, hkv, d), F32)
    for b in range(table.shape[0]):
        for t in range(min(max(int(counts[b]), 0), tokens)):
            pos = int(starts[b]) + t
            if starts[b] < 0 or pos // block >= table.shape[1]:
                continue
            page = int(table[b, pos // block])
            if not 0 <= page < pages:
                continue
            out[0, b, t] = decode(kc[page, :, pos % block], fmt).astype(F32) * ks[page][:, None]
            out[1, b, t] = decode(vc[page, :, :, pos % block], fmt).astype(F32) * vs[page][:, None]
    return out[0], out[1]


def attend(q, kc, vc, ks, vs, table, starts, counts, scale: float, fmt: str):
    """q [B, T, H, D] float64. Returns (out, terms): out [B, T, H, D] with NaN-free zeros where nothing is attended, and
    terms = (sum of p |v|, largest sum of |q k| scale, keys, largest |v|) per (b, t, h) for an error bound."""
    bsz, tq, h, d = q.shape
    pages, hkv, block, _ = kc.shape
    g = h // hkv
    out = np.zeros((bsz, tq, h, d))
    weight = np.zeros((bsz, tq, h, d))
    reach = np.zeros((bsz, tq, h))
    count = np.zeros((bsz, tq, h))
    vmax = np.zeros((bsz, tq, h))
    for b in range(bsz):
        for t in range(min(max(int(counts[b]), 0), tq)):
            n = min(int(starts[b]) + t + 1, table.shape[1] * block)
            if n <= 0:
                continue
            pos = np.arange(n)
            page = table[b, pos // block].astype(np.int64)
            bad = (page < 0) | (page >= pages)
            page = np.where(bad, 0, page)
            for hk in range(hkv):
                k = decode(kc[page, hk, pos % block], fmt) * ks[page, hk].astype(np.float64)[:, None]
                v = decode(vc[page, hk, :, pos % block], fmt) * vs[page, hk].astype(np.float64)[:, None]
                k[bad] = np.nan
                for x in range(hk * g, (hk + 1) * g):
                    s = k @ q[b, t, x] * scale
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    out[b, t, x] = p @ v
                    weight[b, t, x] = p @ np.abs(v)
                    reach[b, t, x] = (np.abs(k) @ np.abs(q[b, t, x])).max() * scale
                    count[b, t, x], vmax[b, t, x] = n, np.abs(v).max()
    return out, (weight, reach, count, vmax)


def verify(logits, draft, counts, probs, u, r, temperature: float):
    """logits [B, T + 1, V], probs [B, T, V] or None, in float64. Returns (n [B], tokens [B, T + 1])."""
    bsz, t1, vocab = logits.shape
    tokens = np.full((bsz, t1), -1, np.int32)
    n_acc = np.zeros(bsz, np.int32)

    def dist(row):
        m = row.max()
        if not np.isfinite(m):
            return None
        e = np.exp((row - m) / temperature)
        return e / e.sum()

    for b in range(bsz):
        n = min(max(int(counts[b]), 0), t1 - 1)
        t = 0
        while t < n:
            x = int(draft[b, t])
            if temperature == 0.0:
                if x != int(np.argmax(logits[b, t])):
                    break
            else:
                p = dist(logits[b, t])
                if p is None or not 0 <= x < vocab:
                    break
                qx = 1.0 if probs is None else float(probs[b, t, x])
                if not float(u[b, t]) * qx < p[x]:
                    break
            tokens[b, t] = x
            t += 1
        n_acc[b] = t
        if temperature == 0.0:
            tokens[b, t] = int(np.argmax(logits[b, t]))
            continue
        p = dist(logits[b, t])
        if p is None:
            continue
        w = p
        if t < n:
            q = np.zeros(vocab)
            if probs is not None:
                q = probs[b, t].astype(np.float64)
            elif 0 <= int(draft[b, t]) < vocab:
                q[int(draft[b, t])] = 1.0
            with np.errstate(invalid="ignore"):
                rest = np.where(p > q, p - q, 0.0)
            if rest.sum() > 0:
                w = rest
        c = np.cumsum(w)
        over = np.nonzero(c > float(r[b]) * c[-1])[0]
        tokens[b, t] = int(over[0]) if over.size else int(np.nonzero(w > 0)[0][-1])
    return n_acc, tokens
