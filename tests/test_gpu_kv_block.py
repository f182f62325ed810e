"""The block-scaled 8-bit KV cache (scratch_llm_amd/quant/kv_block.py) on the GPU against oracle/kv_block_ref.py.

Codes, scales and values read back are compared bit for bit: the definition fixes every rounding. Attention is compared
in float64 with a bound made of: the output's rounding (half a step of its type); the probabilities' rounding to fp16
(2^-11 of each, so of sum p |v|; a probability below 2^-29 of the largest term may be lost, 2^-28 |v|max a key counts both
its sides); and fp32 sums and scores (D + 8 roundings of 2^-24 in a score of at most `reach`, twice, as p enters numerator
and denominator; 2^-18 for the exponential, the logarithm of the scale and the sums)."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import kv_block_ref as R
from tests.conftest import print_case

pytestmark = pytest.mark.gpu
DEV = "cuda"
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def kv():
    from scratch_llm_amd.quant import kv_block

    return kv_block


def make_cache(kv, pages, hkv, d, block, fmt, seed):
    """A cache of random bytes (every code, for E4M3 the NaNs too) and scales, on both sides."""
    g = np.random.default_rng(seed)
    kc = g.integers(0, 256, (pages, hkv, block, d), dtype=np.uint8)
    vc = g.integers(0, 256, (pages, hkv, d, block), dtype=np.uint8)
    ks, vs = (np.exp(g.normal(-4, 0.7, (pages, hkv))).astype(np.float32) for _ in range(2))
    return [kc, vc, ks, vs]


def fill_valid(cache, fmt, seed):
    """The same cache with codes that a quantizer leaves (no NaN, int8 without -128)."""
    g = np.random.default_rng(seed)
    for i in range(2):
        y = g.normal(0, 35.0 if fmt == "int8" else 120.0, cache[i].shape)
        cache[i][...] = R.encode(y.astype(np.float32), 1.0, fmt)
    return cache


def to_dev(cache, fmt):
    kc, vc, ks, vs = cache
    return [torch.from_numpy(kc.copy()).to(DEV).view(CODES[fmt]), torch.from_numpy(vc.copy()).to(DEV).view(CODES[fmt]),
            torch.from_numpy(ks.copy()).to(DEV), torch.from_numpy(vs.copy()).to(DEV)]


def back(dev):
    return [dev[0].view(torch.uint8).cpu().numpy(), dev[1].view(torch.uint8).cpu().numpy(), dev[2].cpu().numpy(),
            dev[3].cpu().numpy()]


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def same_bytes(got, want, what):
    for a, b, name in zip(got, want, ("k codes", "v codes", "k scale", "v scale")):
        bad = np.argwhere(a != b)
        assert bad.size == 0, f"{what}: {name} differs at {bad[:3].tolist()}: {a[tuple(bad[0])]} for {b[tuple(bad[0])]}"


# (B, T, Hkv, D, block, starts, counts): single tokens at every kind of slot, blocks begun and finished, whole prompts,
# rows with nothing, a negative start, positions past the table
WRITES = [
    (1, 1, 1, 64, 16, [0], None),
    (3, 1, 2, 128, 64, [0, 63, 64], None),
    (4, 1, 8, 128, 32, [31, 32, 33, 5], [1, 0, 1, 1]),
    (2, 5, 3, 64, 16, [14, 0], [5, 3]),
    (3, 70, 2, 128, 64, [1, 60, 64], [70, 5, 64]),
    (2, 300, 1, 128, 128, [100, 0], [300, 129]),
    (2, 40, 2, 256, 32, [9, 33], [40, 31]),
    (2, 130, 1, 256, 128, [127, -1], None),
    (3, 33, 1, 64, 32, [95, 200, 130], [33, 33, 0]),  # the table ends at 128
]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("case", range(len(WRITES)))
def test_write_is_exact(kv, case, dtype, fmt):
    b, t, hkv, d, block, starts, counts = WRITES[case]
    print_case("kv write", case, dtype, fmt)
    width = 4 if case == 8 else max(max(starts) + t, 1) // block + 1
    pages = b * width + 2
    cache = make_cache(kv, pages, hkv, d, block, fmt, case)
    g = torch.Generator().manual_seed(100 + case)
    k, v = (torch.randn(b, t, hkv, d, generator=g) * torch.exp(torch.randn(b, t, hkv, 1, generator=g)) for _ in range(2))
    k, v = k.to(DT[dtype]), v.to(DT[dtype])
    table = np.random.default_rng(case).permutation(pages)[:b * width].reshape(b, width).astype(np.int32)
    dev = to_dev(cache, fmt)
    kv.write_kv_blocks(k.to(DEV), v.to(DEV), *dev, i32(table), i32(starts), None if counts is None else i32(counts))
    torch.cuda.synchronize()
    R.write(k.float().numpy(), v.float().numpy(), *cache, table, starts, counts or [t] * b, fmt)
    same_bytes(back(dev), cache, f"write {case}")


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_blocks_grow_token_by_token(kv, fmt):
    """Tokens of rising and falling magnitude one at a time: codes and scales stay the definition's, and every token is
    within what its comment promises: half a step at its write and less than a step of the final scale in all."""
    block, d, n = 32, 64, 75
    cache = make_cache(kv, 4, 1, d, block, fmt, 1)
    dev = to_dev(cache, fmt)
    table = np.array([[2, 0, 3]], np.int32)
    g = torch.Generator().manual_seed(2)
    mag = torch.exp(torch.randn(n, generator=g) * 1.5 + torch.linspace(-3, 3, n))
    x = torch.randn(2, 1, n, 1, d, generator=g) * mag.view(1, 1, n, 1, 1)
    x[0, 0, 40] = 0.0
    x[1, 0, 64] = 0.0  # a block that begins with zeros
    x = x.to(torch.bfloat16)
    for t in range(n):
        kv.write_kv_blocks(x[0, :, t:t + 1].to(DEV), x[1, :, t:t + 1].to(DEV), *dev, i32(table), i32([t]))
        R.write(x[0, :, t:t + 1].float().numpy(), x[1, :, t:t + 1].float().numpy(), *cache, table, [t], [1], fmt)
    same_bytes(back(dev), cache, "growth")
    got = kv.read_kv_blocks(*dev, i32(table), i32([0]), n)
    for i, (y, sc) in enumerate(zip(got, (cache[2], cache[3]))):
        step = np.repeat(sc[table[0], 0], block)[:n, None]
        err = np.abs(y[0, :, 0].cpu().numpy() - x[i, 0, :, 0].float().numpy())
        if fmt == "int8":
            assert (err <= step * (1 + 1e-5)).all()
        else:  # half a step of 3 mantissa bits, and of the subnormals' 2^-9 after each rescale: less than 2^-9 in all
            assert (err <= np.abs(x[i, 0, :, 0].float().numpy()) * 2.0**-4 + step * 2.0**-9 * (1 + 1e-5)).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_special_values(kv, fmt):
    """Infinities saturate, a NaN stays one in E4M3 and is 0 in int8, neither moves the scale; zeros take the floor."""
    cache = make_cache(kv, 2, 1, 64, 16, fmt, 3)
    dev = to_dev(cache, fmt)
    x = torch.randn(2, 1, 20, 1, 64, generator=torch.Generator().manual_seed(4))
    x[:, 0, 3, 0, :3] = torch.tensor([math.inf, -math.inf, math.nan])
    x[:, 0, 16:] = 0.0
    x[0, 0, 5] = math.nan
    table = np.array([[1, 0]], np.int32)
    kv.write_kv_blocks(x[0].to(DEV), x[1].to(DEV), *dev, i32(table), i32([0]))
    R.write(x[0].numpy(), x[1].numpy(), *cache, table, [0], [20], fmt)
    same_bytes(back(dev), cache, "special values")
    assert cache[2][0, 0] == np.float32(1e-12)
    assert np.isfinite(cache[2]).all() and np.isfinite(cache[3]).all()


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("d,rot,block,t", [(128, 128, 64, 1), (64, 32, 16, 37), (256, 64, 128, 140), (128, 96, 32, 65)])
def test_write_with_rope_is_the_two_calls(kv, d, rot, block, t, dtype, fmt, interleaved):
    """Strided rows of a fused projection; rotated keys and queries equal apply_rope's bit for bit, past the table too."""
    from scratch_llm_amd import rope

    print_case("kv write rope", d, rot, block, t, dtype, fmt, interleaved)
    b, h, hkv = 2, 6, 2
    g = torch.Generator().manual_seed(d + t)
    qkv = torch.randn(b, t, h + 2 * hkv, d, generator=g).to(DT[dtype]).to(DEV)
    q, k, v = qkv[:, :, :h], qkv[:, :, h:h + hkv], qkv[:, :, h + hkv:]
    cos, sin = rope.rope_table(rot, 50 + t // 2, device=DEV)
    starts = [7, 50]
    width = (50 + t) // block + 1
    table = np.arange(b * width, dtype=np.int32).reshape(b, width)[:, ::-1].copy()
    cache = make_cache(kv, b * width, hkv, d, block, fmt, 9)
    one, two = to_dev(cache, fmt), to_dev(cache, fmt)
    got = kv.write_kv_blocks(k, v, *one, i32(table), i32(starts), i32([t, max(t - 2, 1)]), q=q, rope=(cos, sin), interleaved=interleaved)
    pos = i32(starts)[:, None] + torch.arange(t, dtype=torch.int32, device=DEV)
    kr = rope.apply_rope(k, pos, cos, sin, interleaved=interleaved)
    qr = rope.apply_rope(q, pos, cos, sin, interleaved=interleaved)
    kv.write_kv_blocks(kr, v, *two, i32(table), i32(starts), i32([t, max(t - 2, 1)]))
    assert torch.equal(got, qr)
    same_bytes(back(one), back(two), "rope + write")


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("d,block,starts,tokens,counts", [
    (64, 16, [0, 5, 40], 30, [30, 7, 0]), (128, 64, [63, 64, 1], 1, None), (128, 128, [100, 0, -1], 200, None),
    (256, 32, [31, 90, 127], 70, [70, 70, 1])])
def test_read_is_exact(kv, d, block, starts, tokens, counts, dtype, fmt):
    """Random bytes (E4M3 NaNs too); a table whose end and whose bad page ids read as zeros."""
    print_case("kv read", d, block, dtype, fmt)
    cache = make_cache(kv, 9, 2, d, block, fmt, 5)
    width = 128 // block + 1
    table = np.random.default_rng(6).integers(0, 9, (3, width)).astype(np.int32)
    table[1, 0], table[2, 1] = 9, -3
    k, v = kv.read_kv_blocks(*to_dev(cache, fmt), i32(table), i32(starts), tokens, None if counts is None else i32(counts),
                             dtype=DT[dtype])
    wk, wv = R.read(*cache, table, starts, counts or [tokens] * 3, tokens, fmt)
    for got, want in ((k, wk), (v, wv)):
        want = torch.from_numpy(want).to(DT[dtype])
        assert torch.equal(torch.nan_to_num(got.cpu(), nan=12345.0), torch.nan_to_num(want, nan=12345.0))


def bound(out, terms, d, dtype):
    weight, reach, count, vmax = terms
    eps = torch.finfo(DT[dtype]).eps / 2
    x = weight * (2.0**-11 + 2.0**-18 + 2 * (d + 8) * 2.0**-24 * reach[..., None]) + (count * vmax)[..., None] * 2.0**-28
    return eps * (np.abs(out) + x) + x + torch.finfo(DT[dtype]).tiny


def check_attention(kv, cache, fmt, q, table, starts, counts, scale=None, dtype="bf16", dev=None):
    b, t, h, d = q.shape
    dev = dev or to_dev(cache, fmt)
    want, terms = R.attend(q.double().numpy(), *cache, table, starts, counts or [t] * b, scale or d**-0.5, fmt)
    mark = torch.full((b, t, h, d), 77.0, dtype=DT[dtype], device=DEV)
    kv.attend_kv_blocks(q.to(DEV), *dev, i32(table), i32(starts), None if counts is None else i32(counts), scale=scale, out=mark)
    got = mark.double().cpu().numpy()
    for i in range(b):
        n = t if counts is None else min(max(counts[i], 0), t)
        assert (got[i, n:] == 77.0).all(), f"row {i}: tokens past its count were written"
        w, g, lim = want[i, :n], got[i, :n], bound(want, terms, d, dtype)[i, :n]
        assert (np.isnan(w) == np.isnan(g)).all(), f"row {i}: NaNs differ"
        err = np.where(np.isnan(w), 0.0, np.abs(w - g))
        over = err > np.where(np.isnan(lim), np.inf, lim)
        at = np.argwhere(over)
        assert not over.any(), f"row {i}: {over.sum()} of {over.size} over the bound, first at {at[0].tolist()}: {g[tuple(at[0])]} for {w[tuple(at[0])]}"


# (B, T, H, Hkv, D, block, starts, counts): one token at lengths around the 64-key steps and pages; shared heads of every
# count, odd ones too; drafts; prompts over several tiles; idle rows
ATTENDS = [
    (4, 1, 4, 1, 128, 64, [0, 62, 63, 64], None),
    (3, 1, 8, 8, 64, 16, [1, 15, 300], None),
    (2, 1, 32, 8, 128, 32, [700, 255], None),
    (3, 1, 3, 1, 256, 128, [127, 128, 500], None),
    (3, 1, 32, 2, 128, 16, [-1, 77, 5], None),
    (1, 1, 40, 2, 64, 64, [1000], None),
    (3, 4, 32, 8, 128, 64, [60, 0, 129], [4, 2, 0]),
    (2, 5, 12, 4, 64, 32, [200, 31], None),
    (2, 7, 6, 1, 256, 16, [90, 3], None),
    (2, 33, 8, 2, 128, 64, [0, 100], [33, 20]),
    (1, 100, 6, 2, 64, 128, [0], None),
    (2, 70, 4, 1, 128, 16, [130, 0], [70, 1]),
    (1, 40, 2, 1, 256, 64, [50], None),
    (2, 70, 8, 2, 64, 64, [186, 100], [70, 66]),
    (1, 130, 4, 1, 64, 32, [700], None),
    (1, 80, 4, 2, 256, 128, [600], None),
    (1, 90, 4, 1, 128, 128, [1500], None),
    (2, 30, 4, 1, 128, 32, [333, 0], [30, 17]),
    (1, 43, 6, 2, 64, 16, [90], None),
    (3, 6, 16, 4, 128, 32, [9000, 4111, 6000], None),
    (4, 13, 16, 4, 64, 128, [9000, 4111, 60, 0], [13, 13, 2, 12]),
    (2, 15, 4, 1, 256, 64, [777, 63], None),
]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("case", range(len(ATTENDS)))
def test_attention(kv, case, dtype, fmt):
    b, t, h, hkv, d, block, starts, counts = ATTENDS[case]
    print_case("kv attention", case, dtype, fmt)
    width = (max(starts) + t + block - 1) // block + 1
    cache = fill_valid(make_cache(kv, b * width + 3, hkv, d, block, fmt, case), fmt, 50 + case)
    table = np.random.default_rng(case).permutation(b * width + 3)[:b * width].reshape(b, width).astype(np.int32)
    q = torch.randn(b, t, h, d, generator=torch.Generator().manual_seed(case)).to(DT[dtype])
    check_attention(kv, cache, fmt, q, table, starts, counts, dtype=dtype)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("t", [1, 6, 40])
def test_attention_ignores_what_it_must_not_see(kv, fmt, t):
    """Every byte past the rows' last position is random (E4M3 NaNs among them), later tokens of a chunk hold NaN, and pages
    past the row's end have NaN scales or ids of no page."""
    print_case("kv attention unseen", fmt, t)
    block, d, hkv, h = 32, 128, 2, 8
    starts = [37, 5, 63]
    width = 6
    cache = fill_valid(make_cache(kv, 20, hkv, d, block, fmt, 8), fmt, 9)
    noise = make_cache(kv, 20, hkv, d, block, fmt, 10)
    table = np.random.default_rng(3).permutation(20)[:18].reshape(3, width).astype(np.int32)
    for b in range(3):
        end = starts[b] + t
        for i in range(width):
            p = table[b, i]
            keep = min(max(end - i * block, 0), block)
            cache[0][p, :, keep:] = noise[0][p, :, keep:]
            cache[1][p, :, :, keep:] = noise[1][p, :, :, keep:]
            if keep == 0:
                cache[2][p] = cache[3][p] = np.nan
                table[b, i] = p if i % 2 else 1 << 20
    if fmt == "e4m3" and t > 2:  # a NaN value and key in the middle of the new tokens: earlier tokens must not see it
        for b in range(3):
            pos = starts[b] + t - 2
            p = table[b, pos // block]
            cache[0][p, 0, pos % block, 5] = 0x7F
            cache[1][p, 1, 9, pos % block] = 0xFF
    q = torch.randn(3, t, h, d, generator=torch.Generator().manual_seed(t)).bfloat16()
    with np.errstate(invalid="ignore"):
        check_attention(kv, cache, fmt, q, table, starts, None)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("t,block,width", [(1, 16, 3), (6, 32, 1), (40, 16, 5), (90, 32, 3), (40, 64, 1)])
def test_attention_past_the_table(kv, t, block, width, fmt):
    """Tokens past the table's end, by a little, by a lot and up to the last int32: they attend all that the table has, which
    is no whole number of 64-key steps; rows that begin inside it."""
    print_case("kv attention past the table", t, block, width, fmt)
    d, hkv, h, end = 128, 1, 4, width * block
    starts = [end - 1, end + 100, (1 << 31) - 1, max(end - t, 0), 0]
    b = len(starts)
    cache = fill_valid(make_cache(kv, b * width + 1, hkv, d, block, fmt, t), fmt, 20 + t)
    table = np.random.default_rng(t).permutation(b * width + 1)[:b * width].reshape(b, width).astype(np.int32)
    q = torch.randn(b, t, h, d, generator=torch.Generator().manual_seed(t)).half()
    check_attention(kv, cache, fmt, q, table, starts, None, dtype="fp16")


def test_rows_that_need_a_copy(kv):
    """Queries, keys and values off 16 bytes, with strides of no whole 16 bytes, and with any stride where there is one token
    or one head: the same as of plain tensors."""
    block, d = 16, 64
    g = torch.Generator().manual_seed(11)
    cache = fill_valid(make_cache(kv, 6, 1, d, block, "int8", 2), "int8", 3)
    table, starts = i32([[1, 3, 5], [0, 2, 4]]), i32([20, 33])
    x = torch.randn(2, 1, 1, d, generator=g).bfloat16().to(DEV)
    want = to_dev(cache, "int8")
    kv.write_kv_blocks(x, x, *want, table, starts)
    plain = kv.attend_kv_blocks(x, *want, table, starts)
    flat = torch.zeros(4 * d + 8, dtype=torch.bfloat16, device=DEV)
    views = [flat[1:2 * d + 1].view(2, 1, 1, d), flat.as_strided((2, 1, 1, d), (d, 3, 5, 1)), flat.as_strided((2, 1, 1, d), (d + 1, 3, 5, 1))]
    for i, y in enumerate(views):
        y.copy_(x)
        got = to_dev(cache, "int8")
        kv.write_kv_blocks(y, y, *got, table, starts)
        same_bytes(back(got), back(want), f"view {i}")
        assert torch.equal(kv.attend_kv_blocks(y, *got, table, starts), plain), i


def test_attention_on_a_bad_page_is_nan(kv):
    cache = fill_valid(make_cache(kv, 8, 1, 64, 16, "int8", 1), "int8", 2)
    table = np.array([[0, 1, 2, 3], [4, 8, 5, 6], [7, -1, 0, 0]], np.int32)
    q = torch.randn(3, 3, 2, 64, generator=torch.Generator().manual_seed(1)).bfloat16()
    out = kv.attend_kv_blocks(q.to(DEV), *to_dev(cache, "int8"), i32(table), i32([40, 40, 14]))
    bad = torch.isnan(out).all(-1).all(-1).cpu()
    assert bad.tolist() == [[False] * 3, [True] * 3, [False, False, True]]
    with np.errstate(invalid="ignore"):
        check_attention(kv, cache, "int8", q, table, [40, 40, 14], None)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_attention_over_scales_far_apart(kv, fmt):
    """Value scales over 30 binary orders, key scales that make one key win, a page of scale zero (never written)."""
    block, d = 16, 128
    cache = fill_valid(make_cache(kv, 12, 1, d, block, fmt, 4), fmt, 5)
    cache[3][:, 0] = 2.0 ** np.linspace(-20, 10, 12)
    cache[2][:, 0] = 2.0 ** np.linspace(-3, -12, 12)
    cache[0][7], cache[1][7], cache[2][7], cache[3][7] = 0, 0, 0.0, 0.0
    table = np.arange(12, dtype=np.int32)[None]
    q = torch.randn(1, 2, 4, d, generator=torch.Generator().manual_seed(5)).bfloat16()
    q[0, 0, 1] *= 1e-30
    q[0, 0, 2] = 0.0
    check_attention(kv, cache, fmt, q, table, [190], None)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("t,h,hkv,d", [(1, 8, 2, 128), (6, 8, 2, 64), (5, 7, 1, 128), (3, 10, 1, 256)])
def test_attention_of_uneven_rows(kv, t, h, hkv, d, fmt):
    """Rows from nothing to thousands of keys in one call, idle ones between and at both ends: workgroups take parts that end
    inside one row and begin inside another, hold several whole rows, or a piece of one."""
    print_case("kv attention uneven", t, h, hkv, d, fmt)
    block = 32
    starts = [9, 4100, 0, 63, -1, 2500, 700, 1, 2, 1300, 64, 5]
    counts = [0, t, t, t, t, t, 1, t, 0, max(t - 2, 1), t, 0]
    b, width = len(starts), 4200 // block
    cache = fill_valid(make_cache(kv, 300, hkv, d, block, fmt, t), fmt, t + 1)
    table = np.random.default_rng(t).integers(0, 300, (b, width)).astype(np.int32)
    q = torch.randn(b, t, h, d, generator=torch.Generator().manual_seed(t)).bfloat16()
    check_attention(kv, cache, fmt, q, table, starts, counts)
    check_attention(kv, cache, fmt, q, table, [0] * b, [0] * b)
    check_attention(kv, cache, fmt, q[:2], table[:2], [3, 4000], [t, t])


@pytest.mark.parametrize("t", [1, 9, 40])
def test_attention_long_and_strided(kv, t):
    """A context that is split over workgroups, queries as a strided view, a scale of the caller's."""
    block, d, hkv, h = 64, 64, 1, 4
    width = 70
    cache = fill_valid(make_cache(kv, width, hkv, d, block, "int8", 4), "int8", 5)
    table = np.random.default_rng(1).permutation(width)[None].astype(np.int32)
    wide = torch.randn(1, t, h + 5, d, generator=torch.Generator().manual_seed(6)).half()
    q = wide[:, :, 1:h + 1]
    want, terms = R.attend(q.double().numpy(), *cache, table, [4321], [t], 0.3, "int8")
    out = kv.attend_kv_blocks(wide.to(DEV)[:, :, 1:h + 1], *to_dev(cache, "int8"), i32(table), i32([4321]), scale=0.3)
    assert (np.abs(out.double().cpu().numpy() - want) <= bound(want, terms, d, "fp16")).all()


def test_offsets_past_32_bits(kv):
    """Pages whose bytes lie past 2^31 and 2^32 of the cache: write, read and attend there."""
    block, d, hkv = 128, 256, 8
    pages = (1 << 32) // (block * d * hkv) + 40
    k = torch.zeros(pages, hkv, block, d, dtype=torch.int8, device=DEV)
    v = torch.zeros(pages, hkv, d, block, dtype=torch.int8, device=DEV)
    s = torch.zeros(2, pages, hkv, device=DEV)
    ids = [pages - 1, 3, pages // 2 + 1, pages - 7]
    table = i32([ids])
    g = torch.Generator().manual_seed(3)
    new = torch.randn(2, 1, 400, hkv, d, generator=g).bfloat16()
    kv.write_kv_blocks(new[0].to(DEV), new[1].to(DEV), k, v, s[0], s[1], table, i32([0]))
    small = make_cache(kv, 4, hkv, d, block, "int8", 1)
    R.write(new[0].float().numpy(), new[1].float().numpy(), *small, np.arange(4)[None], [0], [400], "int8")
    q = torch.randn(1, 1, 16, d, generator=g).bfloat16()
    out = kv.attend_kv_blocks(q.to(DEV), k, v, s[0], s[1], table, i32([399])).double().cpu().numpy()
    want, terms = R.attend(q.double().numpy(), *small, np.arange(4)[None], [399], [1], d**-0.5, "int8")
    assert (np.abs(out - want) <= bound(want, terms, d, "bf16")).all()
    got = kv.read_kv_blocks(k, v, s[0], s[1], table, i32([0]), 400)
    for a, b in zip(got, R.read(*small, np.arange(4)[None], [0], [400], 400, "int8")):
        assert torch.equal(a.cpu(), torch.from_numpy(b))


def test_other_stream_and_graph(kv):
    """Write and attend captured on a side stream and replayed with changing positions, eager calls and other shapes (whose
    workspaces torch hands out anew) between the replays."""
    block, d, hkv, h, b, width = 32, 128, 2, 8, 2, 40
    cache = fill_valid(make_cache(kv, b * width, hkv, d, block, "int8", 4), "int8", 5)
    table = np.random.default_rng(1).permutation(b * width).reshape(b, width).astype(np.int32)
    dev, eager = to_dev(cache, "int8"), to_dev(cache, "int8")
    tb = i32(table)
    starts = i32([1100, 500])
    g = torch.Generator().manual_seed(7)
    q, k, v = (torch.randn(b, 1, n, d, generator=g).bfloat16().to(DEV) for n in (h, hkv, hkv))
    out = torch.zeros(b, 1, h, d, dtype=torch.bfloat16, device=DEV)

    def go(c, o, s):
        kv.write_kv_blocks(k, v, *c, tb, s)
        kv.attend_kv_blocks(q, *c, tb, s, out=o)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go(dev, out, starts)
    for i in range(4):
        x = torch.randn(b, 1, hkv, d, generator=g).bfloat16().to(DEV)
        k.copy_(x)
        v.copy_(x * (i + 1))
        want = torch.zeros_like(out)
        go(eager, want, i32([1100 + i, 500 + i]))
        kv.attend_kv_blocks(q[:1], *eager, tb[:1], i32([200]))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), f"replay {i}"
        starts += 1
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kv.attend_kv_blocks(q, *dev, tb, starts)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, kv.attend_kv_blocks(q, *eager, tb, starts))


def test_empty_calls(kv):
    dev = kv.new_kv_blocks(2, 1, 64, block=16, device=DEV)
    assert all(int(x.view(torch.uint8).max()) == 0 for x in dev)
    e = torch.empty(0, 3, 1, 64, dtype=torch.bfloat16, device=DEV)
    none, tb = i32([]), torch.empty(0, 2, dtype=torch.int32, device=DEV)
    kv.write_kv_blocks(e, e, *dev, tb, none)
    assert kv.attend_kv_blocks(e, *dev, tb, none).shape == (0, 3, 1, 64)
    assert kv.read_kv_blocks(*dev, tb, none, 5)[0].shape == (0, 5, 1, 64)
    assert kv.read_kv_blocks(*dev, i32([[0, 1]]), i32([0]), 0)[0].shape == (1, 0, 1, 64)
    z = torch.empty(1, 0, 1, 64, dtype=torch.bfloat16, device=DEV)
    assert kv.attend_kv_blocks(z, *dev, i32([[0, 1]]), i32([0])).shape == (1, 0, 1, 64)


def test_a_cpu_tensor_among_device_tensors_is_refused(kv):
    """Each tensor argument in turn on the CPU: an error before any launch."""
    from scratch_llm_amd import rope, speculative

    c = list(kv.new_kv_blocks(2, 1, 64, block=16, device=DEV))
    x = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16, device=DEV)
    cos, sin = rope.rope_table(64, 8, device=DEV)
    tb, st = i32([[0, 1]]), i32([0])
    lo, dr, u, r = torch.zeros(1, 2, 8, device=DEV), i32([[1]]), torch.zeros(1, 1, device=DEV), torch.zeros(1, device=DEV)
    calls = [
        (lambda *a: kv.write_kv_blocks(*a[:9], q=a[9], rope=(a[10], a[11])), [x, x, *c, tb, st, i32([1]), x, cos, sin]),
        (lambda *a: kv.read_kv_blocks(*a[:6], 1, a[6]), [*c, tb, st, i32([1])]),
        (lambda *a: kv.attend_kv_blocks(*a[:8], out=a[8]), [x, *c, tb, st, i32([1]), torch.zeros_like(x)]),
        (lambda *a: rope.apply_rope(*a[:4], out=a[4]), [x[0], i32([0]), cos, sin, x[0].clone()]),
        (lambda *a: speculative.verify_draft(*a[:4], draft_probs=a[4], counts=a[5]), [lo, dr, u, r, lo[:, :1].clone(), i32([1])]),
    ]
    for call, args in calls:
        call(*args)
        for i in range(len(args)):
            with pytest.raises(RuntimeError, match="device tensors"):
                call(*args[:i], args[i].cpu(), *args[i + 1:])
