"""Attention behind shared prefixes (scratch_llm_amd/quant/kv_shared.py) on the GPU against oracle/kv_block_ref.py, with the bound of
tests/test_gpu_kv_block.py: the parts are joined as that attention joins its own, in fp32."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv_block_ref as R
from tests.conftest import print_case
from tests.test_gpu_kv_block import DEV, DT, bound, fill_valid, i32, make_cache, to_dev

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ks():
    from scratch_llm_amd.quant import kv_shared

    return kv_shared


def batch(g, leaders, shared, own, block, width, spare=3):
    """A table in which the rows of leader i name the same `shared[i]` blocks, then `own` of theirs; and the number of pages."""
    b = len(leaders)
    pages = sum(shared.values()) + b * own + spare
    order = list(g.permutation(pages))
    front = {i: [order.pop() for _ in range(n)] for i, n in shared.items()}
    table = np.full((b, width), -1, np.int32)
    for i, lead in enumerate(leaders):
        row = front.get(lead, []) + [order.pop() for _ in range(own)]
        table[i, :min(width, len(row))] = row[:width]
    return table, pages


def check(ks, cache, fmt, q, table, starts, counts, leaders, dtype, block, plan_starts=None, plan=None):
    b, t, h, d = q.shape
    hkv = cache[0].shape[1]
    dev = to_dev(cache, fmt)
    want, terms = R.attend(q.double().numpy(), *cache, table, starts, counts or [t] * b, d**-0.5, fmt)
    td = i32(table)
    if plan is None:
        plan = ks.plan_shared_kv(td, i32(plan_starts or starts), i32(leaders), block=block, tokens=t, heads=h, kv_heads=hkv, head_dim=d)
    mark = torch.full((b, t, h, d), 77.0, dtype=DT[dtype], device=DEV)
    ks.attend_shared_kv(q.to(DEV), *dev, td, i32(starts), None if counts is None else i32(counts), shared=plan, out=mark)
    got = mark.double().cpu().numpy()
    lim = bound(want, terms, d, dtype)
    for i in range(b):
        n = t if counts is None else min(max(counts[i], 0), t)
        assert (got[i, n:] == 77.0).all(), f"row {i}: tokens past its count were written"
        w, x, y = want[i, :n], got[i, :n], lim[i, :n]
        assert (np.isnan(w) == np.isnan(x)).all(), f"row {i}: NaNs differ"
        over = np.where(np.isnan(w), 0.0, np.abs(w - x)) > np.where(np.isnan(y), np.inf, y)
        at = np.argwhere(over)
        assert not over.any(), f"row {i}: {over.sum()} of {over.size} over the bound, first at {at[0].tolist()}: {x[tuple(at[0])]} for {w[tuple(at[0])]}"
    return plan


# (T, H, Hkv, D, block, leaders, blocks that each leader's rows share, tokens of each row behind them (0: the start is at the
# border), counts)
CASES = [
    (1, 4, 1, 64, 16, [0, 0], {0: 1}, [0, 5], None),
    (1, 32, 8, 128, 64, [0] * 8, {0: 9}, [1, 70, 3, 64, 63, 0, 130, 9], None),
    (1, 8, 8, 128, 16, [3, -1, 3, 5, 5, -1, 3], {3: 21, 5: 4}, [7, 200, 40, 0, 1, 0, 15], None),
    (1, 3, 1, 256, 128, [0, 0, 0], {0: 3}, [1, 127, 100], None),
    (4, 32, 8, 128, 32, [1, 1, 1, 0], {1: 12}, [40, 3, 0, 300], [4, 2, 0, 3]),
    (7, 6, 1, 256, 16, [0, 0], {0: 40}, [90, 3], None),
    (5, 12, 12, 64, 16, [0, 0, 0, 4, 4], {0: 30, 4: 7}, [33, 2, 16, 0, 77], [5, 5, 1, 5, 5]),
    (16, 16, 2, 64, 128, [0, 0], {0: 6}, [100, 30], None),
    (8, 16, 1, 128, 64, [0, 0, 0], {0: 20}, [5, 64, 70], None),       # 128 query rows a row
    (9, 16, 1, 128, 64, [0, 0, 0], {0: 20}, [5, 64, 70], [9, 3, 0]),  # above: the plain kernels
    (9, 8, 1, 256, 32, [0, 0], {0: 10}, [5, 64], None),
    (1, 16, 2, 128, 64, [0] * 70, {0: 25}, [i * 7 % 90 for i in range(70)], None),  # 560 query rows: the prompt kernel
    (1, 8, 1, 64, 32, [0] * 66 + [-1] * 2 + [80] * 5, {0: 33, 80: 5}, [i * 5 % 60 for i in range(73)], None),
    (2, 8, 1, 256, 16, [0] * 33, {0: 70}, [i % 40 for i in range(33)], [i % 3 for i in range(33)]),
    (1, 4, 2, 128, 32, list(range(40)), {}, [i * 3 for i in range(40)], None),  # groups of one
    (1, 2, 1, 64, 16, [i // 2 for i in range(60)], {i: 1 + i % 9 for i in range(30)}, [i % 33 for i in range(60)], None),
]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_shared(ks, case, dtype, fmt):
    t, h, hkv, d, block, leaders, shared, tail, counts = CASES[case]
    print_case("shared", case, dtype, fmt)
    g = np.random.default_rng(case)
    own = (max(tail) + t + block - 1) // block + 1
    width = max([0, *shared.values()]) + own
    table, pages = batch(g, leaders, shared, own, block, width)
    starts = [shared.get(lead, 0) * block + n for lead, n in zip(leaders, tail)]
    cache = fill_valid(make_cache(None, pages, hkv, d, block, fmt, case), fmt, 50 + case)
    q = torch.randn(len(leaders), t, h, d, generator=torch.Generator().manual_seed(case)).to(DT[dtype])
    check(ks, cache, fmt, q, table, starts, counts, leaders, dtype, block)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_what_is_shared(ks, fmt):
    """Rows that part early, rows whose start lies inside what they share, entries that name no page: the group shares what is
    safe, and the result is the plain one."""
    g = np.random.default_rng(2)
    block, d, hkv, h = 16, 128, 2, 8
    leaders = [0, 0, 0, 3, 3, 5, 5, 7, 7]
    table, pages = batch(g, leaders, {0: 12, 3: 10, 5: 6, 7: 8}, 4, block, 18)
    table[2, 5] = table[2, 13]    # row 2 parts after five blocks
    starts = [200, 210, 195, 61, 170, 100, 96, 140, 135]  # row 3 is inside its fourth block
    table[6, 2] = table[5, 2] = -1  # no page: whoever attends it gets NaN
    table[8, 7] = table[7, 7] = pages + 5
    cache = fill_valid(make_cache(None, pages, hkv, d, block, fmt, 4), fmt, 5)
    q = torch.randn(len(leaders), 1, h, d, generator=torch.Generator().manual_seed(1)).bfloat16()
    with np.errstate(invalid="ignore"):
        check(ks, cache, fmt, q, table, starts, None, leaders, "bf16", block)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("rows", [3, 70])
def test_what_must_not_be_seen(ks, fmt, rows):
    """Random bytes (E4M3 NaNs among them) behind every row's last position, NaN scales and ids of no page past it; a NaN code in a
    shared page reaches every row."""
    g = np.random.default_rng(rows)
    block, d, hkv, h, n = 32, 64, 1, 8, 6
    leaders = [0] * rows
    own = 4
    table, pages = batch(g, leaders, {0: n}, own, block, n + own)
    starts = [n * block + i * 11 % 60 for i in range(rows)]
    cache = fill_valid(make_cache(None, pages, hkv, d, block, fmt, 8), fmt, 9)
    noise = make_cache(None, pages, hkv, d, block, fmt, 10)
    for b in range(rows):
        for j in range(n, n + own):
            p = table[b, j]
            keep = min(max(starts[b] + 1 - j * block, 0), block)
            cache[0][p, :, keep:] = noise[0][p, :, keep:]
            cache[1][p, :, :, keep:] = noise[1][p, :, :, keep:]
            if keep == 0:
                cache[2][p] = cache[3][p] = np.nan
                table[b, j] = p if j % 2 else 1 << 20
    q = torch.randn(rows, 1, h, d, generator=torch.Generator().manual_seed(3)).bfloat16()
    with np.errstate(invalid="ignore"):
        check(ks, cache, fmt, q, table, starts, None, leaders, "bf16", block)
        if fmt == "e4m3":
            cache[1][table[0, 2], 0, 9, 5] = 0x7F
            check(ks, cache, fmt, q, table, starts, None, leaders, "bf16", block)


@pytest.mark.parametrize("rows", [4, 80])
def test_a_plan_serves_while_rows_grow_and_fall_back(ks, rows):
    """One plan for many steps: rows grow, some become idle, and one is cut back into what was shared and attends for itself."""
    g = np.random.default_rng(rows)
    block, d, hkv, h, n = 16, 128, 1, 8, 20
    leaders = [0] * (rows - 1) + [-1]
    table, pages = batch(g, leaders, {0: n}, 5, block, n + 5)
    cache = fill_valid(make_cache(None, pages, hkv, d, block, "int8", 1), "int8", 2)
    begin = [n * block + i % 7 for i in range(rows)]
    begin[-1] = 50
    q = torch.randn(rows, 1, h, d, generator=torch.Generator().manual_seed(4)).half()
    plan = check(ks, cache, "int8", q, table, begin, None, leaders, "fp16", block)
    later = [s + 60 for s in begin]
    check(ks, cache, "int8", q, table, later, None, leaders, "fp16", block, plan=plan)
    later[1], later[2] = n * block - 1, 3
    check(ks, cache, "int8", q, table, later, [1, 1, 1, 0] + [1] * (rows - 4), leaders, "fp16", block, plan=plan)
    later[0] = -1  # attends nothing: zeros
    later[3] = 1 << 30  # past the table
    check(ks, cache, "int8", q, table, later, None, leaders, "fp16", block, plan=plan)


def test_prefixes_of_half_a_step(ks):
    """Shared parts that are no whole number of 64-key steps nor of tiles, in both kernels."""
    for n, d, rows in ((1, 64, 2), (3, 64, 70), (5, 64, 2), (7, 128, 70), (9, 256, 70)):
        g = np.random.default_rng(n)
        block, hkv, h = 16, 1, 8
        leaders = [1] * rows
        table, pages = batch(g, leaders, {1: n}, 2, block, n + 2)
        cache = fill_valid(make_cache(None, pages, hkv, d, block, "e4m3", n), "e4m3", n + 1)
        q = torch.randn(rows, 1, h, d, generator=torch.Generator().manual_seed(n)).bfloat16()
        print_case("half a step", n, d, rows)
        check(ks, cache, "e4m3", q, table, [n * block + i % 17 for i in range(rows)], None, leaders, "bf16", block)


def test_many_groups(ks):
    """Groups of both kernels beside one another, more rows than a workgroup of the plan has threads."""
    g = np.random.default_rng(6)
    block, d, hkv, h = 16, 64, 1, 8
    leaders = [0] * 100 + [200 + i // 3 for i in range(1000)] + [-1] * 20 + [5] * 64
    shared = {0: 9, 5: 31, **{200 + i: i % 6 for i in range(334)}}
    table, pages = batch(g, leaders, shared, 2, block, 33)
    starts = [shared.get(lead, 0) * block + i % 16 for i, lead in enumerate(leaders)]
    cache = fill_valid(make_cache(None, pages, hkv, d, block, "int8", 1), "int8", 2)
    q = torch.randn(len(leaders), 1, h, d, generator=torch.Generator().manual_seed(4)).half()
    check(ks, cache, "int8", q, table, starts, None, leaders, "fp16", block)


def test_a_long_prefix(ks):
    """Pages past 2^31 bytes, parts of tens of thousands of keys."""
    block, d, hkv, h, n, rows = 128, 256, 8, 16, 600, 6
    pages = 9000
    assert pages * hkv * block * d > 1 << 31
    gen = torch.Generator(device=DEV).manual_seed(1)
    kc = torch.randint(-60, 61, (pages, hkv, block, d), generator=gen, device=DEV, dtype=torch.int8)
    vc = torch.randint(-60, 61, (pages, hkv, d, block), generator=gen, device=DEV, dtype=torch.int8)
    sc = [torch.full((pages, hkv), 0.02, device=DEV) for _ in range(2)]
    g = np.random.default_rng(1)
    used = np.sort(g.permutation(np.arange(pages - 2000, pages))[:n + rows])
    table = np.full((rows, n + 1), -1, np.int32)
    table[:, :n] = used[:n]
    table[:, n] = used[n:]
    starts = [n * block + i for i in range(rows)]
    q = torch.randn(rows, 1, h, d, generator=torch.Generator().manual_seed(2)).bfloat16()
    td = i32(table)
    from scratch_llm_amd.quant import kv_block

    plan = ks.plan_shared_kv(td, i32(starts), i32([0] * rows), block=block, tokens=1, heads=h, kv_heads=hkv, head_dim=d)
    got = ks.attend_shared_kv(q.to(DEV), kc, vc, *sc, td, i32(starts), shared=plan).double()
    plain = kv_block.attend_kv_blocks(q.to(DEV), kc, vc, *sc, td, i32(starts)).double()
    # both within the attention's bound of the same result: a few bf16 steps of the largest weights' mean
    k = kc[td[0].long(), 0].double().flatten(0, 1)[:starts[0] + 1] * 0.02
    v = vc[td[0].long(), 0].double().transpose(1, 2).flatten(0, 1)[:starts[0] + 1] * 0.02
    p = torch.softmax(q[0, 0, :2].double().to(DEV) @ k.t().contiguous() / 16.0, -1)
    want, mass = p @ v, p @ v.abs()
    lim = 2.0**-8 * want.abs() + mass * (2.0**-11 + 2.0**-17) * (1 + 2.0**-8) + 2.0**-24
    for x in (got, plain):
        assert ((x[0, 0, :2] - want).abs() <= lim).all()


@pytest.mark.parametrize("empty", [0, 2, 5])
def test_an_emptied_row_leaves_the_others_their_shared_part(ks, empty):
    """The first row, one between and the last. That the others still read together shows in their results: their shared part comes
    through the entries of the first of them, so those of the rest may name a page of NaN scales after the plan is made."""
    g = np.random.default_rng(empty)
    block, d, hkv, h, n, rows = 64, 64, 1, 8, 4, 6
    leaders = [4] * rows
    table, pages = batch(g, leaders, {4: n}, 1, block, n + 1)
    starts = [n * block + 3 + i for i in range(rows)]
    starts[empty] = 0
    table[empty] = -1
    cache = fill_valid(make_cache(None, pages, hkv, d, block, "int8", 1), "int8", 2)
    q = torch.randn(rows, 1, h, d, generator=torch.Generator().manual_seed(4)).half()
    want, terms = R.attend(q.double().numpy(), *cache, table, starts, [1] * rows, d**-0.5, "int8")
    plan = ks.plan_shared_kv(i32(table), i32(starts), i32(leaders), block=block, tokens=1, heads=h, kv_heads=hkv, head_dim=d)
    spare = next(p for p in range(pages) if p not in table)
    cache[2][spare] = cache[3][spare] = np.nan
    others = [i for i in range(rows) if i != empty]
    table[others[1:], :n] = spare
    got = ks.attend_shared_kv(q.to(DEV), *to_dev(cache, "int8"), i32(table), i32(starts), shared=plan).double().cpu().numpy()
    assert (np.abs(got - want) <= bound(want, terms, d, "fp16"))[others].all()


def test_streams_graphs_and_repetition(ks):
    g = np.random.default_rng(9)
    block, d, hkv, h, n, rows = 64, 128, 2, 8, 5, 40
    leaders = [i // 10 * 10 for i in range(rows)]
    table, pages = batch(g, leaders, {i: n for i in range(0, rows, 10)}, 4, block, n + 4)
    cache = fill_valid(make_cache(None, pages, hkv, d, block, "int8", 1), "int8", 2)
    dev = to_dev(cache, "int8")
    td, lead = i32(table), i32(leaders)
    starts = i32([n * block + i for i in range(rows)])
    q = torch.randn(rows, 1, h, d, generator=torch.Generator().manual_seed(4)).bfloat16().to(DEV)
    sizes = dict(block=block, tokens=1, heads=h, kv_heads=hkv, head_dim=d)
    plan = ks.plan_shared_kv(td, starts, lead, **sizes)
    first = ks.attend_shared_kv(q, *dev, td, starts, shared=plan)
    for _ in range(3):
        assert torch.equal(first, ks.attend_shared_kv(q, *dev, td, starts, shared=plan))
    # two streams at once share the plan
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        x = ks.attend_shared_kv(q, *dev, td, starts, shared=plan)
    with torch.cuda.stream(b):
        y = ks.attend_shared_kv(q, *dev, td, starts, shared=plan)
    torch.cuda.synchronize()
    assert torch.equal(x, first) and torch.equal(y, first)
    # a graph that plans and attends, replayed for other groups and longer rows
    out = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ks.plan_shared_kv(td, starts, lead, out=plan, **sizes)
        ks.attend_shared_kv(q, *dev, td, starts, shared=plan, out=out)
        starts.add_(1)
    base = starts.clone()
    for step in range(4):
        lead.copy_(i32(leaders if step % 2 else [i % 7 for i in range(rows)] if step else [-1] * rows))
        graph.replay()
        torch.cuda.synchronize()
        q_host = q.double().cpu().numpy()
        want, terms = R.attend(q_host, *cache, table, (base + step).tolist(), [1] * rows, d**-0.5, "int8")
        lim = bound(want, terms, d, "bf16")
        assert (np.abs(out.double().cpu().numpy() - want) <= lim).all(), step
        torch.ones(1 << 18, device=DEV).sum().item()
    again = ks.attend_shared_kv(q, *dev, td, starts, shared=ks.plan_shared_kv(td, starts, lead, **sizes))
    strided = torch.zeros(rows, 1, h, 2 * d, dtype=torch.bfloat16, device=DEV)
    strided[..., :d] = q
    assert torch.equal(again, ks.attend_shared_kv(strided[..., :d], *dev, td, starts, shared=plan))
