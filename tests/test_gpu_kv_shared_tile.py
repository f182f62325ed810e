"""Attention behind shared prefixes where groups are large enough for the prompt kernel (512 query rows, and 2^23 products of these with
shared keys): against float64 on the device, with the bound of tests/test_gpu_kv_block.py. Every test asserts from the plan that the groups
it means are listed for that kernel, so a border that moves fails it."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.conftest import print_case
from tests.test_gpu_kv_block import DEV, DT, bound, fill_valid, i32, make_cache, to_dev
from tests.test_gpu_kv_shared import batch

pytestmark = pytest.mark.gpu
ITEM = 12  # ints of a workgroup's entry in the plan: lead, first, query rows, keys ..


@pytest.fixture(scope="module")
def ks():
    from scratch_llm_amd.quant import kv_shared

    return kv_shared


def large_groups(plan):
    """(query rows, keys) of the groups that the plan gives to the prompt kernel: its last part lists that kernel's workgroups."""
    tile_rows = 128 if plan.head_dim == 256 else 256
    rows = plan.batch * plan.tokens * (plan.heads // plan.kv_heads)
    if rows < 512:
        return []
    n = -(-rows // tile_rows) + plan.batch // 2 + max(1, 256 // plan.kv_heads)
    items = plan.plan[plan.plan.numel() - 4 * ITEM * n:].view(torch.int32).view(n, ITEM).tolist()
    return sorted({(x[0], x[2], x[3]) for x in items if x[0] >= 0})


def attend64(q, dev, table, starts, counts):
    """Row by row over the row's own table; the terms as oracle/kv_block_ref.py's attend gives them."""
    kc, vc, ks, vs = dev
    b, t, h, d = q.shape
    pages, hkv, block, _ = kc.shape
    g = h // hkv
    out, weight = np.zeros((2, b, t, h, d))
    reach, count, vmax = np.zeros((3, b, t, h))
    for i in range(b):
        c = t if counts is None else min(max(counts[i], 0), t)
        n = min(starts[i] + c, table.shape[1] * block)
        if c == 0 or n <= 0:
            continue
        page = torch.from_numpy(table[i, :-(-n // block)].astype(np.int64)).to(DEV)
        bad = (page < 0) | (page >= pages)
        page = torch.where(bad, 0, page)
        last = torch.clamp(torch.arange(c, device=DEV) + starts[i], max=table.shape[1] * block - 1)
        late = torch.arange(n, device=DEV) > last[:, None]
        for x in range(hkv):
            k = kc[page, x].float().double() * ks[page, x].double()[:, None, None]
            v = vc[page, x].float().double().transpose(1, 2) * vs[page, x].double()[:, None, None]
            k = torch.where(bad[:, None, None], torch.nan, k).flatten(0, 1)[:n]
            v = v.flatten(0, 1)[:n].contiguous()
            qx = q[i, :c, x * g:(x + 1) * g].double().to(DEV).transpose(0, 1).reshape(-1, d)
            s = (qx @ k.t().contiguous()).view(g, c, n) * d**-0.5
            p = torch.softmax(s.masked_fill(late, -torch.inf), -1).view(-1, n)
            heads = slice(x * g, (x + 1) * g)
            for to, y in ((out, p @ v), (weight, p @ v.abs())):
                to[i, :c, heads] = y.view(g, c, d).transpose(0, 1).cpu().numpy()
            reach[i, :c, heads] = ((qx.abs() @ k.abs().t().contiguous()).view(g, c, n) * ~late * d**-0.5).amax(-1).t().cpu().numpy()
            count[i, :c, heads], vmax[i, :c, heads] = n, float(v.abs().max())
    return out, (weight, reach, count, vmax)


def check(ks, dev, q, table, starts, counts, plan, dtype):
    b, t, h, d = q.shape
    want, terms = attend64(q, dev, table, starts, counts)
    mark = torch.full((b, t, h, d), 77.0, dtype=DT[dtype], device=DEV)
    ks.attend_shared_kv(q.to(DEV), *dev, i32(table), i32(starts), None if counts is None else i32(counts), shared=plan, out=mark)
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
    return got


def setup(ks, t, h, hkv, d, block, leaders, shared, tail, fmt, dtype, seed):
    g = np.random.default_rng(seed)
    own = (max(tail) + t + block - 1) // block + 1
    table, pages = batch(g, leaders, shared, own, block, max([0, *shared.values()]) + own)
    starts = [shared.get(lead, 0) * block + n for lead, n in zip(leaders, tail)]
    dev = to_dev(fill_valid(make_cache(None, pages, hkv, d, block, fmt, seed), fmt, 50 + seed), fmt)
    q = torch.randn(len(leaders), t, h, d, generator=torch.Generator().manual_seed(seed)).to(DT[dtype])
    plan = ks.plan_shared_kv(i32(table), i32(starts), i32(leaders), block=block, tokens=t, heads=h, kv_heads=hkv, head_dim=d)
    return dev, q, table, starts, plan


# (T, H, Hkv, D, block, leaders, blocks that each leader's rows share, tokens of each row behind them, counts, the large groups)
CASES = [
    # at the border: 1024 x 8192
    (1, 16, 1, 128, 64, [0] * 64, {0: 128}, [i * 7 % 90 for i in range(64)], None, [(0, 1024, 8192)]),
    # small pages; a last tile of 16 rows; a small group and rows of their own beside it
    (1, 8, 1, 64, 32, [-1] + [0] * 66 + [-1] * 2 + [80] * 5, {0: 500, 80: 5}, [i * 5 % 60 for i in range(74)], None, [(1, 528, 16000)]),
    (2, 8, 1, 256, 16, [0] * 33, {0: 1024}, [i % 40 for i in range(33)], [i % 3 for i in range(33)], [(0, 528, 16384)]),
    (4, 8, 2, 128, 128, [5, -1] * 40, {5: 103}, [i * 11 % 200 for i in range(80)], [4, 1, 0, 2, 3] * 16, [(0, 640, 13184)]),
    (1, 8, 1, 64, 16, [7] * 64, {7: 1025}, [i % 50 for i in range(64)], None, [(0, 512, 16384)]),  # 16 keys past the last whole tile
    (1, 4, 1, 256, 64, [0] * 128, {0: 257}, [i % 70 for i in range(128)], None, [(0, 512, 16448)]),
    # two large groups and a small one in turn
    (1, 16, 1, 128, 16, [0, 9] * 36 + [4] * 3, {0: 1000, 9: 1100, 4: 9}, [i * 3 % 40 for i in range(75)], None, [(0, 576, 16000), (1, 576, 17600)]),
    (1, 32, 1, 64, 64, [0] * 40, {0: 130}, [i * 9 % 100 for i in range(40)], None, [(0, 1280, 8320)]),
    # below the border in either way: the direct kernel
    (1, 8, 1, 64, 64, [0] * 64, {0: 254}, [i % 50 for i in range(64)], None, []),
    (1, 8, 1, 128, 64, [0] * 63, {0: 300}, [i % 50 for i in range(63)], None, []),
]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_large_groups(ks, case, dtype, fmt):
    t, h, hkv, d, block, leaders, shared, tail, counts, large = CASES[case]
    print_case("large groups", case, dtype, fmt)
    dev, q, table, starts, plan = setup(ks, t, h, hkv, d, block, leaders, shared, tail, fmt, dtype, case)
    assert large_groups(plan) == large
    check(ks, dev, q, table, starts, counts, plan, dtype)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_rows_grow_and_fall_back(ks, fmt):
    """One plan for many steps: rows grow, some become idle, one is cut into what was shared, one attends nothing."""
    rows, n, block = 64, 128, 64
    dev, q, table, starts, plan = setup(ks, 1, 16, 1, 128, block, [0] * rows, {0: n}, [i % 7 for i in range(rows)], fmt, "fp16", 3)
    assert large_groups(plan) == [(0, 1024, 8192)]
    later = [s + 50 for s in starts]
    check(ks, dev, q, table, later, None, plan, "fp16")
    later[0], later[1], later[2], later[3] = n * block - 1, 3, -1, 1 << 30
    got = check(ks, dev, q, table, later, [1, 1, 1, 1, 0] + [1] * (rows - 5), plan, "fp16")
    assert (got[2] == 0.0).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_what_reaches_every_row(ks, fmt):
    """A scale of NaN, an id of no page and, for E4M3, a NaN code in the shared part reach all rows that attend it, and only these."""
    rows, n, block, d = 65, 128, 64, 64
    leaders = [0] * 64 + [-1]
    tail = [i % 50 for i in range(rows)]
    for what in ("scale", "page", "code"):
        if what == "code" and fmt == "int8":
            continue
        print_case("reaches every row", fmt, what)
        dev, q, table, starts, plan = setup(ks, 1, 16, 1, d, block, leaders, {0: n}, tail, fmt, "bf16", 4)
        if what == "scale":
            dev[2][table[0, 5].item(), 0] = torch.nan
        elif what == "page":
            table[:64, 77] = 1 << 20
        else:
            dev[1].view(torch.uint8)[table[0, 30].item(), 0, 9, 5] = 0x7F
        assert large_groups(plan) == [(0, 1024, 8192)]
        with np.errstate(invalid="ignore"):
            got = check(ks, dev, q, table, starts, None, plan, "bf16")
        assert np.isnan(got[:64, ..., 9]).all() and not np.isnan(got[64]).any()


def test_repetition_streams_and_graphs(ks):
    """Equal bit for bit in repetition, on two streams at once, and in replays of a graph that plans large groups, others and none."""
    rows, n, block = 64, 128, 64
    dev, q, table, starts, plan = setup(ks, 1, 16, 1, 128, block, [0] * rows, {0: n}, [i % 40 for i in range(rows)], "int8", "bf16", 5)
    qd, td, sd = q.to(DEV), i32(table), i32(starts)
    first = ks.attend_shared_kv(qd, *dev, td, sd, shared=plan)
    for _ in range(3):
        assert torch.equal(first, ks.attend_shared_kv(qd, *dev, td, sd, shared=plan))
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for s in streams:
        with torch.cuda.stream(s):
            outs.append(ks.attend_shared_kv(qd, *dev, td, sd, shared=plan))
    torch.cuda.synchronize()
    assert torch.equal(outs[0], first) and torch.equal(outs[1], first)
    lead, out = i32([0] * rows), torch.zeros_like(qd)
    sizes = dict(block=block, tokens=1, heads=16, kv_heads=1, head_dim=128)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ks.plan_shared_kv(td, sd, lead, out=plan, **sizes)
        ks.attend_shared_kv(qd, *dev, td, sd, shared=plan, out=out)
    for groups in ([0] * rows, [-1] * rows, [i % 2 for i in range(rows)], [0] * rows):
        lead.copy_(i32(groups))
        graph.replay()
        torch.cuda.synchronize()
        other = ks.plan_shared_kv(td, sd, lead, **sizes)
        assert large_groups(other) == ([(0, 1024, 8192)] if groups == [0] * rows else [])
        assert torch.equal(out, ks.attend_shared_kv(qd, *dev, td, sd, shared=other))
        torch.ones(1 << 18, device=DEV).sum().item()


def test_a_long_prefix_in_every_head(ks):
    """Pages past 2^31 bytes behind a large group: every row and head, against float64 over the shared part and the row's own token."""
    block, d, hkv, h, n, rows = 128, 256, 8, 32, 150, 128
    pages = 9000
    assert pages * hkv * block * d > 1 << 31
    gen = torch.Generator(device=DEV).manual_seed(1)
    kc = torch.randint(-60, 61, (pages, hkv, block, d), generator=gen, device=DEV, dtype=torch.int8)
    vc = torch.randint(-60, 61, (pages, hkv, d, block), generator=gen, device=DEV, dtype=torch.int8)
    sc = [torch.rand(pages, hkv, generator=gen, device=DEV) * 0.01 + 0.01 for _ in range(2)]
    g = np.random.default_rng(1)
    used = np.sort(g.permutation(np.arange(pages - 2000, pages))[:n + rows])
    table = np.full((rows, n + 1), -1, np.int32)
    table[:, :n], table[:, n] = used[:n], used[n:]
    starts = [n * block + i for i in range(rows)]
    q = torch.randn(rows, 1, h, d, generator=torch.Generator().manual_seed(2)).bfloat16()
    plan = ks.plan_shared_kv(i32(table), i32(starts), i32([0] * rows), block=block, tokens=1, heads=h, kv_heads=hkv, head_dim=d)
    assert large_groups(plan) == [(0, 512, n * block)]
    check(ks, [kc, vc, *sc], q, table, starts, None, plan, "bf16")


def test_a_long_prefix_of_a_small_group_in_every_head(ks):
    """As above for the direct kernel: parts of many keys, six rows."""
    block, d, hkv, h, n, rows = 128, 256, 8, 16, 600, 6
    pages = 9000
    gen = torch.Generator(device=DEV).manual_seed(1)
    kc = torch.randint(-60, 61, (pages, hkv, block, d), generator=gen, device=DEV, dtype=torch.int8)
    vc = torch.randint(-60, 61, (pages, hkv, d, block), generator=gen, device=DEV, dtype=torch.int8)
    sc = [torch.rand(pages, hkv, generator=gen, device=DEV) * 0.01 + 0.01 for _ in range(2)]
    g = np.random.default_rng(1)
    used = np.sort(g.permutation(np.arange(pages - 2000, pages))[:n + rows])
    table = np.full((rows, n + 1), -1, np.int32)
    table[:, :n], table[:, n] = used[:n], used[n:]
    starts = [n * block + i for i in range(rows)]
    q = torch.randn(rows, 1, h, d, generator=torch.Generator().manual_seed(2)).bfloat16()
    plan = ks.plan_shared_kv(i32(table), i32(starts), i32([0] * rows), block=block, tokens=1, heads=h, kv_heads=hkv, head_dim=d)
    check(ks, [kc, vc, *sc], q, table, starts, None, plan, "bf16")
