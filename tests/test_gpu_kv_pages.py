"""The pages of the block-scaled cache (scratch_llm_amd/quant/kv_pages.py) on the GPU against oracle/kv_pages_ref.py: every
table, count, code and scale bit for bit."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv_pages_ref as R
from tests.conftest import print_case

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def kp():
    from scratch_llm_amd.quant import kv_pages

    return kv_pages


def new_pool(g, layers, pages, hkv, d, block):
    kc = g.integers(0, 256, (layers, pages, hkv, block, d), dtype=np.uint8)
    vc = g.integers(0, 256, (layers, pages, hkv, d, block), dtype=np.uint8)
    return [kc, vc, *(g.normal(0, 1, (layers, pages, hkv)).astype(np.float32) for _ in range(2))]


def dev(x, fmt=None):
    t = torch.from_numpy(np.ascontiguousarray(x)).to(DEV)
    return t if x.dtype != np.uint8 else t.view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn)


def up(pool, fmt="int8"):
    return [dev(x, fmt) for x in pool]


def host(t):
    return (t.view(torch.uint8) if t.element_size() == 1 else t).cpu().numpy()


def same(got, want, what):
    for name, x, y in zip(("k codes", "v codes", "k scale", "v scale", "table", "lengths", "refs"), got, want):
        x = host(x)
        assert x.shape == y.shape and np.array_equal(x.view(np.uint8), np.ascontiguousarray(y).view(np.uint8)), f"{what}: {name}"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def owned(g, rows, width, pages, lengths, block):
    """A table of rows that own scattered pages."""
    table = np.full((rows, width), -1, np.int32)
    order = list(g.permutation(pages))
    for b, n in enumerate(lengths):
        for j in range((n + block - 1) // block):
            table[b, j] = order.pop()
    return table, np.bincount(table[table >= 0].ravel(), minlength=pages).astype(np.int32)


SHAPES = [(1, 1, 64, 16), (2, 3, 64, 16), (3, 8, 128, 64), (2, 12, 256, 128), (1, 5, 256, 32), (2, 1, 128, 128)]  # layers, Hkv, D, block


@pytest.mark.parametrize("layers,hkv,d,block", SHAPES)
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_copy(kp, layers, hkv, d, block, fmt):
    g = np.random.default_rng(1)
    for pages, n in ((2, 1), (9, 4), (67, 33)):
        print_case("copy", layers, hkv, d, block, pages, n)
        pool = new_pool(g, layers, pages, hkv, d, block)
        order = g.permutation(pages)
        src, dst = order[:n].astype(np.int32), order[n:2 * n].astype(np.int32)
        if n > 2:
            src[0], dst[1], src[2] = -1, pages, dst[2]  # no page; the same page
        there = up(pool, fmt)
        kp.copy_kv_pages(dev(src), dev(dst), *there)
        R.copy(pool, src, dst)
        same(there, pool, "copy")


def test_copy_of_one_layer_and_of_nothing(kp):
    g = np.random.default_rng(2)
    pool = new_pool(g, 1, 5, 2, 64, 32)
    there = [x[0] for x in up(pool)]
    kp.copy_kv_pages(i32([3]), i32([1]), *there)
    kp.copy_kv_pages(i32([]), i32([]), *there)
    R.copy(pool, [3], [1])
    same(there, [x[0] for x in pool], "one layer")


# parents, lengths, width, pages, block
FORKS = [
    ([0], [5], 1, 1, 16),
    ([0, 0], [5, 0], 2, 2, 16),              # the last free page
    ([0, 0, 0], [16, 3, 40], 3, 9, 16),      # a full block: nothing to copy
    ([1, 0], [17, 33], 4, 6, 16),            # two rows change places: nobody copies
    ([1, 1, 1, -1], [20, 37, 0, 64], 4, 12, 16),
    ([3, 3, 3, 0], [50, 16, 5, 61], 4, 14, 16),  # the first taker gets the open page, the others copies
    ([5, -7, 1, 2], [9, 8, 7, 6], 2, 8, 16),  # parents that are no row
    ([2, 2, 2, 2, 2], [0, 0, 100, 0, 0], 4, 10, 32),
    ([0, 0, 1, 1], [128, 127, 126, 0], 1, 4, 128),
    ([1, 1], [-5, 300], 2, 5, 64),           # lengths outside the table
]


@pytest.mark.parametrize("case", range(len(FORKS)))
def test_fork(kp, case):
    parents, lengths, width, pages, block = FORKS[case]
    g = np.random.default_rng(case)
    print_case("fork", FORKS[case])
    pool = new_pool(g, 2, pages, 2, 64, block)
    capped = [min(max(n, 0), width * block) for n in lengths]
    table, refs = owned(g, len(parents), width, pages, capped, block)
    lengths = np.array(lengths, np.int32)
    there, t, n, r = up(pool), dev(table), dev(lengths), dev(refs)
    ok = kp.fork_kv_rows(i32(parents), *there, t, n, r)
    want = R.fork(parents, pool, table, lengths, refs, block)
    assert int(ok) == want
    same([*there, t, n, r], [*pool, table, lengths, refs], "fork")


@pytest.mark.parametrize("width,pages", [(4100, 60), (5, 8200), (1, 8192), (300, 8192)])
@pytest.mark.parametrize("rows", [4, 1024, 1025])
def test_fork_at_the_ends_of_its_forms(kp, rows, width, pages):
    """Few rows, entries and pages are planned by one workgroup, more of any by several."""
    g = np.random.default_rng(rows + width + pages)
    block = 16
    print_case("fork", rows, width, pages)
    lengths = np.zeros(rows, np.int32)
    some = g.permutation(rows)[:40]
    lengths[some] = g.integers(0, min(width * block, 40), len(some))
    pool = new_pool(g, 1, pages, 1, 64, block)
    table, refs = owned(g, rows, width, pages, lengths if pages > 200 else lengths * (np.arange(rows) < 4), block)
    lengths = (table >= 0).sum(1).astype(np.int32) * block - g.integers(0, 2, rows).astype(np.int32) * 5
    np.maximum(lengths, 0, out=lengths)
    parents = np.where(g.random(rows) < 0.4, np.arange(rows), g.integers(-1, rows + 1, rows)).astype(np.int32)
    parents[:4] = [some[0], some[0], 0, 2]
    there, t, n, r = up(pool), dev(table), dev(lengths), dev(refs)
    ok = kp.fork_kv_rows(dev(parents), *there, t, n, r)
    assert int(ok) == R.fork(list(parents), pool, table, lengths, refs, block)
    same([*there, t, n, r], [*pool, table, lengths, refs], "fork")


def test_fork_without_room_changes_nothing(kp):
    g = np.random.default_rng(8)
    pool = new_pool(g, 1, 5, 1, 64, 16)
    table, refs = owned(g, 4, 3, 5, [40, 0, 0, 0], 16)
    lengths = np.array([40, 0, 0, 0], np.int32)
    there, t, n, r = up(pool), dev(table), dev(lengths), dev(refs)
    assert int(kp.fork_kv_rows(i32([0, 0, 0, 0]), *there, t, n, r)) == 0  # three copies, two free pages
    same([*there, t, n, r], [*pool, table, lengths, refs], "refused")
    assert int(kp.fork_kv_rows(i32([0, 0, 0, 3]), *there, t, n, r)) == 1
    assert R.fork([0, 0, 0, 3], pool, table, lengths, refs, 16) == 1
    same([*there, t, n, r], [*pool, table, lengths, refs], "two copies")


# starts, counts, width, pages, block
RESERVES = [
    ([0], [1], 1, 1, 16),
    ([0, 0], [0, -3], 2, 2, 16),
    ([15, 16, 17], [1, 1, 1], 3, 9, 16),
    ([0, 40, -1], [100, 5, 50], 5, 20, 16),   # a negative start gets nothing
    ([70, 100], [1000, 28], 8, 20, 16),       # past the table
    ([0, 0, 0], [300, 290, 1], 20, 40, 16),
    ([5, 200], [3, 2147483647], 3, 8, 128),   # a sum past 32 bits
    ([300], [5000], 400, 400, 16),            # more blocks of a row than a workgroup has threads
]


@pytest.mark.parametrize("case", range(len(RESERVES)))
def test_reserve(kp, case):
    starts, counts, width, pages, block = RESERVES[case]
    g = np.random.default_rng(case)
    print_case("reserve", RESERVES[case])
    pool = new_pool(g, 2, pages, 1, 64, block)
    table, refs = owned(g, len(starts), width, pages, [min(max(s, 0), width * block) for s in starts], block)
    there, t, r = up(pool), dev(table), dev(refs)
    ok = kp.reserve_kv_pages(*there, t, i32(starts), i32(counts), r)
    want = R.reserve(pool, table, starts, counts, refs, block)
    assert int(ok) == want
    same([*there, t], [*pool, table], "reserve")
    np.testing.assert_array_equal(host(r), refs)


def test_reserve_copies_shared_pages(kp):
    g = np.random.default_rng(4)
    block, pages = 32, 24
    pool = new_pool(g, 3, pages, 2, 128, block)
    table, refs = owned(g, 5, 4, pages, [70, 0, 0, 33, 0], block)
    table[1], table[2] = table[0], table[0]   # three rows hold one open page
    table[4, 0] = table[3, 0]                  # and two a full one
    refs = np.bincount(table[table >= 0].ravel(), minlength=pages).astype(np.int32)
    starts, counts = [70, 70, 70, 40, 10], [1, 0, 40, 1, 3]
    there, t, r = up(pool, "e4m3"), dev(table), dev(refs)
    ok = kp.reserve_kv_pages(*there, t, i32(starts), i32(counts), r)
    assert int(ok) == R.reserve(pool, table, starts, counts, refs, block) == 1
    same([*there, t], [*pool, table], "shared")
    np.testing.assert_array_equal(host(r), refs)


@pytest.mark.parametrize("width", [16, 17, 4100])
@pytest.mark.parametrize("rows", [3, 1024, 1025])
def test_reserve_at_the_ends_of_its_forms(kp, rows, width):
    """Few rows and entries are planned by one workgroup, more of either by several. Some pages have two holders."""
    g = np.random.default_rng(rows + width)
    block, pages = 16, 4500
    print_case("reserve", rows, width)
    lengths = np.zeros(rows, np.int32)
    some = np.unique(np.r_[g.permutation(rows)[:20], 0, rows - 1])
    lengths[some] = g.integers(0, min(width, 30) * block, len(some))
    pool = new_pool(g, 1, pages, 1, 64, block)
    table, refs = owned(g, rows, width, pages, lengths, block)
    for a, b in zip(some[:-1], some[1:]):  # a cut row writes into pages that another holds too
        n = int(min(lengths[a], lengths[b])) // block
        for j in range(n):
            refs[table[a, j]] -= 1
            table[a, j] = table[b, j]
            refs[table[b, j]] += 1
    starts = (lengths * g.random(rows)).astype(np.int32)
    counts = np.where(g.random(rows) < 0.7, g.integers(0, 2 * block, rows), 0).astype(np.int32)
    counts[0] = 3000  # most of a long row, or past the table
    there, t, r = up(pool), dev(table), dev(refs)
    ok = kp.reserve_kv_pages(*there, t, dev(starts), dev(counts), r)
    assert int(ok) == R.reserve(pool, table, starts, counts, refs, block) == 1
    same([*there, t, dev(starts), r], [*pool, table, starts, refs], "reserve")


def test_reserve_without_room_changes_nothing(kp):
    g = np.random.default_rng(5)
    pool = new_pool(g, 1, 4, 1, 64, 16)
    table, refs = owned(g, 2, 4, 4, [20, 0], 16)
    table[1, 0] = table[0, 0]
    refs[table[0, 0]] += 1
    there, t, r = up(pool), dev(table), dev(refs)
    for starts, counts in (([20, 0], [30, 16]), ([0, 0], [64, 64])):
        assert int(kp.reserve_kv_pages(*there, t, i32(starts), i32(counts), r)) == 0
        same([*there, t], [*pool, table], "refused")
        np.testing.assert_array_equal(host(r), refs)


@pytest.mark.parametrize("width", [1, 5, 300])
def test_free(kp, width):
    g = np.random.default_rng(width)
    block, rows = 16, 7
    pages = rows * width + 3
    lengths = g.integers(0, width * block + 1, rows).astype(np.int32)
    table, refs = owned(g, rows, width, pages, lengths, block)
    table[3] = table[2]
    refs = np.bincount(table[table >= 0].ravel(), minlength=pages).astype(np.int32)
    if width > 2:
        table[5, 1] = pages + 7  # names no page: the entry goes, no count changes
    for keep in ([0] * rows, [-1, 1, 15, 16, 17, width * block, 1 << 30], list(lengths)):
        tb, ln, rf = table.copy(), lengths.copy(), refs.copy()
        t, n, r = dev(tb), dev(ln), dev(rf)
        kp.free_kv_rows(i32([int(x) for x in keep]), t, n, r, block=block)
        R.free(keep, tb, ln, rf, block)
        for x, y in ((t, tb), (n, ln), (r, rf)):
            np.testing.assert_array_equal(host(x), y)


# pages, in use: a share, none, all, the front, the back
@pytest.mark.parametrize("pages", [1, 2, 33, 4096, 4097, 9001])
@pytest.mark.parametrize("how", ["some", "none", "all", "front", "back"])
def test_compact(kp, pages, how):
    print_case("compact", pages, how)
    g = np.random.default_rng(pages)
    pool = new_pool(g, 2 if pages < 100 else 1, pages, 1, 64, 16)
    n = {"some": max(1, int(0.4 * pages)), "none": 0, "all": pages, "front": pages // 2, "back": pages // 2}[how]
    ids = {"front": np.arange(n), "back": np.arange(pages - n, pages)}.get(how)
    ids = g.permutation(pages)[:n] if ids is None else ids
    width = 5
    rows = max(1, -(-n // width))
    table = np.full(rows * width, -1, np.int32)
    table[:n] = g.permutation(ids)
    table = table.reshape(rows, width)
    refs = np.bincount(table[table >= 0].ravel(), minlength=pages).astype(np.int32)
    if n > 1:
        refs[ids[0]] += 2  # a page that the caller holds besides
    there, t, r = up(pool), dev(table), dev(refs)
    live, moved = kp.compact_kv_pages(*there, t, r)
    want_live, want_moved = R.compact(pool, table, refs)
    assert int(live) == want_live
    same([*there, t], [*pool, table], "compact")
    np.testing.assert_array_equal(host(r), refs)
    np.testing.assert_array_equal(host(moved), want_moved)


def test_compact_without_a_table(kp):
    g = np.random.default_rng(9)
    pool = new_pool(g, 1, 8, 1, 64, 16)
    refs = np.array([0, 1, 0, 0, 2, 0, 0, 1], np.int32)
    there, r, none = up(pool), dev(refs), torch.empty(0, 3, dtype=torch.int32, device=DEV)
    live, moved = kp.compact_kv_pages(*there, none, r)
    assert (int(live), R.compact(pool, np.empty((0, 3), np.int32), refs)[0]) == (3, 3)
    same(there, pool, "no table")
    np.testing.assert_array_equal(host(r), refs)


@pytest.mark.parametrize("seed,block,hkv,d", [(1, 16, 2, 64), (2, 64, 3, 128), (3, 128, 1, 256)])
def test_a_serving_history(kp, seed, block, hkv, d):
    """Many calls one after the other without a look at the host, as a server makes them, against the oracle's history."""
    g = np.random.default_rng(seed)
    rows, width, pages = 11, 7, 60
    pool = new_pool(g, 2, pages, hkv, d, block)
    table, lengths, refs = np.full((rows, width), -1, np.int32), np.zeros(rows, np.int32), np.zeros(pages, np.int32)
    there, t, n, r = up(pool), dev(table), dev(lengths), dev(refs)
    oks, want = [], []
    for step in range(40):
        what = int(g.integers(0, 5))
        if what <= 1:
            counts = g.integers(0, block + 5, rows).astype(np.int32)
            c = dev(counts)
            ok = kp.reserve_kv_pages(*there, t, n, c, r)
            n.add_(c * ok).clamp_(max=width * block)
            oks.append(ok)
            want.append(R.reserve(pool, table, lengths, counts, refs, block))
            lengths += want[-1] * counts
            np.minimum(lengths, width * block, out=lengths)
        elif what == 2:
            parents = g.integers(0, rows, rows)
            parents = np.where(g.random(rows) < 0.5, np.arange(rows), parents).astype(np.int32)
            oks.append(kp.fork_kv_rows(dev(parents), *there, t, n, r))
            want.append(R.fork(list(parents), pool, table, lengths, refs, block))
        elif what == 3:
            keep = np.where(g.random(rows) < 0.6, lengths, g.integers(0, width * block, rows)).astype(np.int32)
            kp.free_kv_rows(dev(keep), t, n, r, block=block)
            R.free(keep, table, lengths, refs, block)
        else:
            live, moved = kp.compact_kv_pages(*there, t, r)
            a, b = R.compact(pool, table, refs)
            oks.append(live)
            want.append(a)
    assert [int(x) for x in oks] == want
    same([*there, t, n, r], [*pool, table, lengths, refs], "history")


def test_many_rows_and_pages(kp):
    """More rows than a workgroup has threads, more pages than it scans in one pass."""
    g = np.random.default_rng(12)
    rows, width, block, pages = 2500, 3, 16, 40000
    lengths = g.integers(1, width * block, rows).astype(np.int32)
    pool = new_pool(g, 1, pages, 1, 64, block)
    table, refs = owned(g, rows, width, pages, lengths, block)
    refs[:20000] += 1  # held elsewhere: free pages come late
    parents = (np.arange(rows) // 3 * 3).astype(np.int32)
    there, t, n, r = up(pool), dev(table), dev(lengths), dev(refs)
    ok = kp.fork_kv_rows(dev(parents), *there, t, n, r)
    assert int(ok) == R.fork(list(parents), pool, table, lengths, refs, block) == 1
    same([*there, t, n, r], [*pool, table, lengths, refs], "fork")
    counts = g.integers(0, 2 * block, rows).astype(np.int32)
    ok = kp.reserve_kv_pages(*there, t, n, dev(counts), r)
    assert int(ok) == R.reserve(pool, table, lengths, counts, refs, block) == 1
    same([*there, t, n, r], [*pool, table, lengths, refs], "reserve")


def test_a_pool_past_two_gibibytes(kp):
    """Offsets past 2^31 bytes: the last pages of the last layers."""
    layers, pages, hkv, d, block = 33, 260, 8, 256, 128  # 68 MB of keys a layer
    assert layers * pages * hkv * d * block > 1 << 31
    kc = torch.zeros(layers, pages, hkv, block, d, dtype=torch.int8, device=DEV)
    vc = torch.zeros(layers, pages, hkv, d, block, dtype=torch.int8, device=DEV)
    ks, vs = (torch.zeros(layers, pages, hkv, device=DEV) for _ in range(2))
    for x in (kc, vc):
        x[:, pages - 1] = torch.arange(x[0, 0].numel(), device=DEV).view(x[0, 0].shape).to(torch.int8)
        x[:, pages - 1] += torch.arange(layers, device=DEV, dtype=torch.int8).view(-1, 1, 1, 1)
    ks[:, pages - 1], vs[:, pages - 1] = 3.0, 4.0
    kp.copy_kv_pages(i32([pages - 1, pages - 1]), i32([pages - 2, 0]), kc, vc, ks, vs)
    for x in (kc, vc, ks, vs):
        assert torch.equal(x[:, pages - 2], x[:, pages - 1]) and torch.equal(x[:, 0], x[:, pages - 1])
        assert int(x[:, 1:pages - 2].count_nonzero()) == 0


def test_captured_and_on_another_stream(kp):
    g = np.random.default_rng(20)
    rows, width, pages, block = 6, 5, 40, 16
    pool = new_pool(g, 2, pages, 2, 64, block)
    start = g.integers(1, 60, rows).astype(np.int32)
    table, refs = owned(g, rows, width, pages, start, block)
    parents = np.array([0, 0, 0, 3, 3, 3], np.int32)
    counts = np.full(rows, 7, np.int32)
    there, t, n, r = up(pool), dev(table), dev(start), dev(refs)
    par, cnt, keep = dev(parents), dev(counts), i32([1 << 20] * rows)
    kp.fork_kv_rows(par, *up(pool), t.clone(), n.clone(), r.clone())  # loads the code
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        kp.free_kv_rows(keep, t, n, r, block=block)
        ok1 = kp.fork_kv_rows(par, *there, t, n, r)
        ok2 = kp.reserve_kv_pages(*there, t, n, cnt, r)
        n.add_(cnt)
        live, moved = kp.compact_kv_pages(*there, t, r)
    same([*there, t, n, r], [*pool, table, start, refs], "capturing runs nothing")
    lengths = start
    for step in range(4):
        ks = [3, 0, 9, 1 << 20, 20, 1 << 20] if step % 2 else [1 << 20] * rows
        keep.copy_(i32(ks))
        graph.replay()
        R.free(ks, table, lengths, refs, block)
        want = (R.fork(list(parents), pool, table, lengths, refs, block), R.reserve(pool, table, lengths, counts, refs, block))
        lengths += counts
        want_live, want_moved = R.compact(pool, table, refs)
        torch.cuda.synchronize()
        assert (int(ok1), int(ok2), int(live)) == (*want, want_live)
        same([*there, t, n, r], [*pool, table, lengths, refs], f"replay {step}")
        np.testing.assert_array_equal(host(moved), want_moved)
        torch.zeros(1 << 20, device=DEV).add_(1)  # the program's own work between replays
