"""What the pages of the block-scaled cache refuse, and that the oracle keeps its own books: CPU only, no kernel launches."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import kv_pages_ref as R
from scratch_llm_amd import _lib
from scratch_llm_amd.quant import kv_block, kv_pages

I32 = torch.int32


def pool(pages=6, hkv=2, d=64, block=16, layers=None, dtype=torch.int8):
    one = kv_block.new_kv_blocks(pages, hkv, d, block=block, dtype=dtype, device="cpu")
    return list(one) if layers is None else [x[None].repeat(layers, *[1] * x.ndim) for x in one]


def zeros(*shape):
    return torch.zeros(*shape, dtype=I32)


def calls(c, table, rows, refs):
    return {"fork": lambda: kv_pages.fork_kv_rows(rows, *c, table, rows, refs),
            "reserve": lambda: kv_pages.reserve_kv_pages(*c, table, rows, rows, refs),
            "compact": lambda: kv_pages.compact_kv_pages(*c, table, refs),
            "free": lambda: kv_pages.free_kv_rows(rows, table, rows, refs, block=16),
            "copy": lambda: kv_pages.copy_kv_pages(rows, rows, *c)}


def test_refuse_bad_pools():
    for layers in (None, 3):
        c = pool(layers=layers)
        bad = [([c[0], c[1].transpose(-1, -2), c[2], c[3]], "v_codes"), ([c[0], c[1].view(torch.float8_e4m3fn), c[2], c[3]], "v_codes"),
               ([c[0], c[1], c[2][..., :1], c[3]], "scales"), ([c[0], c[1], c[2].double(), c[3]], "scales"),
               ([c[0][None, None], c[1], c[2], c[3]], "k_codes"), ([c[0][0, 0], c[1], c[2], c[3]], "k_codes"),
               ([c[0], c[1], c[2].transpose(-1, -2).contiguous().transpose(-1, -2), c[3]], "contiguous"),
               ([c[0][..., :48], c[1], c[2], c[3]], "head_dim"), ([c[0][..., :8, :], c[1], c[2], c[3]], "block")]
        for cc, what in bad:
            for name in ("fork", "reserve", "compact", "copy"):
                with pytest.raises(ValueError, match=what):
                    calls(cc, zeros(2, 3), zeros(2), zeros(6))[name]()
    with pytest.raises(TypeError, match="codes must be"):
        c = pool()
        kv_pages.copy_kv_pages(zeros(1), zeros(1), c[0].view(torch.uint8), c[1].view(torch.uint8), c[2], c[3])


def test_refuse_bad_tables():
    c = pool()
    good = (zeros(2, 3), zeros(2), zeros(6))
    bad = [((zeros(2, 3).long(), *good[1:]), "block_table"), ((zeros(3, 2).t(), *good[1:]), "block_table"),
           ((zeros(2, 0), *good[1:]), "block_table"), ((zeros(6), *good[1:]), "block_table"),
           ((good[0], zeros(3), good[2]), "parents|starts|keep"), ((good[0], zeros(2).long(), good[2]), "parents|starts|keep"),
           ((good[0], zeros(4)[::2], good[2]), "parents|starts|keep"), ((good[0], good[1], zeros(6).long()), "refs"),
           ((good[0], good[1], zeros(6, 1)), "refs")]
    for args, what in bad:
        todo = calls(c, *args)
        for name in ("fork", "reserve", "free") if "parents" in what else ("fork", "reserve", "free", "compact"):
            with pytest.raises(ValueError, match=what):
                todo[name]()
    for name in ("fork", "reserve", "compact"):  # refs of another pool
        with pytest.raises(ValueError, match="refs"):
            calls(c, good[0], good[1], zeros(5))[name]()
    with pytest.raises(ValueError, match="block_table"):
        kv_pages.fork_kv_rows(zeros(0), *c, zeros(0, 3), zeros(0), zeros(6))
    with pytest.raises(ValueError, match="block must"):
        kv_pages.free_kv_rows(zeros(2), zeros(2, 3), zeros(2), zeros(6), block=24)
    with pytest.raises(ValueError, match="dst"):
        kv_pages.copy_kv_pages(zeros(2), zeros(3), *c)
    with pytest.raises(ValueError, match="src"):
        kv_pages.copy_kv_pages(zeros(2, 1), zeros(2, 1), *c)


def test_refuse_cpu_tensors():
    for call in calls(pool(), zeros(2, 3), zeros(2), zeros(6)).values():
        with pytest.raises(RuntimeError, match="device tensors"):
            call()


def test_entry_points_refuse():
    lib, p, n = _lib.load(), ctypes.c_void_p(256), None
    good = dict(L=1, B=2, hkv=2, hd=64, block=16, pages=8, width=4)

    def fork(ws=1 << 20, wsp=p, **change):
        a = {**good, **change}
        return lib.sqx_kvpages_fork(p, p, p, p, p, p, p, p, a["L"], a["B"], a["hkv"], a["hd"], a["block"], a["pages"], a["width"], p,
                                    wsp, ws, n)

    for change, what in ((dict(L=0), b"layers"), (dict(L=1 << 16), b"layers"), (dict(hd=96), b"hd=96"), (dict(block=8), b"block=8"),
                         (dict(hkv=0), b"Hkv=0"), (dict(pages=0), b"pages=0"), (dict(pages=1 << 31), b"pages="), (dict(B=0), b"no rows"),
                         (dict(B=1 << 16), b"B=65536"), (dict(width=0), b"0 blocks"), (dict(width=1 << 27), b"blocks"),
                         (dict(L=60000, B=60000), b"too many")):
        assert fork(**change) == -1 and what in lib.sqx_last_error(), (change, lib.sqx_last_error())
    need = lib.sqx_kvpages_fork_workspace_bytes(2, 4, 8)
    assert need > 0 and fork(ws=need - 1) == -3 and fork(wsp=n) == -3 and fork(wsp=ctypes.c_void_p(264)) == -3
    assert lib.sqx_kvpages_copy(p, p, -1, p, p, p, p, 1, 2, 64, 16, 8, n) == -1
    assert lib.sqx_kvpages_copy(p, p, 0, n, n, n, n, 1, 2, 64, 16, 8, n) == 0
    assert lib.sqx_kvpages_copy(p, p, 1, ctypes.c_void_p(8), p, p, p, 1, 2, 64, 16, 8, n) == -1 and b"aligned" in lib.sqx_last_error()
    assert lib.sqx_kvpages_copy(p, p, (1 << 31) - 1, p, p, p, p, 8, 2, 64, 16, 8, n) == -1 and b"too many" in lib.sqx_last_error()
    assert lib.sqx_kvpages_free(p, n, p, p, 2, 16, 8, 4, n) == -1 and lib.sqx_kvpages_free(n, n, n, n, 0, 16, 8, 4, n) == 0
    assert lib.sqx_kvpages_fork_workspace_bytes(0, 4, 8) == lib.sqx_kvpages_reserve_workspace_bytes(1, 4, 0) == 0
    assert lib.sqx_kvpages_fork_workspace_bytes(65535, 1000, 1 << 30) > 1 << 32  # not in 32 bits


def books(table, refs):
    """refs says how often the table names each page."""
    want = np.bincount(table[table >= 0].ravel(), minlength=len(refs))
    assert np.array_equal(refs, want)


def test_oracle_keeps_its_books():
    g = np.random.default_rng(3)
    block, pages, rows, width = 16, 40, 6, 9
    for trial in range(60):
        pool = [g.integers(0, 9, (2, pages, 3)) for _ in range(4)]
        table = np.full((rows, width), -1, np.int32)
        lengths, refs = np.zeros(rows, np.int32), np.zeros(pages, np.int32)
        text = [[] for _ in range(rows)]  # what every row's tokens are, by the page's content at each block
        for step in range(12):
            what = g.integers(0, 4)
            before = (table.copy(), lengths.copy(), refs.copy(), [x.copy() for x in pool])
            if what == 0:
                counts = g.integers(0, 30, rows)
                counts = np.minimum(counts, width * block - lengths)
                ok = R.reserve(pool, table, lengths, counts, refs, block)
                if ok:
                    for b in range(rows):
                        if counts[b]:
                            for j in range(lengths[b] // block, (lengths[b] + counts[b] + block - 1) // block):
                                assert refs[table[b, j]] == 1
                    lengths += counts.astype(np.int32)
            elif what == 1:
                parents = g.integers(-1, rows, rows)
                ok = R.fork(parents, pool, table, lengths, refs, block)
                if ok:
                    for b, p in enumerate(parents):
                        n = before[1][p] if p >= 0 else 0
                        assert lengths[b] == n
                        for j in range((n + block - 1) // block):  # the same content as the parent's
                            for x, y in zip(pool, before[3]):
                                assert np.array_equal(x[:, table[b, j]], y[:, before[0][p, j]])
            elif what == 2:
                keep = g.integers(-3, width * block, rows)
                R.free(keep, table, lengths, refs, block)
                ok = 1
            else:
                held = [[x[:, p].copy() for x in pool] for p in table[table >= 0]]
                live, moved = R.compact(pool, table, refs)
                assert (refs[:live] > 0).all() and (refs[live:] == 0).all()
                for p, content in zip(table[table >= 0], held):
                    assert all(np.array_equal(x[:, p], y) for x, y in zip(pool, content))
                ok = 1
            if not ok:
                assert all(np.array_equal(x, y) for x, y in zip((table, lengths, refs), before))
            books(table, refs)
