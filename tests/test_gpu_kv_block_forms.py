"""Attention over the block-scaled cache in every form that its plan chooses between: E4M3 NaNs that some rows attend and others
must not see, and the same bits at every repetition. Bounds and helpers are those of tests/test_gpu_kv_block.py."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.conftest import print_case
from tests.test_gpu_kv_block import DEV, check_attention, fill_valid, i32, make_cache, to_dev

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def kv():
    from scratch_llm_amd.quant import kv_block

    return kv_block


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("d,t", [(64, 1), (64, 20), (64, 40), (128, 1), (128, 20), (128, 40), (256, 1), (256, 14), (256, 20)])
def test_nan_codes_reach_who_attends_them(kv, d, t, block):
    """Four query heads a kv head: 4 rows (the direct kernel, one tile of 16 rows), 80 (the direct kernel with two tiles; heads of
    256 the tile kernel), 160 (the tile kernel), 56 of heads of 256 (the direct kernel). NaN values and keys among the new
    tokens, in an old token of a whole step and of a masked one; every byte behind the rows' last position is random."""
    print_case("kv attention nan", d, t, block)
    hkv, h = 2, 8
    starts = [70, 5, 127]
    width = (127 + t) // block + 3
    pages = 3 * width
    cache = fill_valid(make_cache(kv, pages, hkv, d, block, "e4m3", d + t), "e4m3", block)
    noise = make_cache(kv, pages, hkv, d, block, "e4m3", 10)
    table = np.random.default_rng(t).permutation(pages).reshape(3, width).astype(np.int32)

    def put(b, pos, head, dim, key):
        p = table[b, pos // block]
        if key:
            cache[0][p, head, pos % block, dim] = 0x7F
        else:
            cache[1][p, head, dim, pos % block] = 0xFF

    for b in range(3):
        end = starts[b] + t
        for i in range(width):
            p, keep = table[b, i], min(max(end - i * block, 0), block)
            cache[0][p, :, keep:] = noise[0][p, :, keep:]
            cache[1][p, :, :, keep:] = noise[1][p, :, :, keep:]
            if keep == 0:
                cache[2][p] = cache[3][p] = np.nan
        put(b, end - 1, 0, 7, False)
        put(b, starts[b] + t // 2, 1, d - 1, False)
        if t > 8:
            put(b, end - 3, 1, 11, True)
            put(b, starts[b] + 1, 0, d // 2 + 1, False)
    put(0, 3, 0, 33, False)   # all of its step is attended by every row
    put(2, 120, 1, 62, False)
    q = torch.randn(3, t, h, d, generator=torch.Generator().manual_seed(t)).bfloat16()
    with np.errstate(invalid="ignore"):
        check_attention(kv, cache, "e4m3", q, table, starts, None)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("b,t,h,hkv,d,block", [(1, 1, 32, 8, 128, 64), (5, 1, 8, 2, 64, 16), (3, 5, 32, 8, 128, 32), (2, 20, 8, 2, 128, 64),
                                               (2, 70, 8, 2, 128, 64), (2, 70, 8, 2, 64, 16), (2, 6, 4, 1, 256, 128), (1, 40, 4, 1, 256, 32)])
def test_repeats_itself_bit_for_bit(kv, b, t, h, hkv, d, block, fmt):
    """The same call on the same cache, alone, behind other calls and beside them on another stream: no sum's order depends on
    which workgroup ends first."""
    print_case("kv attention repeats", b, t, h, hkv, d, block, fmt)
    ctx = 3000
    width = (ctx + t) // block + 1
    dev = to_dev(fill_valid(make_cache(kv, b * width, hkv, d, block, fmt, 1), fmt, 2), fmt)
    table = i32(np.random.default_rng(3).permutation(b * width).reshape(b, width))
    starts = i32([ctx - 700 * i for i in range(b)])
    g = torch.Generator().manual_seed(4)
    q, other = (torch.randn(b, t, h, d, generator=g).bfloat16().to(DEV) for _ in range(2))
    want = kv.attend_kv_blocks(q, *dev, table, starts)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(6):
        with torch.cuda.stream(side):
            kv.attend_kv_blocks(other, *dev, table, starts)
        assert torch.equal(kv.attend_kv_blocks(q, *dev, table, starts), want)
        kv.attend_kv_blocks(other, *dev, table, starts)
    torch.cuda.current_stream().wait_stream(side)
