"""The pages of the block-scaled KV cache on MI355X: handing out, sharing, copying, releasing and moving them.

:mod:`~scratch_llm_amd.quant.kv_block` writes and reads pages that a row's ``block_table`` names; here is who gets which.
Besides the cache and the table, the caller owns ``lengths`` int32 ``[B]`` (tokens of every row) and ``refs`` int32 ``[pages]``,
how many table entries name a page: 0 means free. (A caller may hold pages of its own by counting them up; only
:func:`compact_kv_pages` has to be told of them, see there.) A table entry of -1, or outside the pool, names no page.

The cache is that of one layer, ``k_codes [pages, Hkv, block, D]`` and so on, or of all layers of a model with one table,
``[layers, pages, Hkv, block, D]`` and scales ``[layers, pages, Hkv]``.

* :func:`reserve_kv_pages` gives rows the pages of their next tokens, :func:`free_kv_rows` takes pages back;
* :func:`fork_kv_rows` makes rows continuations of others (several answers to a prompt, beams): full pages are shared, the page
  that a row goes on writing to is its own;
* :func:`copy_kv_pages` copies pages, :func:`compact_kv_pages` moves those in use to the front of the pool.

Everything is device work on the current stream and can be captured in a HIP graph: nothing is read back, so a call that finds
too few free pages changes nothing and says so in the int32 ``[1]`` it returns (1: done, 0: not). Free pages are taken
from the lowest on, row after row, so equal calls give equal tables. ``Int4DecodeLM.new_state(kv_pages=...)`` decodes on such
a pool.
"""

from __future__ import annotations

import functools

import torch
from torch import Tensor

from scratch_llm_amd import _lib
from scratch_llm_amd.quant.kv_block import BLOCKS, _check_sizes

__all__ = ["compact_kv_pages", "copy_kv_pages", "fork_kv_rows", "free_kv_rows", "reserve_kv_pages"]

_F32, _I32 = torch.float32, torch.int32


def _check_pool(kc: Tensor, vc: Tensor, ks: Tensor, vs: Tensor, fn: str) -> tuple[int, int, int, int, int]:
    """Checks a cache of one layer or of several; returns (layers, Hkv, D, block, pages)."""
    shape = kc.shape
    if len(shape) not in (4, 5):
        raise ValueError(f"{fn}: k_codes must be [pages, Hkv, block, D] or [layers, pages, Hkv, block, D], got {tuple(shape)}")
    layers = shape[0] if len(shape) == 5 else 1
    pages, hkv, block, d = shape[-4:]
    _check_sizes(d, block, kc.dtype, fn)
    if vc.shape != (*shape[:-2], d, block) or vc.dtype != kc.dtype:
        raise ValueError(f"{fn}: v_codes must be {(*shape[:-2], d, block)} of {kc.dtype}, got {tuple(vc.shape)} of {vc.dtype}")
    one = shape[:-2]
    if ks.shape != one or vs.shape != one or ks.dtype != _F32 or vs.dtype != _F32:
        raise ValueError(f"{fn}: scales must be float32 {tuple(one)}, got {tuple(ks.shape)} and {tuple(vs.shape)}")
    if not (kc.is_contiguous() and vc.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()):
        raise ValueError(f"{fn}: codes and scales must be contiguous")
    if layers < 1 or pages < 1 or hkv < 1:
        raise ValueError(f"{fn}: an empty cache {tuple(shape)}")
    return layers, hkv, d, block, pages


def _check_ints(fn: str, shape: tuple[int, ...], **tensors: Tensor) -> None:
    """Every tensor is int32 of the shape, without gaps."""
    for name, x in tensors.items():
        if tuple(x.shape) != shape or x.dtype != _I32 or not x.is_contiguous():
            raise ValueError(f"{fn}: {name} must be contiguous int32 {list(shape)}, got {tuple(x.shape)} of {x.dtype}")


def _check_table(table: Tensor, refs: Tensor, pages: int | None, fn: str, rows: bool = True) -> tuple[int, int]:
    if table.ndim != 2 or table.shape[1] < 1 or (rows and table.shape[0] < 1):
        raise ValueError(f"{fn}: block_table must be [B, width], got {tuple(table.shape)}")
    _check_ints(fn, tuple(table.shape), block_table=table)
    if refs.ndim != 1 or refs.shape[0] < 1:
        raise ValueError(f"{fn}: refs must be int32 [pages], got {tuple(refs.shape)}")
    _check_ints(fn, (refs.shape[0] if pages is None else pages,), refs=refs)
    return table.shape[0], table.shape[1]


@functools.lru_cache(maxsize=4096)
def _workspace(what: str, *sizes: int) -> int:
    return int(getattr(_lib.load(), f"sqx_kvpages_{what}_workspace_bytes")(*sizes))


def copy_kv_pages(src: Tensor, dst: Tensor, k_codes: Tensor, v_codes: Tensor, k_scale: Tensor, v_scale: Tensor) -> None:
    """Copy page ``src[i]`` to page ``dst[i]`` (int32 ``[n]`` both), codes and scales of all layers.

    Pairs with an id outside the pool, or the same one twice, are left out. No page may be written by two pairs of one
    call, or written by one and read by another."""
    fn = "copy_kv_pages"
    layers, hkv, d, block, pages = _check_pool(k_codes, v_codes, k_scale, v_scale, fn)
    if src.ndim != 1:
        raise ValueError(f"{fn}: src must be int32 [n], got {tuple(src.shape)}")
    _check_ints(fn, tuple(src.shape), src=src, dst=dst)
    index = _lib.device_index(fn, src, dst, k_codes, v_codes, k_scale, v_scale)
    _lib.launch(index, fn, _lib.load().sqx_kvpages_copy, src.data_ptr(), dst.data_ptr(), src.shape[0], k_codes.data_ptr(),
                v_codes.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), layers, hkv, d, block, pages)


def fork_kv_rows(parents: Tensor, k_codes: Tensor, v_codes: Tensor, k_scale: Tensor, v_scale: Tensor, block_table: Tensor,
                 lengths: Tensor, refs: Tensor) -> Tensor:
    """Make every row b go on from row ``parents[b]`` (int32 ``[B]``) as that was before the call, all rows at once.

    A row that is its own parent stays as it is; a parent outside ``0 .. B - 1`` empties the row. Any other row takes
    its parent's length and shares its full pages; the page that the next token goes to, if the parent has begun it, is
    copied to a free page. (If the parent does not go on from itself, the first row that goes on from it takes that page over
    instead.) What a row held before is released first, and may be handed out by the same call. A page that further rows
    held before, after a cut for instance, stays theirs too: :func:`reserve_kv_pages` parts them. Returns int32 ``[1]``: 1, or 0 if
    there are too few free pages; nothing is changed then."""
    fn = "fork_kv_rows"
    layers, hkv, d, block, pages = _check_pool(k_codes, v_codes, k_scale, v_scale, fn)
    b, width = _check_table(block_table, refs, pages, fn)
    _check_ints(fn, (b,), parents=parents, lengths=lengths)
    index = _lib.device_index(fn, parents, k_codes, v_codes, k_scale, v_scale, block_table, lengths, refs)
    ok = torch.empty(1, dtype=_I32, device=refs.device)
    nb = _workspace("fork", b, width, pages)
    ws = torch.empty(nb // 4, dtype=_I32, device=refs.device)
    _lib.launch(index, fn, _lib.load().sqx_kvpages_fork, parents.data_ptr(), k_codes.data_ptr(), v_codes.data_ptr(),
                k_scale.data_ptr(), v_scale.data_ptr(), block_table.data_ptr(), lengths.data_ptr(), refs.data_ptr(), layers, b, hkv, d,
                block, pages, width, ok.data_ptr(), ws.data_ptr(), nb)
    return ok


def reserve_kv_pages(k_codes: Tensor, v_codes: Tensor, k_scale: Tensor, v_scale: Tensor, block_table: Tensor, starts: Tensor,
                     counts: Tensor, refs: Tensor) -> Tensor:
    """Make positions ``starts[b] .. starts[b] + counts[b] - 1`` of every row (int32 ``[B]`` both) writable by that row alone.

    Blocks of these positions that have no page get a free one, whose codes and scales are what its last owner left; blocks
    whose page others hold too get a copy of it (all who write to it do, if several do; if nobody else holds it, it goes free).
    Blocks before them are left as they are. Rows with a negative start or no tokens get nothing, nor do positions past the table.
    Returns int32 ``[1]``: 1, or 0 if there are too few free pages; nothing is changed then."""
    fn = "reserve_kv_pages"
    layers, hkv, d, block, pages = _check_pool(k_codes, v_codes, k_scale, v_scale, fn)
    b, width = _check_table(block_table, refs, pages, fn)
    _check_ints(fn, (b,), starts=starts, counts=counts)
    index = _lib.device_index(fn, k_codes, v_codes, k_scale, v_scale, block_table, starts, counts, refs)
    ok = torch.empty(1, dtype=_I32, device=refs.device)
    nb = _workspace("reserve", b, width, pages)
    ws = torch.empty(nb // 4, dtype=_I32, device=refs.device)
    _lib.launch(index, fn, _lib.load().sqx_kvpages_reserve, k_codes.data_ptr(), v_codes.data_ptr(), k_scale.data_ptr(),
                v_scale.data_ptr(), block_table.data_ptr(), starts.data_ptr(), counts.data_ptr(), refs.data_ptr(), layers, b, hkv, d,
                block, pages, width, ok.data_ptr(), ws.data_ptr(), nb)
    return ok


def free_kv_rows(keep: Tensor, block_table: Tensor, lengths: Tensor, refs: Tensor, *, block: int) -> None:
    """Release what every row holds behind its first ``keep[b]`` tokens (int32 ``[B]``; 0 or less: all of it): pages of whole
    blocks behind them, whose entries become -1. ``lengths`` becomes the lesser of itself and ``keep``. A row that is cut inside
    a page that others hold too needs :func:`reserve_kv_pages` before it writes there."""
    fn = "free_kv_rows"
    if block not in BLOCKS:
        raise ValueError(f"{fn}: block must be one of {BLOCKS}, got {block}")
    b, width = _check_table(block_table, refs, None, fn)
    _check_ints(fn, (b,), keep=keep, lengths=lengths)
    index = _lib.device_index(fn, keep, block_table, lengths, refs)
    _lib.launch(index, fn, _lib.load().sqx_kvpages_free, keep.data_ptr(), block_table.data_ptr(), lengths.data_ptr(), refs.data_ptr(),
                b, block, refs.shape[0], width)


def compact_kv_pages(k_codes: Tensor, v_codes: Tensor, k_scale: Tensor, v_scale: Tensor, block_table: Tensor,
                     refs: Tensor) -> tuple[Tensor, Tensor]:
    """Move the pages in use (``refs`` above 0) to ids ``0 .. live - 1``: those behind take the free places before, in order.

    ``block_table`` and ``refs`` follow. Returns ``(live int32 [1], moved int32 [pages])``, ``moved`` the new id of every page
    that was in use and -1 for the others; a caller with further tables or pages of its own maps them by it."""
    fn = "compact_kv_pages"
    layers, hkv, d, block, pages = _check_pool(k_codes, v_codes, k_scale, v_scale, fn)
    b, width = _check_table(block_table, refs, pages, fn, rows=False)
    index = _lib.device_index(fn, k_codes, v_codes, k_scale, v_scale, block_table, refs)
    live = torch.empty(1, dtype=_I32, device=refs.device)
    moved = torch.empty(pages, dtype=_I32, device=refs.device)
    nb = _workspace("compact", pages)
    ws = torch.empty(nb // 4, dtype=_I32, device=refs.device)
    _lib.launch(index, fn, _lib.load().sqx_kvpages_compact, k_codes.data_ptr(), v_codes.data_ptr(), k_scale.data_ptr(),
                v_scale.data_ptr(), block_table.data_ptr(), refs.data_ptr(), layers, b, hkv, d, block, pages, width, live.data_ptr(),
                moved.data_ptr(), ws.data_ptr(), nb)
    return live, moved
