"""Attention over the block-scaled KV cache of a batch whose rows share the first part of their contexts, on MI355X.

Several answers to one prompt, or many users behind one system prompt, name the same pages in front
(:func:`~scratch_llm_amd.quant.kv_pages.fork_kv_rows`). :func:`~scratch_llm_amd.quant.kv_block.attend_kv_blocks` reads these pages
once for every row; :func:`attend_shared_kv` reads them once for all rows of a group and joins that with each row's own keys.

:func:`plan_shared_kv` finds on the device what the rows share. A plan is for one number of tokens a row and one set of heads; all
layers and all steps use it until the groups or their shared pages change. Both calls issue device work on the current stream
only and can be captured in a HIP graph.
"""

from __future__ import annotations

import functools
import math
from dataclasses import dataclass

import torch
from torch import Tensor

from scratch_llm_amd import _lib
from scratch_llm_amd.quant.kv_block import _check_cache, _check_sizes, _rows

__all__ = ["MAX_ROWS", "SharedKV", "attend_shared_kv", "plan_shared_kv"]

MAX_ROWS = 4096  # rows of a batch
_I32 = torch.int32


@dataclass(frozen=True)
class SharedKV:
    """What the rows of a batch share, as :func:`plan_shared_kv` found it (``plan``, on the device), and what it was made for."""

    plan: Tensor
    batch: int
    tokens: int
    heads: int
    kv_heads: int
    head_dim: int
    block: int
    width: int


@functools.lru_cache(maxsize=256)
def _plan_bytes(b: int, t: int, h: int, hkv: int, d: int) -> int:
    return int(_lib.load().sqx_kvshared_plan_bytes(b, t, h, hkv, d))


@functools.lru_cache(maxsize=256)
def _workspace(b: int, t: int, h: int, hkv: int, d: int, block: int, width: int) -> int:
    return int(_lib.load().sqx_kvshared_attention_workspace_bytes(b, t, h, hkv, d, block, width))


def plan_shared_kv(block_table: Tensor, starts: Tensor, leaders: Tensor, *, block: int, tokens: int, heads: int, kv_heads: int,
                   head_dim: int, out: SharedKV | None = None) -> SharedKV:
    """Find what the rows of ``block_table`` int32 ``[B, width]`` share, for attention of ``tokens`` new tokens a row.

    Rows with the same number of 0 or above in ``leaders`` (int32 ``[B]``, for instance the row that each was forked from) make a
    group; -1 stands alone. A group shares the blocks in front that all of its rows name alike, as far as they lie whole before
    every row's ``starts[b]`` (int32 ``[B]``), in multiples of 64 tokens (128 with heads of 64). Rows shorter than that stand
    alone (an emptied row stays with its leader's number); longer ones with less in common are better put into a group of their own.

    The plan holds while a group's rows and the table's entries of its shared blocks stay, however far the rows
    grow. (A row whose start falls behind the shared blocks is attended for itself.) ``out``: a plan of the same sizes to write
    over, as a captured graph needs it."""
    fn = "plan_shared_kv"
    if block_table.ndim != 2 or block_table.shape[0] < 1 or block_table.shape[1] < 1:
        raise ValueError(f"{fn}: block_table must be int32 [B, width], got {tuple(block_table.shape)}")
    b, width = block_table.shape
    for name, x, shape in (("block_table", block_table, (b, width)), ("starts", starts, (b,)), ("leaders", leaders, (b,))):
        if tuple(x.shape) != shape or x.dtype != _I32 or not x.is_contiguous():
            raise ValueError(f"{fn}: {name} must be contiguous int32 {list(shape)}, got {tuple(x.shape)} of {x.dtype}")
    if b > MAX_ROWS:
        raise ValueError(f"{fn}: {b} rows, at most {MAX_ROWS}")
    _check_sizes(head_dim, block, torch.int8, fn)
    if not 1 <= tokens < 1 << 20:
        raise ValueError(f"{fn}: tokens must be positive and below {1 << 20}, got {tokens}")
    if kv_heads < 1 or heads < 1 or heads % kv_heads != 0:
        raise ValueError(f"{fn}: {heads} heads over {kv_heads} kv heads")
    sizes = (b, tokens, heads, kv_heads, head_dim)
    nb = _plan_bytes(*sizes)
    if out is None:
        out = SharedKV(torch.empty(nb, dtype=torch.uint8, device=block_table.device), *sizes, block, width)
    elif (out.batch, out.tokens, out.heads, out.kv_heads, out.head_dim, out.block, out.width) != (*sizes, block, width):
        raise ValueError(f"{fn}: out is a plan for other sizes ({out.batch} rows of {out.tokens} tokens, {out.heads} heads over {out.kv_heads} "
                         f"of {out.head_dim}, blocks of {out.block}, a table of {out.width})")
    index = _lib.device_index(fn, block_table, starts, leaders, out.plan)
    _lib.launch(index, fn, _lib.load().sqx_kvshared_plan, block_table.data_ptr(), starts.data_ptr(), leaders.data_ptr(), *sizes, block,
                width, out.plan.data_ptr(), nb)
    return out


def attend_shared_kv(q: Tensor, k_codes: Tensor, v_codes: Tensor, k_scale: Tensor, v_scale: Tensor, block_table: Tensor, starts: Tensor,
                     counts: Tensor | None = None, *, shared: SharedKV, scale: float | None = None, out: Tensor | None = None) -> Tensor:
    """:func:`~scratch_llm_amd.quant.kv_block.attend_kv_blocks`, the keys that ``shared`` names read once for each group.

    Same arguments, and the same result up to the order of its sums: the parts are computed apart and joined in fp32."""
    fn = "attend_shared_kv"
    if q.ndim != 4:
        raise ValueError(f"{fn}: q must be [B, T, H, D], got {tuple(q.shape)}")
    b, t, h, d = q.shape
    pages, hkv, block, dc, fmt = _check_cache(k_codes, v_codes, k_scale, v_scale, block_table, starts, counts, b, fn)
    if d != dc or h % hkv != 0:
        raise ValueError(f"{fn}: q has {h} heads of {d}, the cache {hkv} heads of {dc}")
    width = block_table.shape[1]
    if (shared.batch, shared.tokens, shared.heads, shared.kv_heads, shared.head_dim, shared.block, shared.width) != (b, t, h, hkv, d, block, width):
        raise ValueError(f"{fn}: the plan is for {shared.batch} rows of {shared.tokens} tokens, {shared.heads} heads over {shared.kv_heads} of "
                         f"{shared.head_dim}, blocks of {shared.block}, a table of {shared.width}; the call has {b} rows of {t}, {h} over {hkv} of "
                         f"{d}, {block}, {width}")
    dt = _lib.sqx_dtype(q.dtype)
    if dt == _lib.DTYPE_F32:
        raise TypeError(f"{fn}: q must be bfloat16 or float16, got {q.dtype}")
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    elif not (0.0 < scale <= 1.0e30):
        raise ValueError(f"{fn}: scale must be positive and at most 1e30, got {scale}")
    index = _lib.device_index(fn, q, k_codes, v_codes, k_scale, v_scale, block_table, starts, counts, shared.plan, out)
    q, q_sb, q_st, q_sh = _rows(q)
    if out is None:
        out = (torch.empty if counts is None else torch.zeros)(b, t, h, d, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
        raise ValueError(f"{fn}: out must be contiguous {tuple(q.shape)} of {q.dtype}")
    nb = _workspace(b, t, h, hkv, d, block, width)
    ws = torch.empty(nb, dtype=torch.uint8, device=q.device) if nb else None
    _lib.launch(index, fn, _lib.load().sqx_kvshared_attention, q.data_ptr(), dt, q_sb, q_st, q_sh, fmt, k_codes.data_ptr(),
                v_codes.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), block_table.data_ptr(), starts.data_ptr(),
                _lib.ptr(counts), b, t, h, hkv, d, block, pages, width, scale, shared.plan.data_ptr(), shared.plan.numel(), out.data_ptr(),
                _lib.ptr(ws), nb)
    return out
