"""8-bit KV cache with one scale per block of tokens and head, on MI355X: write, read back, attend.

Where the per-head cache (:mod:`fp8_kv_per_head`, the reference's contract) calibrates one static scale
per head, this one scales every block of 16, 32, 64 or 128 tokens by what it holds, so nothing is
calibrated and nothing saturates, and int8 codes become usable. The cache of a layer is four tensors that
the caller owns:

* ``k_codes [pages, Hkv, block, D]`` and ``v_codes [pages, Hkv, D, block]``, ``torch.int8`` or
  ``torch.float8_e4m3fn`` (the dtype is the format; values are stored transposed, as the second product of
  attention reads them);
* ``k_scale``, ``v_scale`` fp32 ``[pages, Hkv]``. A code ``c`` stands for ``c * scale``.

``block_table`` int32 ``[B, width]`` names the page of each of a row's blocks; rows may share pages that
none of them writes. :func:`new_kv_blocks` allocates a layer. Everything here is device work on the
current stream and can be captured in a HIP graph; ``Int4DecodeLM.new_state(kv_dtype="int8_block")`` (or
``"fp8_block"``) decodes on such a cache.
"""

from __future__ import annotations

import functools
import math

import torch
from torch import Tensor

from scratch_llm_amd import _lib
from scratch_llm_amd.quant.fp8_weights import FP8_DTYPE
from scratch_llm_amd.rope import check_table

__all__ = ["BLOCKS", "HEAD_DIMS", "attend_kv_blocks", "new_kv_blocks", "read_kv_blocks", "write_kv_blocks"]

BLOCKS = (16, 32, 64, 128)
HEAD_DIMS = (64, 128, 256)
_F32, _I32 = torch.float32, torch.int32
_FMT = {torch.int8: _lib.KV_INT8, FP8_DTYPE: _lib.KV_E4M3}


def new_kv_blocks(pages: int, n_kv_heads: int, head_dim: int, *, block: int = 64, dtype: torch.dtype = torch.int8,
                  device: torch.device | str = "cuda") -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """An empty layer: ``(k_codes, v_codes, k_scale, v_scale)``, all zero."""
    if pages < 1 or n_kv_heads < 1:
        raise ValueError("new_kv_blocks: pages and n_kv_heads must be positive")
    _check_sizes(head_dim, block, dtype, "new_kv_blocks")
    # zeroed as bytes: torch has no fill kernel of its own for every 8-bit float
    k = torch.zeros(pages, n_kv_heads, block, head_dim, dtype=torch.uint8, device=device).view(dtype)
    v = torch.zeros(pages, n_kv_heads, head_dim, block, dtype=torch.uint8, device=device).view(dtype)
    s = torch.zeros(2, pages, n_kv_heads, dtype=torch.float32, device=device)
    return k, v, s[0], s[1]


def _check_sizes(head_dim: int, block: int, dtype: torch.dtype, fn: str) -> None:
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"{fn}: head_dim must be one of {HEAD_DIMS}, got {head_dim}")
    if block not in BLOCKS:
        raise ValueError(f"{fn}: block must be one of {BLOCKS}, got {block}")
    if dtype not in _FMT:
        raise TypeError(f"{fn}: codes must be torch.int8 or {FP8_DTYPE}, got {dtype}")


def _check_cache(kc: Tensor, vc: Tensor, ks: Tensor, vs: Tensor, table: Tensor, starts: Tensor, counts: Tensor | None,
                 batch: int, fn: str) -> tuple[int, int, int, int, int]:
    """Checks the cache, its table and the rows' positions; returns (pages, Hkv, block, D, format)."""
    shape = kc.shape
    if len(shape) != 4:
        raise ValueError(f"{fn}: k_codes must be [pages, Hkv, block, D], got {tuple(shape)}")
    pages, hkv, block, d = shape
    dtype = kc.dtype
    fmt = _FMT.get(dtype)
    if fmt is None or d not in HEAD_DIMS or block not in BLOCKS:
        _check_sizes(d, block, dtype, fn)
    if vc.shape != (pages, hkv, d, block) or vc.dtype != dtype:
        raise ValueError(f"{fn}: v_codes must be {(pages, hkv, d, block)} of {dtype}, got {tuple(vc.shape)} of {vc.dtype}")
    one = (pages, hkv)
    if ks.shape != one or vs.shape != one or ks.dtype != _F32 or vs.dtype != _F32:
        raise ValueError(f"{fn}: scales must be float32 {one}, got {tuple(ks.shape)} and {tuple(vs.shape)}")
    width = table.shape
    if len(width) != 2 or width[0] != batch or width[1] < 1 or table.dtype != _I32:
        raise ValueError(f"{fn}: block_table must be int32 [{batch}, width], got {tuple(width)} of {table.dtype}")
    rows = (batch,)
    if starts.shape != rows or starts.dtype != _I32:
        raise ValueError(f"{fn}: starts must be int32 [{batch}], got {tuple(starts.shape)} of {starts.dtype}")
    if counts is not None and (counts.shape != rows or counts.dtype != _I32):
        raise ValueError(f"{fn}: counts must be int32 [{batch}], got {tuple(counts.shape)} of {counts.dtype}")
    if not (kc.is_contiguous() and vc.is_contiguous() and ks.is_contiguous() and vs.is_contiguous() and table.is_contiguous()
            and starts.is_contiguous() and (counts is None or counts.is_contiguous())):
        raise ValueError(f"{fn}: codes, scales, block_table, starts and counts must be contiguous")
    return pages, hkv, block, d, fmt


def _rows(x: Tensor) -> tuple[Tensor, int, int, int]:
    """x and its strides of row, token and head where the kernels can take them, else those of a contiguous copy."""
    sb, st, sh, sd = x.stride()
    if sd == 1 and (sb | st | sh) & 7 == 0 and x.data_ptr() & 15 == 0:
        return x, sb, st, sh
    x = x.contiguous()
    if x.data_ptr() & 15:
        x = x.clone()
    _, t, h, d = x.shape  # not x.stride(): a dimension of one token or head keeps any
    return x, t * h * d, h * d, d


def write_kv_blocks(k: Tensor, v: Tensor, k_codes: Tensor, v_codes: Tensor, k_scale: Tensor, v_scale: Tensor,
                    block_table: Tensor, starts: Tensor, counts: Tensor | None = None, *, q: Tensor | None = None,
                    rope: tuple[Tensor, Tensor] | None = None, interleaved: bool = True) -> Tensor | None:
    """Quantize and store new tokens ``k, v [B, T, Hkv, D]`` at positions ``starts[b] ..`` of every row.

    ``counts`` (int32 ``[B]``; default T) is how many of a row's T tokens are stored. With ``rope=(cos, sin)``
    (:func:`scratch_llm_amd.rope.rope_table`; a multiple of 16 columns) keys are rotated by position first and
    rounded to their type, and the rotated ``q [B, T, H, D]`` is returned, if given (all T tokens), as
    :func:`~scratch_llm_amd.rope.apply_rope` rotates it.

    A block whose first token is written takes the scale ``amax * fl(1 / 127)`` (int8) or ``amax * fl(1 / 448)`` (E4M3)
    of the tokens written, an fp32 product, at least 1e-12. A block that keeps earlier tokens has its scale doubled until the new
    ones fit, and its codes halved with it: the rescales together cost a token less than one step of the
    block's final scale. Infinities saturate; a NaN is stored as NaN in E4M3 and as 0 in int8.

    So what a block's tokens lose depends on all that was ever written into it, tokens that are written over later
    included. To take tokens out again, keep the open block's codes and scales beside and put them back.

    Tokens at a negative start, outside the table, or on a page id outside the cache are not stored. No page may be
    written twice by one call, by two rows or by two blocks of one."""
    fn = "write_kv_blocks"
    if k.ndim != 4 or k.shape != v.shape or k.dtype != v.dtype:
        raise ValueError(f"{fn}: k and v must be [B, T, Hkv, D] alike, got {tuple(k.shape)} of {k.dtype}, {tuple(v.shape)} of {v.dtype}")
    b, t, hkv, d = k.shape
    pages, hc, block, dc, fmt = _check_cache(k_codes, v_codes, k_scale, v_scale, block_table, starts, counts, b, fn)
    if (hkv, d) != (hc, dc):
        raise ValueError(f"{fn}: k has {hkv} heads of {d}, the cache {hc} heads of {dc}")
    dt = _lib.sqx_dtype(k.dtype)
    cos = sin = None
    rot = heads = 0
    if rope is not None:
        cos, sin = rope
        rot = check_table(cos, sin, d, fn)
        if rot % 16 != 0:
            raise ValueError(f"{fn}: the table rotates {rot} columns (a multiple of 16 is needed; rotate with apply_rope first)")
    if q is not None:
        if rope is None:
            raise ValueError(f"{fn}: q is only rotated here: give rope")
        if q.ndim != 4 or q.shape[0] != b or q.shape[1] != t or q.shape[3] != d or q.dtype != k.dtype:
            raise ValueError(f"{fn}: q must be [{b}, {t}, H, {d}] of {k.dtype}, got {tuple(q.shape)} of {q.dtype}")
    index = _lib.device_index(fn, k, v, k_codes, v_codes, k_scale, v_scale, block_table, starts, counts, q, cos, sin)
    k, k_sb, k_st, k_sh = _rows(k)
    v, v_sb, v_st, v_sh = _rows(v)
    qp = q_out = qo = cp = sp = None
    q_sb = q_st = q_sh = rope_rows = 0
    if rope is not None:
        cp, sp, rope_rows = cos.data_ptr(), sin.data_ptr(), cos.shape[0]
    if q is not None:
        heads = q.shape[2]
        q, q_sb, q_st, q_sh = _rows(q)
        q_out = torch.empty(b, t, heads, d, dtype=q.dtype, device=q.device)
        qp, qo = q.data_ptr(), q_out.data_ptr()
    _lib.launch(index, fn, _lib.load().sqx_kvblock_write, k.data_ptr(), v.data_ptr(), dt, k_sb, k_st, k_sh, v_sb, v_st, v_sh,
                qp, q_sb, q_st, q_sh, qo, cp, sp, rope_rows, rot, interleaved, fmt, k_codes.data_ptr(), v_codes.data_ptr(),
                k_scale.data_ptr(), v_scale.data_ptr(), block_table.data_ptr(), starts.data_ptr(), _lib.ptr(counts), b, t,
                heads, hkv, d, block, pages, block_table.shape[1])
    return q_out


def read_kv_blocks(k_codes: Tensor, v_codes: Tensor, k_scale: Tensor, v_scale: Tensor, block_table: Tensor,
                   starts: Tensor, tokens: int, counts: Tensor | None = None, *,
                   dtype: torch.dtype = torch.float32) -> tuple[Tensor, Tensor]:
    """``(k, v) [B, tokens, Hkv, D]``: the values of positions ``starts[b] .. starts[b] + tokens - 1`` of every row,
    ``fp32(code) * scale`` rounded once to ``dtype``. Zeros from ``counts[b]`` on, at a negative start, outside the
    table and on a page id outside the cache."""
    fn = "read_kv_blocks"
    b = block_table.shape[0] if block_table.ndim else 0
    pages, hkv, block, d, fmt = _check_cache(k_codes, v_codes, k_scale, v_scale, block_table, starts, counts, b, fn)
    if tokens < 0:
        raise ValueError(f"{fn}: tokens must not be negative, got {tokens}")
    dt = _lib.sqx_dtype(dtype)
    index = _lib.device_index(fn, k_codes, v_codes, k_scale, v_scale, block_table, starts, counts)
    k, v = (torch.empty(b, tokens, hkv, d, dtype=dtype, device=k_codes.device) for _ in range(2))
    _lib.launch(index, fn, _lib.load().sqx_kvblock_read, fmt, k_codes.data_ptr(), v_codes.data_ptr(), k_scale.data_ptr(),
                v_scale.data_ptr(), block_table.data_ptr(), starts.data_ptr(), _lib.ptr(counts), b, tokens, hkv, d, block,
                pages, block_table.shape[1], dt, k.data_ptr(), v.data_ptr())
    return k, v


@functools.lru_cache(maxsize=4096)
def _attention_workspace(b: int, t: int, h: int, hkv: int, d: int, block: int, width: int) -> int:
    return int(_lib.load().sqx_kvblock_attention_workspace_bytes(b, t, h, hkv, d, block, width))


def attend_kv_blocks(q: Tensor, k_codes: Tensor, v_codes: Tensor, k_scale: Tensor, v_scale: Tensor, block_table: Tensor,
                     starts: Tensor, counts: Tensor | None = None, *, scale: float | None = None,
                     out: Tensor | None = None) -> Tensor:
    """Causal attention of new tokens ``q [B, T, H, D]`` (bfloat16 or float16) over a cache that holds them already.

    Token t of row b stands at position ``starts[b] + t`` and attends every position at and before it, ``H / Hkv``
    query heads to a kv head; ``scale`` defaults to ``1 / sqrt(D)``. Tokens from ``counts[b]`` on are left as they are
    in ``out`` (in a new output they are zero). A token at a negative position attends nothing and gets zeros; one
    that attends a position on a page id outside the cache gets NaN. Positions past the table do not exist. The work is laid out
    for the table's width, as the lengths are on the device: with one row and a few thousand keys a table many times as wide
    costs a fifth."""
    fn = "attend_kv_blocks"
    if q.ndim != 4:
        raise ValueError(f"{fn}: q must be [B, T, H, D], got {tuple(q.shape)}")
    b, t, h, d = q.shape
    pages, hkv, block, dc, fmt = _check_cache(k_codes, v_codes, k_scale, v_scale, block_table, starts, counts, b, fn)
    if d != dc or h % hkv != 0:
        raise ValueError(f"{fn}: q has {h} heads of {d}, the cache {hkv} heads of {dc}")
    dt = _lib.sqx_dtype(q.dtype)
    if dt == _lib.DTYPE_F32:
        raise TypeError(f"{fn}: q must be bfloat16 or float16, got {q.dtype}")
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    elif not (0.0 < scale <= 1.0e30):
        raise ValueError(f"{fn}: scale must be positive and at most 1e30, got {scale}")
    index = _lib.device_index(fn, q, k_codes, v_codes, k_scale, v_scale, block_table, starts, counts, out)
    q, q_sb, q_st, q_sh = _rows(q)
    if out is None:
        out = (torch.empty if counts is None else torch.zeros)(b, t, h, d, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
        raise ValueError(f"{fn}: out must be contiguous {tuple(q.shape)} of {q.dtype}")
    width = block_table.shape[1]
    nb = _attention_workspace(b, t, h, hkv, d, block, width)
    ws = torch.empty(nb // 4, dtype=_F32, device=q.device) if nb else None
    _lib.launch(index, fn, _lib.load().sqx_kvblock_attention, q.data_ptr(), dt, q_sb, q_st, q_sh, fmt, k_codes.data_ptr(),
                v_codes.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), block_table.data_ptr(), starts.data_ptr(),
                _lib.ptr(counts), b, t, h, hkv, d, block, pages, width, scale, out.data_ptr(), _lib.ptr(ws), nb)
    return out
