"""Rotary positions on MI355X: the table of a model's angles, with the usual long-context scalings, and the rotation.

The reference rotates interleaved pairs of whole heads with one table (``RotaryPositionalEmbedding``,
src/scratch_llm/model.py:185-224). :func:`apply_rope` also takes pairs laid out in halves and heads of
which only the first columns are rotated; the table's width says how many. The write into the
block-scaled cache (:func:`scratch_llm_amd.quant.kv_block.write_kv_blocks`) applies the same rotation to
a step's queries and keys, bit for bit.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch
from torch import Tensor

from scratch_llm_amd import _lib

__all__ = ["RopeScaling", "apply_rope", "rope_frequencies", "rope_table"]


@dataclass(frozen=True)
class RopeScaling:
    """How a table reaches past the ``original_len`` positions that a model was trained on.

    ``linear``: every frequency divided by ``factor``. ``by_parts``: wavelengths below ``original_len /
    high_freq_factor`` stay, those above ``original_len / low_freq_factor`` are divided, between them the
    two are mixed in proportion. ``yarn``: the mix runs over the pair's index, between the pairs that turn
    ``beta_fast`` and ``beta_slow`` times in ``original_len`` positions, and cos and sin carry
    ``attention_factor`` (by default ``0.1 ln(factor) + 1``)."""

    kind: str
    factor: float
    original_len: int = 0
    low_freq_factor: float = 1.0
    high_freq_factor: float = 4.0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    attention_factor: float | None = None

    def validate(self) -> None:
        if self.kind not in ("linear", "by_parts", "yarn"):
            raise ValueError(f"scaling kind must be 'linear', 'by_parts' or 'yarn', got {self.kind!r}")
        if not (math.isfinite(self.factor) and self.factor >= 1.0):
            raise ValueError(f"scaling factor must be at least 1, got {self.factor}")
        if self.kind != "linear" and self.original_len < 1:
            raise ValueError(f"{self.kind} scaling needs original_len, got {self.original_len}")
        if self.kind == "by_parts" and not 0.0 < self.low_freq_factor < self.high_freq_factor:
            raise ValueError("by_parts scaling needs 0 < low_freq_factor < high_freq_factor")
        if self.kind == "yarn" and not 0.0 < self.beta_slow < self.beta_fast:
            raise ValueError("yarn scaling needs 0 < beta_slow < beta_fast")


def rope_frequencies(rot_dim: int, theta: float = 10000.0, scaling: RopeScaling | None = None) -> tuple[Tensor, float]:
    """``(frequencies [rot_dim / 2] in float64, factor of cos and sin)``: ``theta^(-2i / rot_dim)``, scaled."""
    if rot_dim < 2 or rot_dim % 2 != 0:
        raise ValueError(f"rot_dim must be even and positive, got {rot_dim}")
    if not theta > 1.0:
        raise ValueError(f"theta must exceed 1, got {theta}")
    i = torch.arange(rot_dim // 2, dtype=torch.float64)
    freq = float(theta) ** (-2.0 * i / rot_dim)
    if scaling is None:
        return freq, 1.0
    scaling.validate()
    slow = freq / scaling.factor
    if scaling.kind == "linear":
        return slow, 1.0
    if scaling.kind == "by_parts":
        turns = scaling.original_len * freq / (2.0 * math.pi)  # over the trained length
        lo, hi = scaling.low_freq_factor, scaling.high_freq_factor
        keep = ((turns - lo) / (hi - lo)).clamp(0.0, 1.0)
        return slow + keep * (freq - slow), 1.0

    def pair_of(turns: float) -> float:  # the (fractional) pair that makes so many turns over the trained length
        return rot_dim * math.log(scaling.original_len / (turns * 2.0 * math.pi)) / (2.0 * math.log(theta))

    lo = max(math.floor(pair_of(scaling.beta_fast)), 0)
    hi = min(math.ceil(pair_of(scaling.beta_slow)), rot_dim - 1)
    ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
    att = scaling.attention_factor
    return freq + ramp * (slow - freq), (0.1 * math.log(scaling.factor) + 1.0) if att is None else float(att)


def rope_table(rot_dim: int, max_seq_len: int, theta: float = 10000.0, scaling: RopeScaling | None = None,
               device: torch.device | str | None = None) -> tuple[Tensor, Tensor]:
    """cos and sin, fp32 ``[max_seq_len, rot_dim / 2]``: angles, cosines and factors in float64 on the host, rounded
    once (an fp32 angle at position 100000 is off by up to 0.004). Interleaved and halved layouts share a table."""
    if max_seq_len < 1:
        raise ValueError(f"max_seq_len must be positive, got {max_seq_len}")
    freq, att = rope_frequencies(rot_dim, theta, scaling)
    ang = torch.outer(torch.arange(max_seq_len, dtype=torch.float64), freq)
    cos, sin = (ang.cos() * att).float(), (ang.sin() * att).float()
    return (cos, sin) if device is None else (cos.to(device), sin.to(device))


def check_table(cos: Tensor, sin: Tensor, head_dim: int, fn: str) -> int:
    """The rotated columns that a table covers; raises where it is no table for such heads."""
    shape = cos.shape
    if len(shape) != 2 or shape != sin.shape or shape[0] < 1 or shape[1] < 1:
        raise ValueError(f"{fn}: cos and sin must be [positions, rot / 2] alike, got {tuple(shape)} and {tuple(sin.shape)}")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise TypeError(f"{fn}: cos and sin must be float32, got {cos.dtype} and {sin.dtype}")
    if not (cos.is_contiguous() and sin.is_contiguous()):
        raise ValueError(f"{fn}: cos and sin must be contiguous")
    rot = 2 * shape[1]
    if rot > head_dim:
        raise ValueError(f"{fn}: the table rotates {rot} columns of heads of {head_dim}")
    return rot


def apply_rope(x: Tensor, positions: Tensor, cos: Tensor, sin: Tensor, *, interleaved: bool = True,
               out: Tensor | None = None) -> Tensor:
    """Rotate heads ``x [..., heads, d]`` by their tokens' ``positions [...]``.

    The first ``2 * cos.shape[1]`` columns of a head are rotated, in pairs (2i, 2i + 1) (``interleaved``) or
    (i, i + half); the others are copied. fp32 arithmetic with every product and sum rounded on its own,
    rounded once to ``x``'s type (float32, bfloat16 or float16). Positions outside the table take its first
    or last row. ``out`` may be ``x``."""
    fn = "apply_rope"
    shape = x.shape
    if len(shape) < 2:
        raise ValueError(f"{fn}: x must be [..., heads, d], got {tuple(shape)}")
    if positions.shape != shape[:-2]:
        raise ValueError(f"{fn}: positions {tuple(positions.shape)} do not match x {tuple(shape)}")
    heads, d = shape[-2], shape[-1]
    rot = check_table(cos, sin, d, fn)
    dt = _lib.sqx_dtype(x.dtype)
    if positions.dtype != torch.int32 and positions.dtype != torch.int64:
        raise TypeError(f"{fn}: positions must be int32 or int64, got {positions.dtype}")
    index = _lib.device_index(fn, x, positions, cos, sin, out)
    if x.stride(-1) != 1:
        x = x.contiguous()
    rows = x if len(shape) == 3 else x.reshape(-1, heads, d)  # a copy where the leading strides do not combine
    if positions.dtype == torch.int64:
        positions = positions.clamp(0, cos.shape[0] - 1).to(torch.int32)
    if not positions.is_contiguous():
        positions = positions.contiguous()
    if out is None:
        out = to = torch.empty(*shape, dtype=x.dtype, device=x.device)
        on, oh = heads * d, d
    else:
        if out.shape != shape or out.dtype != x.dtype or out.stride(-1) != 1:
            raise ValueError(f"{fn}: out must be {tuple(shape)} of {x.dtype} with consecutive columns")
        try:
            to = out if len(shape) == 3 else out.view(-1, heads, d)
        except RuntimeError:
            raise ValueError(f"{fn}: the leading strides of out {out.stride()} do not combine") from None
        on, oh, _ = to.stride()
    xn, xh, _ = rows.stride()
    _lib.launch(index, fn, _lib.load().sqx_rope, rows.data_ptr(), dt, rows.shape[0], heads, d, xn, xh, positions.data_ptr(),
                cos.data_ptr(), sin.data_ptr(), cos.shape[0], rot, interleaved, to.data_ptr(), on, oh)
    return out
