"""Sampling on MI355X: the next token of every row from its logits, with temperature, top-k, top-p and min-p.

The reference picks greedily or samples one row on the host (src/scratch_llm/sampling.py:80-86). Here a batch is sampled on the
device, with settings for all rows or for each, and without a sort of the vocabulary. Random numbers are inputs, so a run can be
repeated and a call captured in a HIP graph. :func:`scratch_llm_amd.speculative.verify_draft` draws behind drafted tokens.
"""

from __future__ import annotations

import functools
from dataclasses import dataclass

import torch
from torch import Tensor

from scratch_llm_amd import _lib

__all__ = ["MAX_VOCAB", "Sampling", "sample_tokens"]

MAX_VOCAB = 1 << 20


@dataclass(frozen=True)
class Sampling:
    """The settings of :func:`sample_tokens` (see there), numbers or tensors of one value a row."""

    temperature: float | Tensor = 1.0
    top_k: int | Tensor = 0
    top_p: float | Tensor = 1.0
    min_p: float | Tensor = 0.0

    def check(self, b: int, fn: str) -> None:
        for name, x, dtype in (("temperature", self.temperature, torch.float32), ("top_k", self.top_k, torch.int32),
                               ("top_p", self.top_p, torch.float32), ("min_p", self.min_p, torch.float32)):
            if isinstance(x, Tensor) and (tuple(x.shape) != (b,) or x.dtype != dtype or not x.is_contiguous()):
                raise ValueError(f"{fn}: {name} must be a number or contiguous {dtype} [{b}], got {tuple(x.shape)} of {x.dtype}")
        t, k, p, m = self.temperature, self.top_k, self.top_p, self.min_p
        if not isinstance(t, Tensor) and not (t == 0.0 or 1e-4 <= t <= 1e4):
            raise ValueError(f"{fn}: temperature must be 0 or within 1e-4 .. 1e4, got {t}")
        if not isinstance(k, Tensor) and (isinstance(k, float) or k < 0):
            raise ValueError(f"{fn}: top_k must be a whole number of at least 0, got {k}")
        if not isinstance(p, Tensor) and not 0.0 < p <= 1.0:
            raise ValueError(f"{fn}: top_p must be above 0 and at most 1, got {p}")
        if not isinstance(m, Tensor) and not 0.0 <= m <= 1.0:
            raise ValueError(f"{fn}: min_p must be within 0 .. 1, got {m}")

    def tensors(self) -> tuple[Tensor | None, ...]:
        return tuple(x if isinstance(x, Tensor) else None for x in (self.temperature, self.top_k, self.top_p, self.min_p))

    def arguments(self) -> tuple:
        """The settings as ``sqx_sample`` takes them: a pointer and a number each."""
        out = []
        for x, number in ((self.temperature, float), (self.top_k, int), (self.top_p, float), (self.min_p, float)):
            out += [x.data_ptr(), number(0)] if isinstance(x, Tensor) else [None, min(number(x), (1 << 31) - 1)]
        return tuple(out)


@functools.lru_cache(maxsize=256)
def workspace_bytes(b: int, v: int) -> int:
    return int(_lib.load().sqx_sample_workspace_bytes(b, v))


def sample_tokens(logits: Tensor, u: Tensor, *, temperature: float | Tensor = 1.0, top_k: int | Tensor = 0,
                  top_p: float | Tensor = 1.0, min_p: float | Tensor = 0.0, out: Tensor | None = None) -> Tensor:
    """Draw a token from every row of ``logits [B, V]`` (float32, bfloat16 or float16; V up to 2^20): int32 ``[B]``.

    With ``m`` a row's maximum and ``w_i = exp((logits_i - m) / temperature)``, tokens stand in the order of their logits,
    equal ones by their id. Of these the limits keep, one after the other: the first ``top_k`` (0: all); those with less than
    ``top_p`` of the kept tokens' weight before them (1: all; the first always stays); those with ``w_i >= min_p``. The draw is the
    least id whose cumulative kept weight, ids ascending, exceeds ``u[b]`` times the whole (``u`` float32 ``[B]`` in [0, 1)).
    Weights and sums are float64, or whole numbers that hold as much; a token about 32 temperatures or more below the maximum,
    whose weight is below 2^-45, is not drawn. The call's workspace is 12 KB for every 8192 tokens of a row.

    ``temperature`` 0 takes the maximum (the first of equals; a NaN counts as the maximum). At others a row that is no
    distribution (NaN, +inf, or -inf everywhere) gives -1. -inf masks a token.

    Each setting is a number or a tensor ``[B]`` (float32, ``top_k`` int32), whose values are taken as: temperature not above
    0 is 0, others within 1e-4 .. 1e4; top_k below 1 is 0; top_p not above 0 keeps the first token; min_p above 1 is 1; a limit of NaN is none."""
    fn = "sample_tokens"
    if logits.ndim != 2:
        raise ValueError(f"{fn}: logits must be [B, V], got {tuple(logits.shape)}")
    b, v = logits.shape
    if not 1 <= v <= MAX_VOCAB:
        raise ValueError(f"{fn}: a vocabulary of {v}, 1 to {MAX_VOCAB}")
    if b >= 1 << 16:
        raise ValueError(f"{fn}: {b} rows, at most {(1 << 16) - 1}")
    dt = _lib.sqx_dtype(logits.dtype)
    if tuple(u.shape) != (b,) or u.dtype != torch.float32:
        raise ValueError(f"{fn}: u must be float32 [{b}], got {tuple(u.shape)} of {u.dtype}")
    s = Sampling(temperature, top_k, top_p, min_p)
    s.check(b, fn)
    if out is not None and (tuple(out.shape) != (b,) or out.dtype != torch.int32 or not out.is_contiguous()):
        raise ValueError(f"{fn}: out must be contiguous int32 [{b}], got {tuple(out.shape)} of {out.dtype}")
    index = _lib.device_index(fn, logits, u, *s.tensors(), out)
    if not logits.is_contiguous():
        logits = logits.contiguous()
    if not u.is_contiguous():
        u = u.contiguous()
    if out is None:
        out = torch.empty(b, dtype=torch.int32, device=logits.device)
    nb = workspace_bytes(b, v)
    ws = torch.empty(nb, dtype=torch.uint8, device=logits.device)
    _lib.launch(index, fn, _lib.load().sqx_sample, logits.data_ptr(), dt, u.data_ptr(), *s.arguments(), b, v, out.data_ptr(),
                ws.data_ptr(), nb)
    return out
