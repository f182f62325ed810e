"""Verification of drafted tokens on MI355X: speculative sampling's accept and resample step, and its last sample.

The reference samples one token from one row of logits (src/scratch_llm/sampling.py:80-86). Here a target
model has scored several drafted tokens of every row in one pass (:meth:`Int4DecodeLM.extend`), and
:func:`verify_draft` says how many of them to keep and which token follows, such that the kept tokens
are distributed as the softmax of those logits says. The logits are the target's own as far as scoring several tokens
at once leaves them so: over the block-scaled cache a chunk's tokens share their blocks' scales, later drafts' among
them (:mod:`scratch_llm_amd.quant.kv_block`), and its linears round in another order than one token's. Random
numbers are inputs, so a run can be repeated.
"""

from __future__ import annotations

import torch
from torch import Tensor

from scratch_llm_amd import _lib

__all__ = ["MAX_DRAFTS", "verify_draft"]

MAX_DRAFTS = 63  # drafted tokens per row of one call


def check_arguments(fn: str, b: int, t: int, v: int, draft: Tensor, u: Tensor | None, r: Tensor | None, draft_probs: Tensor | None,
                    counts: Tensor | None, temperature: float) -> tuple[float, Tensor | None, Tensor | None, Tensor | None]:
    """Everything that :func:`verify_draft` refuses of its arguments beside logits [b, t + 1, v]. Returns ``(temperature, u,
    r, draft_probs)`` as they are used: at temperature 0 the last three are not."""
    if tuple(draft.shape) != (b, t):
        raise ValueError(f"{fn}: draft must be {(b, t)} for logits {(b, t + 1, v)}, got {tuple(draft.shape)}")
    if t > MAX_DRAFTS:
        raise ValueError(f"{fn}: {t} drafted tokens, at most {MAX_DRAFTS}")
    if b * (t + 1) >= 1 << 16:
        raise ValueError(f"{fn}: {b} rows of {t} drafts and the token behind them, together at most {(1 << 16) - 1}")
    if v < 1:
        raise ValueError(f"{fn}: empty vocabulary")
    temperature = float(temperature)
    if not (temperature == 0.0 or 1e-4 <= temperature <= 1e4):
        raise ValueError(f"{fn}: temperature must be 0 or within 1e-4 .. 1e4, got {temperature}")
    if temperature == 0.0:
        u = r = draft_probs = None
    else:
        for name, x, shape in (("u", u, (b, t)), ("r", r, (b,))):
            if x is None or tuple(x.shape) != shape or x.dtype != torch.float32:
                raise ValueError(f"{fn}: {name} must be float32 {shape}")
        if draft_probs is not None:
            if tuple(draft_probs.shape) != (b, t, v):
                raise ValueError(f"{fn}: draft_probs must be {(b, t, v)}, got {tuple(draft_probs.shape)}")
            _lib.sqx_dtype(draft_probs.dtype)
    for name, x in (("draft", draft), ("counts", counts)):
        if x is not None and x.dtype != torch.int32:
            raise TypeError(f"{fn}: {name} must be int32, got {x.dtype}")
    if counts is not None and tuple(counts.shape) != (b,):
        raise ValueError(f"{fn}: counts must be {(b,)}, got {tuple(counts.shape)}")
    return temperature, u, r, draft_probs


def verify_draft(logits: Tensor, draft: Tensor, u: Tensor | None, r: Tensor | None, *, draft_probs: Tensor | None = None,
                 counts: Tensor | None = None, temperature: float = 1.0) -> tuple[Tensor, Tensor]:
    """Check ``draft [B, T]`` (int32 ids) against ``logits [B, T + 1, V]``: row t scores the token after t drafts.

    With ``p_t = softmax(logits[:, t] / temperature)`` and ``q_t = draft_probs[:, t]`` (``[B, T, V]``; None: the
    draft was certain of its token), draft t is accepted while ``u[b, t] * q_t(x_t) < p_t(x_t)``. The token that
    follows is drawn from ``max(p - q, 0)`` of the first rejected row, or from ``p`` of the row behind the
    drafts: the least id whose cumulative weight exceeds ``r[b]`` times the total. What the pick is made from is
    float64; the ``p_t(x_t)`` that a draft is accepted by is within 2^-18 of itself. ``temperature=0`` accepts while the
    draft is its row's argmax (the first of equals; a NaN counts as the maximum) and then takes the argmax (``u``, ``r``
    and ``draft_probs`` may be None). ``counts`` (int32 ``[B]``) says how many drafts a row has (default T).

    ``u [B, T]`` and ``r [B]`` are float32 in [0, 1). Returns ``(n_accepted int32 [B], tokens int32 [B, T + 1])``:
    the accepted drafts, the next token, then -1. An id outside the vocabulary is rejected. At temperatures above 0 a row
    that is no distribution (NaN, +inf, or -inf everywhere) rejects its draft and gives -1; at 0 every row has an argmax."""
    fn = "verify_draft"
    if logits.ndim != 3 or draft.ndim != 2:
        raise ValueError(f"{fn}: logits must be [B, T + 1, V] and draft [B, T], got {tuple(logits.shape)}, {tuple(draft.shape)}")
    b, t1, v = logits.shape
    t = t1 - 1
    temperature, u, r, draft_probs = check_arguments(fn, b, t, v, draft, u, r, draft_probs, counts, temperature)
    dt = _lib.sqx_dtype(logits.dtype)
    pdt = _lib.DTYPE_F32 if draft_probs is None else _lib.sqx_dtype(draft_probs.dtype)
    index = _lib.device_index(fn, logits, draft, u, r, draft_probs, counts)
    logits, draft, u, r, draft_probs, counts = (
        x if x is None or x.is_contiguous() else x.contiguous() for x in (logits, draft, u, r, draft_probs, counts))
    lib = _lib.load()
    dev = logits.device
    n = torch.empty(b, dtype=torch.int32, device=dev)
    tokens = torch.empty(b, t1, dtype=torch.int32, device=dev)
    nb = lib.sqx_verify_draft_workspace_bytes(b, t, v)
    ws = torch.empty(max(nb // 8, 1), dtype=torch.float64, device=dev)
    _lib.launch(index, fn, lib.sqx_verify_draft, logits.data_ptr(), dt, draft.data_ptr(), _lib.ptr(counts),
                _lib.ptr(draft_probs), pdt, _lib.ptr(u), _lib.ptr(r), temperature, b, t, v, n.data_ptr(), tokens.data_ptr(),
                ws.data_ptr(), nb)
    return n, tokens
