"""Sampling with temperature, top-k, top-p and min-p in float64, row by row: the oracle of scratch_llm_amd/sampling.py."""

from __future__ import annotations

import math

import numpy as np


def kept(logits: np.ndarray, temperature: float, top_k: int, top_p: float, min_p: float) -> np.ndarray:
    """The weights of one row, 0 where a limit excludes a token."""
    l = logits.astype(np.float64)
    order = np.lexsort((np.arange(len(l)), -l))  # by logit, equal ones by id; -0 equals 0
    w = np.exp((l[order] - l[order[0]]) / temperature)
    if top_k >= 1:
        w[top_k:] = 0.0
    c = np.cumsum(w)
    if not top_p >= 1.0 and not math.isnan(top_p):
        out = ~(c - w < top_p * c[-1])
        out[0] = False
        w = np.where(out, 0.0, w)
    if min_p > 0.0:
        w = np.where(w >= min(min_p, 1.0), w, 0.0)
    back = np.zeros_like(w)
    back[order] = w
    return back


def sample(logits: np.ndarray, u: float, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0) -> int:
    if not temperature > 0.0:
        return int(np.argmax(logits))
    temperature = min(max(temperature, 1e-4), 1e4)
    if np.isnan(logits).any() or not np.isfinite(logits.max()):
        return -1
    c = np.cumsum(kept(logits, temperature, top_k, top_p, min_p))
    over = np.flatnonzero(c > float(u) * c[-1])
    if len(over):
        return int(over[0])
    return int(np.flatnonzero(np.diff(c, prepend=0.0) > 0)[-1])
