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


class Exact:
    """One row with sums of whole numbers, for rows whose decisions fall far below the rounding of a float64 sum: weights are
    float64 (those of at most 32 temperatures behind the maximum), scaled by 2^100 and so whole."""

    SCALE = 100

    def __init__(self, logits: np.ndarray, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0) -> None:
        l = logits.astype(np.float64)
        order = np.lexsort((np.arange(len(l)), -l))
        w = [int(x) for x in np.ldexp(np.exp((l[order] - l[order[0]]) / temperature), self.SCALE)]
        stay = len(w) if top_k < 1 else min(top_k, len(w))
        self.margin = math.inf  # of the decisions so far, relative to the weight that they are about
        if top_p < 1.0:
            num, den = float(top_p).as_integer_ratio()
            total, before, cut = sum(w[:stay]), 0, 0
            for i in range(stay):  # kept while den * before < num * total
                if i > 0 and den * before >= num * total:
                    break
                cut = i + 1
                last, before = before, before + w[i]
            for x in (last, before):
                self.margin = min(self.margin, abs(den * x - num * total) / (den * total))
            stay = cut
        if min_p > 0.0:
            floor = int(math.ldexp(min(min_p, 1.0), self.SCALE))
            stay = sum(1 for x in w[:stay] if x >= floor)
        self.ids = sorted(int(i) for i in order[:stay])
        weight = dict(zip(order[:stay].tolist(), w))
        self.upto, run = [], 0
        for i in self.ids:
            run += weight[i]
            self.upto.append(run)

    def draw(self, u: float) -> tuple[int, float]:
        """The token, and how far the nearest decision is from falling otherwise, as a part of the weight."""
        num, den = float(u).as_integer_ratio()
        total = self.upto[-1]
        lo, hi = 0, len(self.upto) - 1
        while lo < hi:  # the least with den * upto > num * total
            mid = (lo + hi) // 2
            lo, hi = (lo, mid) if den * self.upto[mid] > num * total else (mid + 1, hi)
        edges = [self.upto[lo]] + ([self.upto[lo - 1]] if lo else [])
        return self.ids[lo], min([self.margin] + [abs(den * x - num * total) / (den * total) for x in edges])
