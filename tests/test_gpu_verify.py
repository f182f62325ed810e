"""verify_draft (scratch_llm_amd/speculative.py) on the GPU against oracle/kv_block_ref.py: whole numbers, compared exactly.

Picks are made in float64 on both sides: one can differ only where a cumulative sum lies within about 1e-12 of its
threshold, which over a vocabulary of v tokens has a chance of about v 1e-12 a row. A draft is judged by probabilities good
to 2^-18, mostly to 2^-22: a decision can differ where u q is that near to p, about one in a million."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import kv_block_ref as R
from tests.conftest import print_case

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def make(b, t, v, dtype, pdtype, seed):
    g = torch.Generator().manual_seed(seed)
    base = 2.5 * torch.randn(b, t + 1, v, generator=g)
    logits = base.to(DT[dtype])
    q = torch.softmax(base[:, :t] + 0.3 * torch.randn(b, t, v, generator=g), -1)
    draft = torch.multinomial(q.reshape(b * t, v), 1, generator=g).view(b, t).int() if t else torch.zeros(b, 0, dtype=torch.int32)
    likely = logits[:, :t].argmax(-1).int()
    draft = torch.where(torch.rand(b, t, generator=g) < 0.4, likely, draft)
    probs = None if pdtype is None else q.to(DT[pdtype])
    return logits, draft, probs, torch.rand(b, t, generator=g), torch.rand(b, generator=g)


def run(logits, draft, probs, u, r, counts, temp):
    from scratch_llm_amd import speculative

    d = lambda x: None if x is None else x.to(DEV)
    n, tok = speculative.verify_draft(d(logits), d(draft), d(u), d(r), draft_probs=d(probs),
                                      counts=None if counts is None else torch.tensor(counts, dtype=torch.int32, device=DEV),
                                      temperature=temp)
    wn, wt = R.verify(logits.double().numpy(), draft.numpy(), counts or [draft.shape[1]] * draft.shape[0],
                      None if probs is None else probs.double().numpy(), None if u is None else u.numpy(),
                      None if r is None else r.numpy(), temp)
    assert n.cpu().tolist() == wn.tolist()
    assert tok.cpu().tolist() == wt.tolist()
    return wn


@pytest.mark.parametrize("temp", [1.0, 0.7, 0.0])
@pytest.mark.parametrize("dtype,pdtype", [("bf16", "fp32"), ("fp32", None), ("fp16", "bf16"), ("bf16", "fp16"), ("fp32", "fp32")])
@pytest.mark.parametrize("b,t,v", [(1, 1, 2), (3, 4, 50), (2, 7, 8192), (2, 2, 8193), (5, 3, 20001), (2, 0, 1000), (1, 63, 40),
                                   (2, 3, 128256)])
def test_verify(b, t, v, dtype, pdtype, temp):
    print_case("verify", b, t, v, dtype, pdtype, temp)
    logits, draft, probs, u, r = make(b, t, v, dtype, pdtype, b * 1000 + t + v)
    counts = None if b < 3 else [(i * 2) % (t + 1) for i in range(b)]
    run(logits, draft, probs, u, r, counts, temp)


def test_everything_happens():
    """Over many rows: no draft kept, some, all; the pick from the residual and from the last row."""
    logits, draft, probs, u, r = make(200, 3, 300, "fp32", "fp32", 5)
    n = run(logits, draft, probs, u, r, None, 1.0)
    assert set(n.tolist()) == {0, 1, 2, 3}


def test_borders():
    """Random numbers at both ends; a draft equal to the target (nothing left of p - q); ids outside the vocabulary; masked
    tokens of -inf, one with all others masked; rows that are no distribution; counts outside 0 .. T."""
    logits, draft, probs, u, r = make(16, 3, 513, "fp32", "fp32", 6)
    u[0], r[0] = 0.0, 0.0
    u[1], r[1] = 1.0 - 2.0**-24, 1.0 - 2.0**-24
    logits[2, :, 100:] = -math.inf
    logits[3, :, :] = -math.inf
    logits[3, :, 77] = 1.0
    draft[3] = 77
    draft[4, 1], draft[5, 0], draft[6, 2] = 513, -1, 1 << 30
    logits[7, 0, 5] = math.nan
    logits[8, 1, 5] = math.inf
    logits[9, 3, :] = -math.inf
    logits[10, 0] = -math.inf
    probs[11] = 0.0
    probs[12, 0, 3] = math.nan
    probs[13] = 1.0  # above p everywhere: nothing is left, drawn from p
    u[13] = 0.999
    logits[14] *= 200.0  # p of all but one token underflows or nearly
    for counts in (None, [3] * 8 + [-1, 9, 0, 1, 2, 3, 4, 1]):
        run(logits, draft, probs, u, r, counts, 1.0)
        run(logits, draft, None, u, r, counts, 1.0)


@pytest.mark.parametrize("temp", [1.0, 1e-4, 1e4])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_large_logits(dtype, temp):
    """Rows masked with the type's lowest value, all of a row too; logits up to the type's largest, equal ones among them."""
    logits, draft, probs, u, r = make(12, 2, 9000, "fp32", "fp32", 16)
    low = torch.finfo(DT[dtype]).min
    top = torch.finfo(DT[dtype]).max
    logits[0, :, 5000:] = low
    logits[1] = low
    logits[2, :, 1:] = low
    logits[3] = top
    logits[4] = torch.where(torch.rand(3, 9000, generator=torch.Generator().manual_seed(3)) < 0.5, top, low)
    logits[5] = -1e4
    logits[6] = torch.where(torch.rand(3, 9000, generator=torch.Generator().manual_seed(4)) < 0.01, 0.3 * top, 0.1 * top)
    logits[7] = 0.77 * top
    logits[8] = 0.77 * low
    logits[9, :, ::2] = -math.inf
    for p in (probs, None):
        run(logits.to(DT[dtype]), draft, p, u, r, None, temp)


def test_greedy_ties_and_nan():
    """Ties go to the lowest id within and across slices; a NaN is the maximum, the first one counts."""
    logits = torch.zeros(4, 2, 20000)
    logits[0, 0, [50, 9000, 19999]] = 1.0
    logits[1, 0, 15000] = math.nan
    logits[1, 0, 19000] = math.nan
    logits[1, 0, 3] = math.inf
    logits[2] = -math.inf
    draft = torch.tensor([[50], [15000], [0], [1]], dtype=torch.int32)
    n = run(logits, draft, None, None, None, None, 0.0)
    assert n.tolist() == [1, 1, 1, 0]


def test_replayed_in_a_graph():
    from scratch_llm_amd import speculative

    logits, draft, probs, u, r = (x.to(DEV) for x in make(4, 3, 20000, "bf16", "fp32", 8))
    graph = torch.cuda.CUDAGraph()
    speculative.verify_draft(logits, draft, u, r, draft_probs=probs)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = speculative.verify_draft(logits, draft, u, r, draft_probs=probs)
    for i in range(4):
        u.copy_(torch.rand(4, 3, generator=torch.Generator().manual_seed(i)))
        r.copy_(torch.rand(4, generator=torch.Generator().manual_seed(i + 9)))
        want = speculative.verify_draft(logits, draft, u, r, draft_probs=probs)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
