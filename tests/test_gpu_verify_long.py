"""verify_draft where one pass over a wave is not enough: more drafts than a wave judges at a time (16), and vocabularies of more
slices than a wave holds (64 of 8192). Compared as tests/test_gpu_verify.py compares."""

from __future__ import annotations

import pytest
import torch

from tests.conftest import print_case
from tests.test_gpu_verify import make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("temp", [1.0, 0.0])
@pytest.mark.parametrize("t", [16, 17, 32, 47, 63])
def test_stops_at_every_draft(t, temp):
    """Row i keeps i drafts: the others' numbers, or the greedy pick, are set so that draft i is the first rejected."""
    print_case("verify stops", t, temp)
    b = t + 1
    logits, draft, probs, u, r = make(b, t, 100, "fp32", "fp32", t)
    draft = logits[:, :t].argmax(-1).int()
    u[:] = 0.0
    for i in range(t):
        u[i, i] = 1.0 - 2.0**-24
        draft[i, i] = logits[i, i].argmin()  # the least likely: even certain of itself it is rejected
    for q in (None, 0.5 + 0.0 * probs):
        n = run(logits, draft, q, u, r, None, temp)
        assert n.tolist() == list(range(b))
    counts = [(5 * i) % (t + 2) for i in range(b)]
    n = run(logits, draft, None, u, r, counts, temp)
    assert n.tolist() == [min(i, c, t) for i, c in enumerate(counts)]


@pytest.mark.parametrize("temp", [1.0, 0.0])
@pytest.mark.parametrize("dtype,pdtype,v", [("bf16", "bf16", 64 * 8192), ("bf16", None, 64 * 8192 + 8), ("fp16", "fp32", 600001),
                                            ("fp32", None, 1100003)])
def test_vocabularies_of_many_slices(v, dtype, pdtype, temp):
    """The pick anywhere, in the last slice, and where all that has a weight lies behind the 64th."""
    print_case("verify many slices", v, dtype, pdtype, temp)
    b, t = 4, 1
    logits, draft, probs, u, r = make(b, t, v, dtype, pdtype, v % 1000)
    r[1], u[1] = 1.0 - 2.0**-24, 0.0
    logits[2, :, : 64 * 8192 - 3] = -float("inf")
    u[3] = 1.0 - 2.0**-24
    run(logits, draft, probs, u, r, None, temp)
