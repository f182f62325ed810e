"""Draws that fall into a tail of many light tokens, against sums of whole numbers (oracle/sample_ref.py, Exact): weights and their sums
hold what float64 holds, also where more tokens than the sorted list has share the bin that a limit ends in.

A decision may fall otherwise within 2^-44 of the whole weight: weights are good to 2^-47 of themselves and the heavy ones to more, each
is rounded to 2^-49 of itself before 8192 of them are added up exactly, some hundred float64 roundings of sums make 2^-46, and where a
limit is looked for digit by digit, 2^17 tokens of equal weight are each off by up to 2^-62 of the whole, 2^-45. Draws nearer to a border
than that are left out, a few in a hundred at most; a float64 sum of that many equal terms, one after the other, may be off by 2^-36."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import sample_ref as R
from tests.conftest import print_case

pytestmark = pytest.mark.gpu
DEV = "cuda"
V = 1 << 17
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


def one_high(g, at, spread=0.0, dtype="fp32"):
    """A logit of 0 and a tail around `at`, rounded to the type."""
    x = torch.from_numpy(np.float32(at + spread * g.normal(0, 1, V))).clamp_(max=-10.0).clamp_(min=-31.0)
    x[70001] = 0.0
    return x.to(DT[dtype])


def around(g, at, spread, v=V):
    return torch.from_numpy(np.float32(at + spread * g.normal(0, 1, v)))


# name: (logits, settings); tails of 2.6e-5, 0.002, 6.7e-7 and 6e-5 of the weight
ROWS = {
    "equal -22": lambda g: (one_high(g, -22.0), dict(top_p=0.99999)),
    "equal -22, by k too": lambda g: (one_high(g, -22.0), dict(top_p=0.99999, top_k=120000)),
    "equal -22, no limit": lambda g: (one_high(g, -22.0), dict()),
    "equal -22, few": lambda g: (one_high(g, -22.0), dict(top_p=1 - 1e-7, top_k=700)),
    "equal -18": lambda g: (one_high(g, -18.0), dict(top_p=0.999)),
    "equal -18, min_p": lambda g: (one_high(g, -18.0), dict(min_p=1.5e-8)),
    "equal -26": lambda g: (one_high(g, -26.0), dict(top_p=1 - 3e-7)),
    "equal -27, no limit": lambda g: (one_high(g, -27.0), dict()),
    "equal -28, no limit": lambda g: (one_high(g, -28.0), dict()),
    "spread -22": lambda g: (one_high(g, -22.0, 1.0), dict(top_p=1 - 2e-5)),
    "spread -22, by k too": lambda g: (one_high(g, -22.0, 1.0), dict(top_p=1 - 1e-5, top_k=100000)),
    "spread -22, min_p": lambda g: (one_high(g, -22.0, 1.0), dict(min_p=math.exp(-22.7))),
    "spread -22, no limit": lambda g: (one_high(g, -22.0, 1.0), dict()),
    "spread -25, no limit": lambda g: (one_high(g, -25.0, 1.0), dict()),
    "steps -22": lambda g: (one_high(g, -22.0, 2.0, "bf16"), dict(top_p=1 - 2e-5)),
    "wide steps -22": lambda g: (one_high(g, -22.0, 1.0, "bf16"), dict(top_p=1 - 2e-5)),
    "bf16 around 40": lambda g: (around(g, 40.0, 2.0).bfloat16(), dict(top_p=0.95)),
    "bf16 around 40, all limits": lambda g: (around(g, 40.0, 2.0).bfloat16(), dict(top_p=0.9, top_k=60000, min_p=1e-3)),
    "flat": lambda g: (torch.zeros(1 << 20), dict(top_p=0.4)),
    "nearly flat": lambda g: (around(g, 0.0, 2.0), dict(top_p=0.7, temperature=20.0)),
}


@pytest.mark.parametrize("name", ROWS)
def test_tails(name):
    from scratch_llm_amd.sampling import sample_tokens

    print_case("tail", name)
    g = np.random.default_rng(list(ROWS).index(name))
    x, kw = ROWS[name](g)
    exact = R.Exact(x.float().numpy(), **kw)
    # in earnest, over what the tail before the high logit has of the weight, over what it has behind it
    high = 70001 / x.numel()
    tail = 1.0 - 1.0 / math.fsum(np.exp((x.double().numpy()[exact.ids] - float(x.max())) / kw.get("temperature", 1.0)))
    if not name.startswith(("equal", "spread", "steps", "wide")):
        high, tail = 0.5, 1.0
    u = np.concatenate((g.random(8), tail * high * g.random(40), 1.0 - tail * (1.0 - high) * g.random(40), [0.0, 1.0 - 2.0**-24]))
    u = np.minimum(np.float32(u), np.float32(1.0 - 2.0**-24))
    got = sample_tokens(x.to(DEV).expand(len(u), x.numel()), torch.from_numpy(u).to(DEV), **kw).tolist()
    want = [exact.draw(float(v)) for v in u]
    sure = [m > 2.0**-44 for _, m in want]
    assert sum(sure) >= 0.9 * len(u)
    off = [(float(v), a, b) for v, a, (b, _), s in zip(u, got, want, sure) if s and a != b]
    assert not off, f"{len(off)} of {sum(sure)}: {off[:5]}"


@pytest.mark.parametrize("first", [0, 5000])
def test_the_last_draw_in_a_faint_tail(first):
    """The largest random number falls among equal tokens of 2^-41 of the heavy one's weight, in the same 8192 tokens as it or soon behind
    them: what these hold in all decides which."""
    from scratch_llm_amd.sampling import sample_tokens

    u = 1.0 - 2.0**-24
    sure = 0
    for at in np.float32(np.log(2.0**-24 * (1.0 + np.linspace(0.005, 0.055, 12) + first / V) / (V - 1))):
        x = torch.full((V,), float(at))
        x[first] = 0.0
        want, margin = R.Exact(x.numpy()).draw(u)
        got = sample_tokens(x.to(DEV)[None], torch.tensor([u], device=DEV))
        if margin > 2.0**-44:
            sure += 1
            assert first < want and got.tolist() == [want], at
    assert sure >= 6
