"""What sampling refuses, and the oracle's definition at the limits: CPU only, no kernel launches."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import sample_ref as R
from scratch_llm_amd import _lib, sampling


def test_refuses():
    x, u = torch.zeros(3, 10), torch.zeros(3)
    call = sampling.sample_tokens
    for kw, what in ((dict(temperature=-1.0), "temperature"), (dict(temperature=1e-5), "temperature"), (dict(temperature=math.nan), "temperature"),
                     (dict(temperature=2e4), "temperature"), (dict(top_k=-1), "top_k"), (dict(top_k=1.5), "top_k"), (dict(top_p=0.0), "top_p"),
                     (dict(top_p=1.01), "top_p"), (dict(top_p=math.nan), "top_p"), (dict(min_p=-0.1), "min_p"), (dict(min_p=1.1), "min_p"),
                     (dict(temperature=torch.ones(2)), "temperature"), (dict(temperature=torch.ones(3).double()), "temperature"),
                     (dict(top_k=torch.ones(3)), "top_k"), (dict(top_k=torch.ones(3).long()), "top_k"), (dict(top_p=torch.ones(3, 1)), "top_p"),
                     (dict(min_p=torch.ones(6)[::2]), "min_p"), (dict(out=torch.zeros(3)), "out"), (dict(out=torch.zeros(2, dtype=torch.int32)), "out")):
        with pytest.raises(ValueError, match=what):
            call(x, u, **kw)
    for bad in (torch.zeros(2), torch.zeros(3, 1), torch.zeros(3).double()):
        with pytest.raises(ValueError, match="u must"):
            call(x, bad)
    with pytest.raises(ValueError, match="logits"):
        call(x[0], u)
    with pytest.raises(ValueError, match="vocabulary"):
        call(torch.zeros(3, 0), u)
    with pytest.raises(ValueError, match="vocabulary"):
        call(torch.zeros(1, 1).expand(1, (1 << 20) + 1), u[:1])
    with pytest.raises(ValueError, match="rows"):
        call(torch.zeros(1, 1).expand(1 << 16, 1), torch.zeros(1 << 16))
    with pytest.raises(TypeError, match="dtype"):
        call(x.double(), u)
    with pytest.raises(RuntimeError, match="device tensors"):
        call(x, u)


def test_entry_point_refuses():
    lib, p, n = _lib.load(), ctypes.c_void_p(256), None
    good = dict(dtype=0, temp=1.0, k=0, p=1.0, m=0.0, B=2, V=100, ws=1 << 20)

    def call(ptr=p, wsp=p, **change):
        a = {**good, **change}
        return lib.sqx_sample(ptr, a["dtype"], p, n, a["temp"], n, a["k"], n, a["p"], n, a["m"], a["B"], a["V"], p, wsp, a["ws"], n)

    for change, what in ((dict(dtype=3), b"F32, BF16 or F16"), (dict(temp=-1.0), b"temperature"), (dict(temp=math.nan), b"temperature"),
                         (dict(k=-1), b"top_k"), (dict(p=0.0), b"top_p"), (dict(p=math.nan), b"top_p"), (dict(m=1.5), b"min_p"),
                         (dict(B=1 << 16), b"rows"), (dict(V=0), b"V=0"), (dict(V=(1 << 20) + 1), b"V="), (dict(ptr=n), b"null"),
                         (dict(ptr=ctypes.c_void_p(258)), b"misaligned")):
        assert call(**change) == -1 and what in lib.sqx_last_error(), (change, lib.sqx_last_error())
    need = lib.sqx_sample_workspace_bytes(2, 100)
    assert call(ws=need - 1) == -3 and call(wsp=n) == -3 and call(wsp=ctypes.c_void_p(264)) == -3
    assert call(B=0) == 0 and lib.sqx_sample_workspace_bytes(0, 100) == 0


def test_oracle_limits():
    l = np.log(np.array([0.1, 0.4, 0.3, 0.2]))
    near = lambda a, b: np.testing.assert_allclose(a, np.array(b) / 0.4, rtol=1e-12)  # noqa: E731
    near(R.kept(l, 1.0, 0, 1.0, 0.0), [0.1, 0.4, 0.3, 0.2])
    near(R.kept(l, 1.0, 2, 1.0, 0.0), [0, 0.4, 0.3, 0])
    near(R.kept(l, 1.0, 0, 0.69, 0.0), [0, 0.4, 0.3, 0])
    near(R.kept(l, 1.0, 0, 0.71, 0.0), [0, 0.4, 0.3, 0.2])
    near(R.kept(l, 1.0, 2, 0.56, 0.0), [0, 0.4, 0, 0])   # of the two's 0.7
    near(R.kept(l, 1.0, 0, 1.0, 0.6), [0, 0.4, 0.3, 0])
    tie = np.zeros(10)
    assert R.kept(tie, 1.0, 3, 1.0, 0.0).tolist() == [1, 1, 1] + [0] * 7
    assert R.kept(tie, 1.0, 0, 0.5, 0.0).tolist() == [1] * 5 + [0] * 5
    assert R.sample(tie, 0.0) == 0 and R.sample(tie, 0.99) == 9 and R.sample(tie, 0.1) == 1
    assert R.sample(np.array([np.nan, 1.0]), 0.5) == -1 and R.sample(np.array([-np.inf, -np.inf]), 0.5) == -1
    assert R.sample(np.array([1.0, np.nan, 3.0]), 0.5, temperature=0.0) == 1
