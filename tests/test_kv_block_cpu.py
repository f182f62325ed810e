"""What the block-scaled cache, the rotary tables and the draft verification refuse, and the host mathematics of the tables:
CPU only, no kernel launches."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import kv_block_ref as R
from scratch_llm_amd import _lib, rope, speculative
from scratch_llm_amd.quant import kv_block as kv

BF = torch.bfloat16


def cache(pages=4, hkv=2, d=64, block=16, dtype=torch.int8):
    return list(kv.new_kv_blocks(pages, hkv, d, block=block, dtype=dtype, device="cpu"))


def args(b=2, width=3):
    return torch.zeros(b, width, dtype=torch.int32), torch.zeros(b, dtype=torch.int32)


def test_new_cache():
    k, v, ks, vs = cache(3, 2, 128, 32, torch.float8_e4m3fn)
    assert k.shape == (3, 2, 32, 128) and v.shape == (3, 2, 128, 32) and ks.shape == vs.shape == (3, 2)
    assert k.dtype == v.dtype == torch.float8_e4m3fn and ks.dtype == torch.float32 and ks.is_contiguous() and vs.is_contiguous()
    for bad in (dict(head_dim=96), dict(block=48), dict(pages=0), dict(n_kv_heads=0)):
        with pytest.raises(ValueError):
            kv.new_kv_blocks(**{**dict(pages=2, n_kv_heads=1, head_dim=64, block=16, device="cpu"), **bad})
    with pytest.raises(TypeError):
        kv.new_kv_blocks(2, 1, 64, dtype=torch.float16, device="cpu")


def calls(c, t, s, x=None, counts=None):
    x = torch.zeros(2, 1, 2, 64, dtype=BF) if x is None else x
    return (lambda: kv.write_kv_blocks(x, x, *c, t, s, counts), lambda: kv.read_kv_blocks(*c, t, s, 4, counts),
            lambda: kv.attend_kv_blocks(x, *c, t, s, counts))


def test_every_entry_refuses_bad_caches():
    t, s = args()
    c = cache()
    cases = [
        ([c[0], c[1].transpose(2, 3), c[2], c[3]], t, s, None, "v_codes"),
        ([c[0], c[1].view(torch.float8_e4m3fn), c[2], c[3]], t, s, None, "v_codes"),
        ([c[0][0], c[1], c[2], c[3]], t, s, None, "k_codes"),
        ([c[0], c[1], c[2][:3], c[3]], t, s, None, "scales"),
        ([c[0], c[1], c[2].double(), c[3]], t, s, None, "scales"),
        (c, t.long(), s, None, "block_table"),
        (c, t[:1], s, None, "block_table|starts|alike"),
        (c, torch.zeros(2, 0, dtype=torch.int32), s, None, "block_table"),
        (c, t, s.long(), None, "starts"),
        (c, t, torch.zeros(3, dtype=torch.int32), None, "starts"),
        (c, t, s, torch.zeros(2), "counts"),
        (c, t, s, torch.zeros(1, dtype=torch.int32), "counts"),
        (c, torch.zeros(3, 2, dtype=torch.int32).t(), s, None, "contiguous"),
        ([c[0], c[1], torch.zeros(2, 4).t(), c[3]], t, s, None, "contiguous"),
    ]
    for cc, tt, ss, counts, what in cases:
        for call in calls(cc, tt, ss, counts=counts):
            with pytest.raises(ValueError, match=what):
                call()
    for call in calls(c, t, s):
        with pytest.raises(RuntimeError, match="device tensors"):
            call()
    with pytest.raises(TypeError, match="codes must be"):
        kv.read_kv_blocks(c[0].view(torch.uint8), c[1].view(torch.uint8), c[2], c[3], t, s, 1)


def test_write_refuses():
    t, s = args()
    c = cache()
    k = torch.zeros(2, 5, 2, 64, dtype=BF)
    cos, sin = rope.rope_table(64, 8)
    bad = [
        (dict(k=k[0], v=k[0]), "alike"), (dict(v=k.half()), "alike"), (dict(v=k[:, :4]), "alike"),
        (dict(k=k[:, :, :1], v=k[:, :, :1]), "heads"), (dict(q=k), "give rope"),
        (dict(q=k.half(), rope=(cos, sin)), "q must be"), (dict(q=k[:, :4], rope=(cos, sin)), "q must be"),
        (dict(rope=(cos, sin[:4])), "alike"), (dict(rope=rope.rope_table(128, 8)), "columns"),
        (dict(rope=rope.rope_table(40, 8)), "multiple of 16"), (dict(rope=(cos.t(), sin.t())), "contiguous|columns"),
    ]
    for change, what in bad:
        a = {**dict(k=k, v=k), **change}
        with pytest.raises(ValueError, match=what):
            kv.write_kv_blocks(a.pop("k"), a.pop("v"), *c, t, s, **a)
    with pytest.raises(TypeError, match="float32"):
        kv.write_kv_blocks(k, k, *c, t, s, rope=(cos.double(), sin.double()))
    with pytest.raises(TypeError, match="dtype"):
        kv.write_kv_blocks(k.double(), k.double(), *c, t, s)


def test_attend_and_read_refuse():
    t, s = args()
    c = cache()
    q = torch.zeros(2, 1, 4, 64, dtype=BF)
    for change, what in ((dict(q=q[0]), "q must be"), (dict(q=q[:, :, :3]), "heads"), (dict(q=q[..., :32]), "heads"),
                         (dict(scale=0.0), "scale"), (dict(scale=math.inf), "scale"), (dict(scale=-1.0), "scale"),
                         (dict(scale=1e31), "scale")):
        a = {**dict(q=q), **change}
        with pytest.raises(ValueError, match=what):
            kv.attend_kv_blocks(a.pop("q"), *c, t, s, **a)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        kv.attend_kv_blocks(q.float(), *c, t, s)
    with pytest.raises(ValueError, match="tokens"):
        kv.read_kv_blocks(*c, t, s, -1)
    with pytest.raises(TypeError, match="dtype"):
        kv.read_kv_blocks(*c, t, s, 1, dtype=torch.float64)


def test_rope_refuses():
    x = torch.zeros(3, 2, 64)
    cos, sin = rope.rope_table(64, 8)
    pos = torch.zeros(3, dtype=torch.int32)
    for a, what in (((x, pos[:2], cos, sin), "positions"), ((x[0, 0], pos, cos, sin), r"\[..., heads, d\]"),
                    ((x[..., :32], pos, cos, sin), "columns"), ((x, pos, cos[0], sin[0]), "alike")):
        with pytest.raises(ValueError, match=what):
            rope.apply_rope(*a)
    with pytest.raises(TypeError):
        rope.apply_rope(x, pos.float(), cos, sin)
    with pytest.raises(TypeError):
        rope.apply_rope(x.double(), pos, cos, sin)
    with pytest.raises(RuntimeError, match="device tensors"):
        rope.apply_rope(x, pos, cos, sin)


def test_verify_refuses():
    lo, dr, u, r = torch.zeros(2, 4, 10), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, 3), torch.zeros(2)
    ok = dict(logits=lo, draft=dr, u=u, r=r)
    for change, what in ((dict(draft=dr[:, :2]), "draft"), (dict(logits=lo[0]), "logits"), (dict(u=None), "u must be"),
                         (dict(u=u.double()), "u must be"), (dict(r=u), "r must be"), (dict(temperature=-1.0), "temperature"),
                         (dict(temperature=1e-9), "temperature"), (dict(temperature=math.nan), "temperature"),
                         (dict(draft_probs=torch.zeros(2, 4, 10)), "draft_probs"),
                         (dict(counts=torch.zeros(3, dtype=torch.int32)), "counts"),
                         (dict(logits=torch.zeros(1, 65, 4), draft=torch.zeros(1, 64, dtype=torch.int32)), "at most 63")):
        a = {**ok, **change}
        with pytest.raises(ValueError, match=what):
            speculative.verify_draft(a.pop("logits"), a.pop("draft"), a.pop("u"), a.pop("r"), **a)
    for change in (dict(draft=dr.long()), dict(counts=torch.zeros(2)), dict(logits=lo.double())):
        a = {**ok, **change}
        with pytest.raises(TypeError):
            speculative.verify_draft(a.pop("logits"), a.pop("draft"), a.pop("u"), a.pop("r"), **a)
    with pytest.raises(RuntimeError, match="device tensors"):
        speculative.verify_draft(lo, dr, u, r)


def test_c_entries_refuse():
    """Every check of the C entry points, before anything reaches the GPU (a non-null pointer is never followed)."""
    lib, p = _lib.load(), ctypes.c_void_p(256)

    def write(**c):
        a = dict(k=p, v=p, dt=1, ks=(64, 64, 64), vs=(64, 64, 64), q=None, qs=(0, 0, 0), qo=None, cos=None, sin=None, rr=0, rot=0,
                 inter=1, fmt=0, kc=p, B=1, T=1, H=0, Hkv=1, hd=64, block=16, pages=2, width=2)
        a.update(c)
        return lib.sqx_kvblock_write(a["k"], a["v"], a["dt"], *a["ks"], *a["vs"], a["q"], *a["qs"], a["qo"], a["cos"], a["sin"],
                                     a["rr"], a["rot"], a["inter"], a["fmt"], a["kc"], p, p, p, p, p, None, a["B"], a["T"], a["H"],
                                     a["Hkv"], a["hd"], a["block"], a["pages"], a["width"], None)

    for bad in (dict(dt=3), dict(fmt=2), dict(block=48), dict(hd=96), dict(Hkv=0), dict(pages=0), dict(width=0), dict(B=-1),
                dict(T=1 << 24), dict(k=None), dict(kc=ctypes.c_void_p(8)), dict(ks=(64, 4, 64)), dict(ks=(-64, 64, 64)),
                dict(cos=p), dict(cos=p, sin=p, rr=4, rot=8), dict(cos=p, sin=p, rr=0, rot=16), dict(q=p, qo=p),
                dict(q=p, cos=p, sin=p, rr=4, rot=16, H=4), dict(width=1 << 27)):
        assert write(**bad) == -1, bad
        assert b"sqx_kvblock_write" in lib.sqx_last_error()
    assert write(B=0) == 0 and write(T=0) == 0

    def attend(**c):
        a = dict(q=p, dt=1, qs=(64, 64, 64), fmt=0, B=1, T=1, H=4, Hkv=1, hd=64, block=16, pages=2, width=2, scale=0.1, out=p)
        a.update(c)
        return lib.sqx_kvblock_attention(a["q"], a["dt"], *a["qs"], a["fmt"], p, p, p, p, p, p, None, a["B"], a["T"], a["H"],
                                         a["Hkv"], a["hd"], a["block"], a["pages"], a["width"], a["scale"], a["out"], None, 0, None)

    for bad in (dict(dt=0), dict(H=3, Hkv=2), dict(scale=0.0), dict(scale=float("nan")), dict(scale=2e30), dict(q=None), dict(out=ctypes.c_void_p(4)),
                dict(qs=(64, 64, 4)), dict(hd=80), dict(T=(1 << 24) - 1, H=64)):
        assert attend(**bad) == -1, bad
    assert lib.sqx_kvblock_attention_workspace_bytes(1, 1, 32, 8, 128, 64, 4096) > 0
    assert attend(width=4096, block=64) == -3 and b"workspace" in lib.sqx_last_error()
    assert lib.sqx_kvblock_attention_workspace_bytes(4096, 1, 32, 8, 128, 64, 4096) == 0
    assert lib.sqx_kvblock_attention_workspace_bytes(1, 1, 3, 2, 128, 64, 16) == 0

    def verify(**c):
        a = dict(logits=p, dt=1, draft=p, probs=None, pdt=0, u=p, r=p, temp=1.0, B=1, T=2, V=10, ws=p, nb=1 << 20)
        a.update(c)
        return lib.sqx_verify_draft(a["logits"], a["dt"], a["draft"], None, a["probs"], a["pdt"], a["u"], a["r"], a["temp"], a["B"],
                                    a["T"], a["V"], p, p, a["ws"], a["nb"], None)

    for bad in (dict(dt=7), dict(T=64), dict(V=0), dict(temp=-1.0), dict(temp=1e-6), dict(logits=None), dict(draft=None), dict(u=None),
                dict(ws=ctypes.c_void_p(4)), dict(probs=p, pdt=9), dict(B=1 << 16)):
        assert verify(**bad) == -1, bad
    assert verify(nb=8) == -3
    n = [3, 1, 8, 0]
    for bad in (dict(dt=5), dict(rot=3), dict(rot=128), dict(rows=0), dict(x=None), dict(x=ctypes.c_void_p(3)), dict(d=0),
                dict(n=1 << 24), dict(h=0)):
        a = dict(x=p, dt=1, d=64, rot=64, rows=4, n=n[0], h=n[1])
        a.update(bad)
        assert lib.sqx_rope(a["x"], a["dt"], a["n"], a["h"], a["d"], 64, 64, p, p, p, a["rows"], a["rot"], 1, p, 64, 64, None) == -1, bad


def test_rope_tables():
    """Against the angles in extended precision, position by position, and each scaling against its definition."""
    cos, sin = rope.rope_table(8, 200001, 500000.0)
    for p in (0, 1, 77777, 200000):
        for i in range(4):
            a = np.longdouble(p) * np.longdouble(500000.0) ** (np.longdouble(-2 * i) / 8)
            # the angle in float64 is within 2^-52 of itself, then half an ulp of fp32
            assert abs(float(np.cos(a)) - cos[p, i].item()) <= 2.0**-24 + p * 2.0**-51
            assert abs(float(np.sin(a)) - sin[p, i].item()) <= 2.0**-24 + p * 2.0**-51
    base, one = rope.rope_frequencies(64, 10000.0)
    assert one == 1.0 and torch.allclose(base, 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32), rtol=1e-14)
    lin, _ = rope.rope_frequencies(64, scaling=rope.RopeScaling("linear", 8.0))
    assert torch.equal(lin, base / 8)
    part, f = rope.rope_frequencies(64, scaling=rope.RopeScaling("by_parts", 8.0, 8192, 1.0, 4.0))
    assert f == 1.0
    for i in range(32):
        wave = 2 * math.pi / base[i].item()
        if wave < 8192 / 4:
            want = base[i].item()
        elif wave > 8192:
            want = base[i].item() / 8
        else:
            m = (8192 / wave - 1) / 3
            want = (1 - m) * base[i].item() / 8 + m * base[i].item()
        assert math.isclose(part[i].item(), want, rel_tol=1e-12)
    yarn, f = rope.rope_frequencies(64, scaling=rope.RopeScaling("yarn", 16.0, 4096))
    assert math.isclose(f, 0.1 * math.log(16.0) + 1)
    lo = math.floor(64 * math.log(4096 / (32 * 2 * math.pi)) / (2 * math.log(10000.0)))
    hi = math.ceil(64 * math.log(4096 / (2 * math.pi)) / (2 * math.log(10000.0)))
    for i in range(32):
        g = min(max((i - lo) / (hi - lo), 0.0), 1.0)
        assert math.isclose(yarn[i].item(), base[i].item() * (1 - g) + base[i].item() / 16 * g, rel_tol=1e-12)
    c, s = rope.rope_table(64, 5, scaling=rope.RopeScaling("yarn", 16.0, 4096, attention_factor=2.0))
    assert torch.equal(c[0], torch.full((32,), 2.0)) and torch.equal(s[0], torch.zeros(32))


def test_rope_tables_refuse():
    for bad in (dict(rot_dim=7), dict(rot_dim=0), dict(theta=1.0), dict(max_seq_len=0)):
        with pytest.raises(ValueError):
            rope.rope_table(**{**dict(rot_dim=8, max_seq_len=4), **bad})
    for bad in (rope.RopeScaling("other", 2.0), rope.RopeScaling("linear", 0.5), rope.RopeScaling("yarn", 2.0),
                rope.RopeScaling("by_parts", 2.0, 64, 4.0, 1.0), rope.RopeScaling("yarn", 2.0, 64, beta_fast=1.0, beta_slow=2.0),
                rope.RopeScaling("linear", math.nan)):
        with pytest.raises(ValueError):
            rope.rope_frequencies(8, scaling=bad)


def test_oracle_growth_is_bounded():
    """The promise of the growing scale, on the oracle: whatever a block sees, a token is off by less than one step of the
    final scale (int8), and quantizing with the final scale from the start would be off by half of one."""
    g = np.random.default_rng(0)
    for trial in range(30):
        block, d = 32, 8
        kc, vc = np.zeros((1, 1, block, d), np.uint8), np.zeros((1, 1, d, block), np.uint8)
        ks, vs = np.zeros((1, 1), np.float32), np.zeros((1, 1), np.float32)
        x = (g.normal(size=(1, block, 1, d)) * np.exp(np.cumsum(np.abs(g.normal(0, 0.2, (1, block, 1, 1))), 1))).astype(np.float32)
        for t in range(block):
            R.write(x[:, t:t + 1], x[:, t:t + 1], kc, vc, ks, vs, np.zeros((1, 1), np.int32), [t], [1], "int8")
        k, v = R.read(kc, vc, ks, vs, np.zeros((1, 1), np.int32), [0], [block], block, "int8")
        assert np.array_equal(k, v)
        assert (np.abs(k - x) < ks[0, 0] * (1 + 1e-6)).all()
        assert ks[0, 0] <= 2 * np.abs(x).max() / 127 * (1 + 1e-6)


def test_oracle_verify_keeps_the_target_distribution():
    """Speculative sampling's law on the oracle, by integrating over the random numbers: with one draft, the first kept
    token is distributed as the target."""
    g = np.random.default_rng(1)
    v, n = 5, 6000
    logits = np.repeat(g.normal(size=(1, 2, v)), n, 0)
    p = np.exp(logits[0, 0]) / np.exp(logits[0, 0]).sum()
    q = g.dirichlet(np.ones(v))
    draft = g.choice(v, size=(n, 1), p=q).astype(np.int32)
    _, tok = R.verify(logits, draft, [1] * n, np.repeat(q[None, None], n, 0), g.random((n, 1)), g.random(n), 1.0)
    freq = np.bincount(tok[:, 0], minlength=v) / n
    assert np.abs(freq - p).max() < 5 * math.sqrt(0.25 / n)


class _Fake:
    """As much of a tensor as the device check reads."""

    def __init__(self, index):
        self.index = index
        self.device = torch.device("cpu") if index < 0 else torch.device("cuda", index)

    def get_device(self):
        return self.index


def test_device_index_takes_one_device_only():
    a, b, c = _Fake(0), _Fake(1), _Fake(-1)
    assert _lib.device_index("f", a, None, a) == 0 and _lib.device_index("f", b) == 1
    for mixed in ((c, a), (a, c), (a, c, a), (c,)):
        with pytest.raises(RuntimeError, match="device tensors"):
            _lib.device_index("f", *mixed)
    for mixed in ((a, b), (b, a, b)):
        with pytest.raises(RuntimeError, match="different devices"):
            _lib.device_index("f", *mixed)
    for none in ((), (None,)):
        with pytest.raises(RuntimeError, match="no tensor"):
            _lib.device_index("f", *none)
