"""apply_rope (scratch_llm_amd/rope.py) on the GPU against a float64 rotation (oracle/kv_block_ref.py).

Two products and a sum in fp32 are within 2^-23 (|a c| + |b s|) of the value (two roundings each, 2^-24 of their part);
the result rounds once to its type: half a step."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import kv_block_ref as R
from tests.conftest import print_case

pytestmark = pytest.mark.gpu
DEV = "cuda"


def check(x, pos, cos, sin, interleaved, got):
    xs = x.double().reshape(-1, *x.shape[-2:]).numpy()
    ps = pos.reshape(-1).numpy()
    c, s = cos.numpy(), sin.numpy()
    want = R.rope(xs, ps, c, s, interleaved)
    mag = R.rope(np.abs(xs), ps, np.abs(c), -np.abs(s), interleaved)  # |a c| + |b s| in the first of each pair
    mag = np.maximum(mag, R.rope(np.abs(xs), ps, np.abs(c), np.abs(s), interleaved))
    eps = torch.finfo(x.dtype).eps / 2
    d = 2.0**-23 * np.abs(mag)
    err = np.abs(got.double().cpu().reshape(want.shape).numpy() - want)
    assert (err <= eps * (np.abs(want) + d) + d + torch.finfo(x.dtype).tiny).all()
    rest = 2 * cos.shape[1]
    assert (got.double().cpu().reshape(want.shape).numpy()[..., rest:] == xs[..., rest:]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("n,heads,d,rot", [(1, 40, 128, 128), (5, 3, 64, 32), (17, 1, 256, 64), (3, 2, 80, 80), (4, 5, 96, 20),
                                           (2, 3, 2048, 2048), (2, 7, 7, 6), (9, 33, 128, 16)])
def test_rope(n, heads, d, rot, interleaved, dtype):
    from scratch_llm_amd import rope

    print_case("rope", n, heads, d, rot, interleaved, dtype)
    g = torch.Generator().manual_seed(n * d)
    x = torch.randn(n, heads, d, generator=g).to(dtype)
    cos, sin = rope.rope_table(rot, 300, scaling=rope.RopeScaling("yarn", 4.0, 64))
    pos = torch.randint(-3, 320, (n,), generator=g, dtype=torch.int32)
    got = rope.apply_rope(x.to(DEV), pos.to(DEV), cos.to(DEV), sin.to(DEV), interleaved=interleaved)
    check(x, pos, cos, sin, interleaved, got)


@pytest.mark.parametrize("interleaved", [True, False])
def test_rope_views_and_in_place(interleaved):
    """Heads of a fused projection [B, T, H + 2 Hkv, d] as views, int64 positions, rotated in place."""
    from scratch_llm_amd import rope

    g = torch.Generator().manual_seed(1)
    fused = torch.randn(2, 9, 12, 64, generator=g).bfloat16()
    cos, sin = (t.to(DEV) for t in rope.rope_table(48, 40))
    pos = torch.randint(0, 40, (2, 9), generator=g)
    dev = fused.to(DEV)
    view = dev[:, :, 2:9]
    got = rope.apply_rope(view, pos.to(DEV), cos, sin, interleaved=interleaved)
    check(fused[:, :, 2:9], pos, cos.cpu(), sin.cpu(), interleaved, got)
    back = rope.apply_rope(view, pos.to(DEV), cos, sin, interleaved=interleaved, out=view)
    assert back is view and torch.equal(dev[:, :, 2:9], got)
    assert torch.equal(dev[:, :, :2].cpu(), fused[:, :, :2]) and torch.equal(dev[:, :, 9:].cpu(), fused[:, :, 9:])
    one = torch.randn(1, 1, 3, generator=g)[:, :, ::2]  # strided columns: a copy
    c2, s2 = (t.to(DEV) for t in rope.rope_table(2, 4))
    check(one, torch.tensor([2]), c2.cpu(), s2.cpu(), True, rope.apply_rope(one.to(DEV), torch.tensor([2], device=DEV), c2, s2))
    assert rope.apply_rope(dev[:0], pos[:0].to(DEV), cos, sin).shape == (0, 9, 12, 64)


def test_rope_matches_the_decode_kernels():
    """The decode step's interleaved rotation (sqx_rope_kv) and this one agree bit for bit on the same table."""
    from scratch_llm_amd import _lib, decode, rope

    b, h, hkv, hd, tmax = 3, 8, 2, 128, 64
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(b, (h + 2 * hkv) * hd, generator=g).bfloat16().to(DEV)
    lengths = torch.tensor([0, 17, 63], dtype=torch.int32, device=DEV)
    cos, sin = (t.to(DEV).contiguous() for t in decode.rope_tables(hd, tmax, 10000.0))
    q = torch.empty(b, h * hd, dtype=torch.bfloat16, device=DEV)
    k, v = (torch.zeros(b, hkv, tmax, hd, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    assert _lib.load().sqx_rope_kv(qkv.data_ptr(), lengths.data_ptr(), cos.data_ptr(), sin.data_ptr(), tmax, b, h, hkv, hd, tmax,
                                   q.data_ptr(), k.data_ptr(), v.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    got = rope.apply_rope(qkv.view(b, h + 2 * hkv, hd)[:, :h + hkv], lengths, cos, sin)
    assert torch.equal(got[:, :h].reshape(b, -1), q)
    assert torch.equal(got[:, h:], k[torch.arange(b), :, lengths.long()])
