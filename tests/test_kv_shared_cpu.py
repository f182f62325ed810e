"""What attention behind shared prefixes refuses: CPU only, no kernel launches."""

from __future__ import annotations

import ctypes
from dataclasses import replace

import pytest
import torch

from scratch_llm_amd import _lib
from scratch_llm_amd.quant import kv_block, kv_shared

I32 = torch.int32


def zeros(*shape):
    return torch.zeros(*shape, dtype=I32)


SIZES = dict(block=16, tokens=1, heads=4, kv_heads=2, head_dim=64)


def test_plan_refuses():
    plan = kv_shared.plan_shared_kv
    good = (zeros(2, 3), zeros(2), zeros(2))
    for args, what in (((zeros(6), *good[1:]), "block_table"), ((zeros(0, 3), zeros(0), zeros(0)), "block_table"),
                       ((zeros(2, 0), *good[1:]), "block_table"), ((zeros(2, 3).long(), *good[1:]), "block_table"),
                       ((zeros(3, 2).t(), *good[1:]), "block_table"), ((good[0], zeros(3), good[2]), "starts"),
                       ((good[0], good[1], zeros(2).long()), "leaders"), ((good[0], good[1], zeros(4)[::2]), "leaders")):
        with pytest.raises(ValueError, match=what):
            plan(*args, **SIZES)
    for change, what in ((dict(block=24), "block"), (dict(head_dim=96), "head_dim"), (dict(tokens=0), "tokens"), (dict(heads=3), "heads"),
                         (dict(kv_heads=0), "heads"), (dict(heads=0), "heads")):
        with pytest.raises(ValueError, match=what):
            plan(*good, **{**SIZES, **change})
    with pytest.raises(ValueError, match="4097 rows"):
        plan(zeros(4097, 1), zeros(4097), zeros(4097), **SIZES)
    with pytest.raises(RuntimeError, match="device tensors"):
        plan(*good, **SIZES)
    other = kv_shared.SharedKV(torch.zeros(64, dtype=torch.uint8), 2, 1, 4, 2, 64, 16, 4)
    with pytest.raises(ValueError, match="other sizes"):
        plan(*good, **SIZES, out=other)


def test_attend_refuses():
    c = list(kv_block.new_kv_blocks(4, 2, 64, block=16, device="cpu"))
    t, s, q = zeros(2, 3), zeros(2), torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16)
    sizes = dict(batch=2, tokens=1, heads=4, kv_heads=2, head_dim=64, block=16, width=3)
    shared = kv_shared.SharedKV(torch.zeros(64, dtype=torch.uint8), *sizes.values())
    call = kv_shared.attend_shared_kv
    for name in sizes:
        with pytest.raises(ValueError, match="the plan is for"):
            call(q, *c, t, s, shared=replace(shared, **{name: sizes[name] + 1}))
    for kw, what in ((dict(scale=0.0), "scale"), (dict(out=q[:1]), "out"), (dict(out=q.half()), "out"), (dict(counts=zeros(3)), "counts")):
        with pytest.raises((ValueError, RuntimeError), match=what + "|device"):
            call(q, *c, t, s, shared=shared, **kw)
    for bad, what in ((q[0], "q must"), (q[:, :, :3], "heads"), (q[..., :32], "heads")):
        with pytest.raises(ValueError, match=what):
            call(bad, *c, t, s, shared=shared)
    with pytest.raises(TypeError, match="bfloat16"):
        call(q.float(), *c, t, s, shared=shared)
    with pytest.raises(RuntimeError, match="device tensors"):
        call(q, *c, t, s, shared=shared)


def test_entry_points_refuse():
    lib, p, n = _lib.load(), ctypes.c_void_p(256), None
    good = dict(B=2, T=1, H=4, Hkv=2, hd=64, block=16, pages=8, width=3)
    nb = lib.sqx_kvshared_plan_bytes(2, 1, 4, 2, 64)
    wb = lib.sqx_kvshared_attention_workspace_bytes(2, 1, 4, 2, 64, 16, 3)
    assert nb > 0 and wb > 0

    def plan(ptr=p, table=p, bytes_=nb, **change):
        a = {**good, **change}
        return lib.sqx_kvshared_plan(table, p, p, a["B"], a["T"], a["H"], a["Hkv"], a["hd"], a["block"], a["width"], ptr, bytes_, n)

    def attend(dtype=1, scale=1.0, plan_ptr=p, plan_bytes=nb, ws=p, ws_bytes=wb, q=p, **change):
        a = {**good, **change}
        return lib.sqx_kvshared_attention(q, dtype, 64, 64, 64, 0, p, p, p, p, p, p, n, a["B"], a["T"], a["H"], a["Hkv"], a["hd"], a["block"],
                                          a["pages"], a["width"], scale, plan_ptr, plan_bytes, p, ws, ws_bytes, n)

    for change, what in ((dict(B=0), b"rows"), (dict(B=4097), b"rows"), (dict(T=0), b"shape"), (dict(H=3), b"shape"), (dict(hd=32), b"head_dim"),
                         (dict(block=8), b"block"), (dict(width=0), b"blocks"), (dict(width=1 << 26), b"blocks")):
        for call in (plan, attend):
            assert call(**change) == -1, change
        assert plan(**change) == -1 and what in lib.sqx_last_error(), (change, lib.sqx_last_error())
    assert plan(table=n) == -1 and plan(ptr=n) == -3 and plan(bytes_=nb - 1) == -3 and plan(ptr=ctypes.c_void_p(264)) == -3
    assert attend(dtype=0) == -1 and attend(scale=0.0) == -1 and attend(pages=0) == -1 and attend(q=ctypes.c_void_p(8)) == -1
    assert attend(plan_ptr=n) == -3 and attend(plan_bytes=nb - 1) == -3 and attend(ws=n) == -3 and attend(ws_bytes=wb - 1) == -3
    # rows that take the plain kernels have no workgroups to list, however many
    assert lib.sqx_kvshared_plan_bytes(2, (1 << 20) - 1, 8192, 1, 128) == lib.sqx_kvshared_plan_bytes(4096, 33, 4, 1, 128) == 16
    assert plan(T=(1 << 20) - 1, H=8192, Hkv=1, bytes_=16) == 0 and plan(T=(1 << 20) - 1, H=8192, Hkv=1, bytes_=15) == -3
    assert lib.sqx_kvshared_plan_bytes(0, 1, 4, 2, 64) == 0 and lib.sqx_kvshared_plan_bytes(2, 1, 5, 2, 64) == 0
