"""Times that stand in the comments of the kernels of `perf/more_operators.py`, and beside its cases in the documents.

    python3 perf/more_forms.py passes CASE[,CASE]   a case's passes one after the other, for rocprofv3 --kernel-trace --stats
    python3 perf/more_forms.py attend [LETTERS]     attention behind shared prefixes and the cache attention of each row, us a call
    python3 perf/more_forms.py border               groups around the border from which the prompt kernel takes them
    python3 perf/more_forms.py sample               sampling by its settings and its rows, us a call
    python3 perf/more_forms.py steps                steps of the decode model, Llama-3-8B shapes, us a captured step

`--lib FILE` takes another build of the library, for instance one whose borders are moved so that either kernel takes a group.
Calls are captured ten times in a graph and replayed; the median of seven replays counts.
"""

from __future__ import annotations

import argparse
import dataclasses
import statistics
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import torch  # noqa: E402

from perf import more_operators as M  # noqa: E402
from scratch_llm_amd import _lib  # noqa: E402

ATTEND = {  # letter: what differs from 32 heads over 8 of 128, int8, bf16, blocks of 64, one token a row
    "A": dict(b=64, n=64, shared=8192, ctx=450), "B": dict(b=96, n=16, shared=15000, ctx=900, fmt="e4m3", block=32),
    "C": dict(b=8, n=8, shared=2000, ctx=150), "D": dict(b=32, n=32, shared=8192, ctx=300),
    "E": dict(b=128, n=128, shared=8192, ctx=300), "F": dict(b=256, n=256, shared=4096, ctx=300),
    "G": dict(b=16, n=16, shared=32768, ctx=300), "H": dict(b=64, n=32, shared=16384, ctx=300),
    "I": dict(b=64, n=64, shared=8192, ctx=450, fmt="e4m3"), "J": dict(b=48, n=2, shared=4000, ctx=300),
    "K": dict(b=12, n=4, t=5, h=12, hkv=12, d=64, block=16, fmt="e4m3", shared=3333, ctx=400),
}
BORDER = {  # query rows of the group x shared keys, a handful of keys of each row's own
    "512 x 8192": dict(b=128, n=128, shared=8192), "1024 x 4096": dict(b=256, n=256, shared=4096),
    "2048 x 2048": dict(b=512, n=512, shared=2048), "512 x 16384": dict(b=128, n=128, shared=16384),
    "1024 x 8192": dict(b=256, n=256, shared=8192), "2048 x 4096": dict(b=512, n=512, shared=4096),
    "512 x 32768": dict(b=128, n=128, shared=32768), "1024 x 16384": dict(b=256, n=256, shared=16384),
    "2048 x 8192": dict(b=512, n=512, shared=8192),
    "1024 x 8192, E4M3": dict(b=256, n=256, shared=8192, fmt="e4m3"), "1024 x 16384, E4M3": dict(b=256, n=256, shared=16384, fmt="e4m3"),
    "1024 x 8192, heads of 64": dict(b=256, n=256, shared=8192, d=64), "1024 x 16384, heads of 64": dict(b=256, n=256, shared=16384, d=64),
    "512 x 16384, 16 over 4 heads of 256": dict(b=128, n=128, shared=16384, h=16, hkv=4, d=256),
    "512 x 32768, 16 over 4 heads of 256": dict(b=128, n=128, shared=32768, h=16, hkv=4, d=256),
    "1024 x 8192, 16 over 1 head": dict(b=64, n=64, shared=8192, h=16, hkv=1),
    "1024 x 16384, 16 over 1 head": dict(b=64, n=64, shared=16384, h=16, hkv=1),
}


def timed(call, each: int = 1, warm: int = 3) -> float:
    """us of one of the `each` calls that call() makes."""
    for _ in range(warm):
        call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for _ in range(10):
            call()
    g.replay()
    took = []
    for _ in range(7):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        g.replay()
        b.record()
        torch.cuda.synchronize()
        took.append(a.elapsed_time(b) * 1e3 / (10 * each))
    return statistics.median(took)


def passes(names: list[str]) -> None:
    M.own = True
    for case in M.listed():
        if case["name"] in names:
            states = [M.prepare(case, seed) for seed in range(3)]
            for i in range(12):
                M.run(states[i % 3])
            torch.cuda.synchronize()
            del states


def attend(cases: dict[str, dict], plain: bool, layers: int = 3) -> None:
    from scratch_llm_amd.quant import kv_block, kv_shared

    for name, what in cases.items():
        case = {**dict(kind="attend", layers=layers, t=1, h=32, hkv=8, d=128, block=64, fmt="int8", dtype="bf16", ctx=30), **what}
        st = M.prepare(case, 1)
        cache = list(zip(*st["cache"]))
        plan = kv_shared.plan_shared_kv(st["table"], st["starts"], st["leaders"], block=case["block"], tokens=case["t"], heads=case["h"],
                                        kv_heads=case["hkv"], head_dim=case["d"])
        outs = [torch.empty_like(q) for q in st["q"]]

        def shared():
            for q, layer, out in zip(st["q"], cache, outs):
                kv_shared.attend_shared_kv(q, *layer, st["table"], st["starts"], shared=plan, out=out)

        def each():
            for q, layer, out in zip(st["q"], cache, outs):
                kv_block.attend_kv_blocks(q, *layer, st["table"], st["starts"], out=out)

        tail = f", each row for itself {timed(each, layers):.1f}" if plain else ""
        print(f"{name}: shared {timed(shared, layers):.1f}{tail}", flush=True)
        del st, cache, plan, outs


def sample() -> None:
    from scratch_llm_amd.sampling import sample_tokens

    gen = torch.Generator(device="cuda").manual_seed(1)
    x, u = 2.0 * torch.randn(64, 128256, generator=gen, device="cuda"), torch.rand(64, generator=gen, device="cuda")
    around, flat = (x + 40.0).bfloat16(), torch.zeros(64, 128256, dtype=torch.bfloat16, device="cuda")
    x = x.bfloat16()
    forms = [("greedy", x, dict(temperature=0.0)), ("no limit", x, {}), ("top-k 50", x, dict(top_k=50)), ("top-k 3000", x, dict(top_k=3000)),
             ("min-p 0.05", x, dict(min_p=0.05)), ("top-p 0.9", x, dict(top_p=0.9)), ("top-p 0.95", x, dict(top_p=0.95)),
             ("top-k 3000, top-p 0.9", x, dict(top_k=3000, top_p=0.9)), ("around 40, top-p 0.95", around, dict(top_p=0.95)),
             ("T = 20, top-p 0.9", x, dict(temperature=20.0, top_p=0.9)), ("T = 1e4, top-k 50", x, dict(temperature=1e4, top_k=50)),
             ("T = 1e4, top-p 0.9", x, dict(temperature=1e4, top_p=0.9)), ("equal, top-k 50", flat, dict(top_k=50)),
             ("equal, top-p 0.9", flat, dict(top_p=0.9))]
    for name, logits, kw in forms:
        print(f"{name}: {timed(lambda: sample_tokens(logits, u, **kw)):.1f}", flush=True)


def steps() -> None:
    from scratch_llm_amd.decode import LLAMA3_8B, Int4DecodeLM
    from scratch_llm_amd.sampling import Sampling

    model = Int4DecodeLM.random_init(dataclasses.replace(LLAMA3_8B, context_length=8704), "cuda")

    def i32(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    def step(st, n: int) -> str:
        model.step(st)
        graph, took = model.capture(st), []
        for _ in range(25):
            st.set_lengths([n] * st.batch)
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            graph.replay()
            b.record()
            torch.cuda.synchronize()
            took.append(a.elapsed_time(b) * 1e3)
        return f"{statistics.median(took[5:]):.0f}"

    for rows, n in ((8, 2048), (64, 2048), (64, 8192)):
        out = []
        for pool in (False, True):
            st = model.new_state(rows, n + 256, kv_dtype="int8_block", kv_pages=rows * (n // 64 + 4) if pool else None)
            if pool:
                st.reserve(i32([n] * rows))
            st.set_lengths([n] * rows)
            out.append(step(st, n))
            if not pool:
                st.u.fill_(0.4)
                for s in (Sampling(top_p=0.95), Sampling(top_k=50, temperature=0.8)):
                    st.set_sampling(s)
                    out.append(step(st, n))
            del st
        st = model.new_state(rows, n + 256, kv_dtype="int8_block", kv_pages=n // 64 + 4 * rows)
        st.reserve(i32([n] + [0] * (rows - 1)))
        st.set_lengths([n] + [0] * (rows - 1))
        if not int(st.fork(i32([0] * rows))):
            raise RuntimeError("the pool is too small")
        out.append(step(st, n))
        st.share(i32([0] * rows))
        out.append(step(st, n))
        st.u.fill_(0.4)
        st.set_sampling(Sampling(top_p=0.95))
        out.append(step(st, n))
        print(f"{n} keys, {rows} rows: own pages {out[0]}, top-p {out[1]}, top-k {out[2]}, own pages of a pool {out[3]}, forked {out[4]}, "
              f"shared {out[5]}, and top-p {out[6]}", flush=True)
        del st


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("what", choices=["passes", "attend", "border", "sample", "steps"])
    ap.add_argument("which", nargs="?", default="")
    ap.add_argument("--lib", type=Path)
    args = ap.parse_args()
    if args.lib is not None:
        _lib.LIB_PATH = args.lib.resolve()
    if args.what == "passes":
        passes(args.which.split(","))
    elif args.what == "attend":
        attend({k: v for k, v in ATTEND.items() if not args.which or k in args.which}, plain=True)
    elif args.what == "border":
        attend(BORDER, plain=False)
    else:
        {"sample": sample, "steps": steps}[args.what]()


if __name__ == "__main__":
    main()
