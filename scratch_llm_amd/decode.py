"""One decode step of a Llama-shaped model whose linears are INT4-g128, on MI355X.

The reference decodes by calling ``TransformerLM.forward`` (src/scratch_llm/model.py:439-505) with
one token per row against a slot KV cache (kv_cache.py:80-262, dense ``BatchedKVCache`` storage)
and picking the next token greedily (sampling.py:80-83); with the quantized drop-ins every Linear
is ``w4a16_linear`` (int4_group.py:148-164). This module is that step on the library's kernels:

* the INT4 linears on the tiled weights (the streaming decode kernel below 64 rows, the
  dequant-GEMM from 64 rows), with q|k|v fused into one projection and gate|up into another
  (concatenating rows keeps every group scale: groups run along the input dimension);
* everything between them from sqx_decode.hip: residual add + RMSNorm, split-key GQA attention
  with RoPE and the cache write folded in, SiLU-gate, embedding rows, greedy pick, ``advance``.

A step allocates nothing: :class:`DecodeState` holds the cache and every buffer for one batch
size, so :meth:`Int4DecodeLM.capture` can record the whole step in a HIP graph whose replays
decode token after token (the pick of one replay is the input of the next).

On the block-scaled 8-bit cache (``kv_dtype="int8_block"`` or ``"fp8_block"``,
:mod:`scratch_llm_amd.quant.kv_block`) the model also takes several tokens a row: a chunk of a prompt
(:meth:`Int4DecodeLM.extend`) and drafted tokens with their verification (:meth:`Int4DecodeLM.verify`).
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Callable

import torch
from torch import Tensor

from scratch_llm_amd import _lib, speculative
from scratch_llm_amd.quant import int4_group as i4
from scratch_llm_amd.quant import kv_block
from scratch_llm_amd.quant.fp8_weights import FP8_DTYPE

__all__ = ["DecodeConfig", "DecodeState", "Int4DecodeLM", "LLAMA3_8B", "rope_tables"]

# Batches of 2..64 rows run the linears through sqx_int4_skinny's shape choice (the GEMV or a
# decode-regime kernel, K split into the state's workspace); larger batches run the prefill GEMM.
_SKINNY_MAX_M = i4.GEMM_MIN_M - 1
_WRITE_ROWS = (1 << 16) - 1  # rows that one write into the block-scaled cache takes
_BLOCK_KV = {"int8_block": torch.int8, "fp8_block": FP8_DTYPE}


@dataclass(frozen=True)
class DecodeConfig:
    """Architecture of the decoded model (the fields of model.py:57-112 that a decode step reads)."""

    vocab_size: int = 128256
    d_model: int = 4096
    n_layers: int = 32
    n_heads: int = 32
    n_kv_heads: int = 8
    d_ff: int = 14336
    context_length: int = 2048
    rope_theta: float = 10000.0
    norm_eps: float = 1e-5
    group_size: int = 128

    @property
    def head_dim(self) -> int:
        return self.d_model // self.n_heads

    def validate(self) -> None:
        if self.d_model % self.n_heads != 0:
            raise ValueError(f"d_model={self.d_model} not divisible by n_heads={self.n_heads}")
        if self.n_heads % self.n_kv_heads != 0:
            raise ValueError(f"n_heads={self.n_heads} not divisible by n_kv_heads={self.n_kv_heads}")
        if self.head_dim != 128:
            raise ValueError(f"head_dim={self.head_dim}: the decode attention kernel is built for 128")
        if self.n_heads // self.n_kv_heads not in (1, 2, 4, 8):
            raise ValueError(f"{self.n_heads // self.n_kv_heads} query heads per kv head (1, 2, 4 or 8 are built)")
        for name, k in (("d_model", self.d_model), ("d_ff", self.d_ff)):
            if k % self.group_size != 0:
                raise ValueError(f"{name}={k} not divisible by group_size={self.group_size}")


LLAMA3_8B = DecodeConfig()


def rope_tables(head_dim: int, max_seq_len: int, theta: float) -> tuple[Tensor, Tensor]:
    """cos/sin [max_seq_len, head_dim/2] fp32, computed on the host exactly as the reference's
    RotaryPositionalEmbedding buffers are (model.py:196-202, built on the CPU at construction)."""
    inv_freq = 1.0 / (theta ** (torch.arange(0, head_dim, 2).float() / head_dim))
    positions = torch.arange(max_seq_len).float()
    freqs = torch.outer(positions, inv_freq)
    return freqs.cos(), freqs.sin()


@dataclass
class _Layer:
    attn_norm: Tensor
    wqkv: i4.Int4Tiled
    wo: i4.Int4Tiled
    ffn_norm: Tensor
    w13: i4.Int4Tiled
    w2: i4.Int4Tiled


class DecodeState:
    """The slot cache and the step's buffers for one batch size (BatchedKVCache, kv_cache.py:234-262).

    ``k``/``v``: ``[n_layers, B, Hkv, max_ctx, hd]``, bf16, or with ``kv_dtype="fp8"`` E4M3 codes (uint8)
    with fp32 per-(layer, kv head) scales ``k_scale``/``v_scale`` ``[n_layers, Hkv]`` (the per-head FP8
    cache of fp8_kv_per_head.py; set them with :meth:`set_kv_scales` before decoding, static after).
    With ``kv_dtype="int8_block"`` or ``"fp8_block"`` it is the paged block-scaled cache of
    :mod:`~scratch_llm_amd.quant.kv_block`: ``k`` ``[n_layers, pages, Hkv, kv_block, hd]`` and ``v``
    ``[n_layers, pages, Hkv, hd, kv_block]`` int8 or E4M3 codes, ``k_scale``/``v_scale`` ``[n_layers, pages, Hkv]``, and
    ``block_table`` int32 ``[B, ceil(max_ctx / kv_block)]``, at first row after row (a server may point it elsewhere).
    Nothing is calibrated. Rows that are not active store nothing, and tokens past a row's table are not stored.
    ``lengths`` int32 ``[B]`` (valid positions before the next write); ``active`` uint8 ``[B]`` (rows that
    ``advance`` bumps); ``tokens`` int32 ``[B]``: the step's input ids, overwritten by its greedy picks;
    ``logits`` bf16 ``[B, vocab]``.
    """

    def __init__(self, model: "Int4DecodeLM", batch: int, max_ctx: int, kv_dtype: str = "bf16", kv_block_size: int = 64) -> None:
        cfg, dev = model.cfg, model.device
        if batch < 1 or max_ctx < 1:
            raise ValueError("batch and max_ctx must be >= 1")
        if max_ctx > cfg.context_length:
            raise ValueError(f"max_ctx={max_ctx} exceeds context_length={cfg.context_length}")
        if kv_dtype not in ("bf16", "fp8", *_BLOCK_KV):
            raise ValueError(f"kv_dtype must be 'bf16', 'fp8', 'int8_block' or 'fp8_block', got {kv_dtype!r}")
        self.batch, self.max_ctx, self.kv_dtype = batch, max_ctx, kv_dtype
        hkv, hd, d = cfg.n_kv_heads, cfg.head_dim, cfg.d_model
        self.k_scale = self.v_scale = self.block_table = self.counts = None
        self.block_kv = kv_dtype in _BLOCK_KV
        if self.block_kv:
            if kv_block_size not in kv_block.BLOCKS:
                raise ValueError(f"kv_block_size: block must be one of {kv_block.BLOCKS}, got {kv_block_size}")
            width = -(-max_ctx // kv_block_size)
            layer = kv_block.new_kv_blocks(cfg.n_layers * batch * width, hkv, hd, block=kv_block_size, dtype=_BLOCK_KV[kv_dtype],
                                           device=dev)
            self.k, self.v, self.k_scale, self.v_scale = (t.view(cfg.n_layers, batch * width, *t.shape[1:]) for t in layer)
            self.block_table = torch.arange(batch * width, dtype=torch.int32, device=dev).view(batch, width)
            self.counts = torch.ones(batch, dtype=torch.int32, device=dev)  # tokens that a step stores: `active` as int32
            self._kv = [(self.k[i], self.v[i], self.k_scale[i], self.v_scale[i]) for i in range(cfg.n_layers)]
        else:
            shape = (cfg.n_layers, batch, hkv, max_ctx, hd)
            kvt = torch.bfloat16 if kv_dtype == "bf16" else torch.uint8
            self.k = torch.zeros(shape, dtype=kvt, device=dev)
            self.v = torch.zeros(shape, dtype=kvt, device=dev)
        if kv_dtype == "fp8":
            self.k_scale = torch.ones(cfg.n_layers, hkv, dtype=torch.float32, device=dev)
            self.v_scale = torch.ones(cfg.n_layers, hkv, dtype=torch.float32, device=dev)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.active = torch.ones(batch, dtype=torch.uint8, device=dev)
        self.tokens = torch.zeros(batch, dtype=torch.int32, device=dev)
        bf = dict(dtype=torch.bfloat16, device=dev)
        self.x = [torch.empty(batch, d, **bf), torch.empty(batch, d, **bf)]  # residual stream (ping-pong)
        self.h = torch.empty(batch, d, **bf)  # normalised input of the next projection
        self.delta = torch.empty(batch, d, **bf)  # o_proj / w2 output
        # steps without norm launches: sums of squares of the residual stream per 16 columns [batch, d/16],
        # left by the linear that wrote it for the norm in the next linear
        self.nss = -(-d // 16)
        self.ss = torch.empty(batch, self.nss, dtype=torch.float32, device=dev)
        self.qkv = torch.empty(batch, (cfg.n_heads + 2 * hkv) * hd, **bf)
        self.q = torch.empty(batch, cfg.n_heads * hd, **bf)  # rotated q (one-row steps: the qkv epilogue's)
        self.attn = torch.zeros(batch, cfg.n_heads * hd, **bf)
        self.gu = torch.empty(batch, 2 * cfg.d_ff, **bf)
        self.act = torch.empty(batch, cfg.d_ff, **bf)
        self.logits = torch.empty(batch, cfg.vocab_size, **bf)
        lib = _lib.load()
        nb = max(int(lib.sqx_attn_workspace_bytes(batch, cfg.n_heads, hkv, max_ctx)),
                 int(lib.sqx_attn_partials_workspace_bytes(batch, cfg.n_heads, max_ctx)))
        if self.block_kv:
            nb = int(lib.sqx_kvblock_attention_workspace_bytes(batch, 1, cfg.n_heads, hkv, hd, kv_block_size,
                                                               self.block_table.shape[1]))
        self.attn_ws = torch.empty(max(nb // 4, 4), dtype=torch.float32, device=dev)
        nb = int(lib.sqx_argmax_workspace_bytes(batch, cfg.vocab_size))
        self.argmax_ws = torch.empty(max(nb // 4, 4), dtype=torch.float32, device=dev)
        gw = 0
        for tw in model.linears():  # K splits of the decode-regime linears, or the prefill GEMM's
            if 2 <= batch <= _SKINNY_MAX_M:
                gw = max(gw, int(lib.sqx_int4_skinny_workspace_bytes(batch, tw.rows, tw.cols, 0)))
            elif batch > _SKINNY_MAX_M:
                gw = max(gw, int(lib.sqx_gemm_workspace_bytes(batch, tw.rows, tw.cols)))
        self.gemm_ws = torch.empty(max(gw // 4, 4), dtype=torch.float32, device=dev) if gw > 0 else None

    def set_kv_scales(self, layer: int, k_scale: Tensor, v_scale: Tensor) -> None:
        """Install a layer's per-head scales (``(Hkv,)`` or ``(1, Hkv, 1, 1)``, e.g. ``per_head_scale`` of a
        calibration block; fp8_kv_per_head.py:160-173)."""
        if self.kv_dtype != "fp8":
            raise ValueError("per-head scales belong to an fp8 cache")
        for dst, src in ((self.k_scale, k_scale), (self.v_scale, v_scale)):
            if src.numel() != dst.shape[1]:
                raise ValueError(f"scale must have {dst.shape[1]} elements (one per kv head), got {tuple(src.shape)}")
            dst[layer].copy_(src.reshape(-1).to(torch.float32))

    def write_kv(self, layer: int, k: Tensor, v: Tensor, start: int = 0) -> None:
        """Store a block ``[B, Hkv, T, hd]`` of keys and values at positions ``start..start+T`` of every slot
        (a prefill's output, keys rotated): copied for a bf16 cache, quantized with the layer's scales for an fp8 one,
        block by block for a block-scaled one (whose blocks before ``start`` have to be written first)."""
        t = k.shape[2]
        if k.shape != v.shape or k.shape[0] != self.batch or start < 0 or start + t > self.max_ctx:
            raise ValueError(f"block {tuple(k.shape)} does not fit the cache at {start}")
        if self.block_kv:
            starts = torch.full((self.batch,), start, dtype=torch.int32, device=k.device)
            kv_block.write_kv_blocks(k.transpose(1, 2), v.transpose(1, 2), *self.kv_layer(layer), self.block_table, starts)
            return
        if self.kv_dtype == "bf16":
            self.k[layer, :, :, start:start + t].copy_(k)
            self.v[layer, :, :, start:start + t].copy_(v)
            return
        from scratch_llm_amd.quant import fp8_kv_per_head as kv8

        ks = self.k_scale[layer].view(1, -1, 1, 1)
        vs = self.v_scale[layer].view(1, -1, 1, 1)
        self.k[layer, :, :, start:start + t].copy_(kv8.quantize_per_head(k, ks).view(torch.uint8))
        self.v[layer, :, :, start:start + t].copy_(kv8.quantize_per_head(v, vs).view(torch.uint8))

    def kv_layer(self, layer: int) -> tuple[Tensor, Tensor, Tensor, Tensor]:
        """A layer of the block-scaled cache as the functions of :mod:`~scratch_llm_amd.quant.kv_block` take it."""
        if not self.block_kv:
            raise ValueError(f"a {self.kv_dtype} cache has no blocks")
        return self._kv[layer]

    def check_rows(self, fn: str) -> None:
        """Raises where ``block_table`` or ``lengths`` are not what the kernels of the block-scaled cache read by their bare
        addresses: int32, one row a slot, without gaps, on the model's device. The table may have any width."""
        table, n = self.block_table, self.lengths
        if (table.ndim != 2 or table.shape[0] != self.batch or table.shape[1] < 1 or table.dtype != torch.int32
                or not table.is_contiguous()):
            raise ValueError(f"{fn}: block_table must be contiguous int32 [{self.batch}, width], got {tuple(table.shape)} of {table.dtype}")
        if tuple(n.shape) != (self.batch,) or n.dtype != torch.int32 or not n.is_contiguous():
            raise ValueError(f"{fn}: lengths must be contiguous int32 [{self.batch}], got {tuple(n.shape)} of {n.dtype}")
        _lib.require_device(table, n, self.k, fn=fn)

    def set_lengths(self, lengths) -> None:
        """Set every slot's valid length (a host list or tensor), e.g. after filling the cache."""
        t = torch.as_tensor(lengths, dtype=torch.int32)
        if t.shape != (self.batch,) or bool((t < 0).any()) or bool((t > self.max_ctx).any()):
            raise ValueError(f"lengths must be {self.batch} values in [0, {self.max_ctx}]")
        self.lengths.copy_(t)

    def set_tokens(self, tokens, vocab_size: int) -> None:
        t = torch.as_tensor(tokens, dtype=torch.int64)
        if t.shape != (self.batch,):
            raise ValueError(f"expected {self.batch} token ids, got shape {tuple(t.shape)}")
        if t.device.type == "cpu" and (bool((t < 0).any()) or bool((t >= vocab_size).any())):
            raise IndexError(f"token id out of range [0, {vocab_size})")
        self.tokens.copy_(t.to(torch.int32))


class _Rows:
    """The buffers of one pass over ``rows`` token rows (those of a :class:`DecodeState` that do not depend on its cache),
    allocated on the current stream by the pass itself."""

    def __init__(self, model: "Int4DecodeLM", rows: int, head_only: bool = False, each_qkv: bool = False) -> None:
        cfg, lib = model.cfg, _lib.load()
        bf = dict(dtype=torch.bfloat16, device=model.device)
        d, hd = cfg.d_model, cfg.head_dim
        self.batch = rows
        self.h = torch.empty(rows, d, **bf)
        used = [model.lm_head]
        if not head_only:
            used = model.linears()
            self.x = [torch.empty(rows, d, **bf), torch.empty(rows, d, **bf)]
            self.delta = torch.empty(rows, d, **bf)
            # of one layer after the other, or of every layer to keep
            self.qkv = torch.empty(cfg.n_layers if each_qkv else 1, rows, (cfg.n_heads + 2 * cfg.n_kv_heads) * hd, **bf)
            self.q = torch.empty(rows, cfg.n_heads * hd, **bf)
            self.attn = torch.zeros(rows, cfg.n_heads * hd, **bf)  # rows past their count are not written
            self.gu = torch.empty(rows, 2 * cfg.d_ff, **bf)
            self.act = torch.empty(rows, cfg.d_ff, **bf)
        query = lib.sqx_int4_skinny_workspace_bytes if rows <= _SKINNY_MAX_M else lib.sqx_gemm_workspace_bytes
        tail = (0,) if rows <= _SKINNY_MAX_M else ()
        gw = max(int(query(rows, *shape, *tail)) for shape in {(tw.rows, tw.cols) for tw in used}) if rows > 1 else 0
        self.gemm_ws = torch.empty(gw // 4, dtype=torch.float32, device=model.device) if gw > 0 else None


class Int4DecodeLM:
    """A TransformerLM (model.py:439-505) with every Linear, the LM head included, in the reference's
    symmetric INT4-g128 format, decoding on one MI355X."""

    def __init__(self, cfg: DecodeConfig, embed: Tensor, layers: list[_Layer], final_norm: Tensor,
                 lm_head: i4.Int4Tiled) -> None:
        cfg.validate()
        self.cfg = cfg
        self.embed = embed
        self.layers = layers
        self.final_norm = final_norm
        self.lm_head = lm_head
        self.device = embed.device
        # Whether the general step's norm runs inside the next linear's prologue: it does not pay (every
        # workgroup of the wide qkv / gate-up / lm_head projections would recompute the whole row's
        # norm), so it stays a kernel of its own unless asked for. SwiGLU's product needs no prologue:
        # the fused gate|up weight's rows alternate in groups of 8, so the fused step forms silu(g) * u
        # in the gate/up epilogue and the general step runs the SiLU kernel of that layout.
        self.fuse_norm = False
        # One-row steps: the o and down projections end in the residual add and leave the sums of
        # squares per 16 columns and bf16(h * gain) of the next norm; the next projection (qkv, gate/up,
        # the lm_head) multiplies its product by the norm's row factor formed from the sums, so no norm
        # after layer 0's costs a launch.
        self.fuse_norm_sums = True
        # Batched steps: when the o / down projection splits K, its fp32 partials go straight to the
        # next residual add + RMSNorm, which adds them in the linear's own order (no reduce launch).
        self.fuse_split_norm = True
        # Batched steps: when the q|k|v projection splits K, the attention kernel adds its fp32 partials
        # (in the projection's own order) as it loads q and the new key and value (no reduce launch).
        self.fuse_qkv_parts = True
        # One-row steps, when set: attention leaves its key-chunk partials (at most 8 per head) and the
        # o projection merges them while it loads its activations (no combine launch). Off: every
        # o-projection workgroup merges every head, which cost more than the launch it saves.
        self.fuse_attn_merge = False
        cos, sin = rope_tables(cfg.head_dim, cfg.context_length, cfg.rope_theta)
        self.cos = cos.to(self.device)
        self.sin = sin.to(self.device)

    # ------------------------------------------------------------------ construction
    @classmethod
    def from_state_dict(cls, cfg: DecodeConfig, get: Callable[[str], Tensor], device: torch.device | str) -> "Int4DecodeLM":
        """Quantize a float model given by its reference parameter names (``token_emb.weight``,
        ``blocks.{i}.attn.{q,k,v,o}_proj.weight``, ``blocks.{i}.ffn.{w1,w2,w3}.weight``,
        ``blocks.{i}.{attn,ffn}_norm.weight``, ``final_norm.weight``, ``lm_head.weight``; model.py:
        125-133, 148-156, 227-253, 372-392, 439-452). ``get(name)`` returns the tensor; each weight
        is quantized on the device with quantize_groupwise_int4 (bit-exact with int4_group.py:108-129)."""
        cfg.validate()
        dev = torch.device(device)
        g = cfg.group_size

        def qw(*names: str, pairs8: bool = False) -> i4.Int4Tiled:
            qs = [i4.quantize_groupwise_int4(get(n).to(dev, torch.float32), g) for n in names]
            if pairs8:  # gate and up rows alternate in groups of 8: tile t holds gate 8t.. then up 8t..
                (q1, s1), (q3, s3) = qs
                q = torch.stack([q1.view(-1, 8, q1.shape[1]), q3.view(-1, 8, q3.shape[1])], 1).reshape(-1, q1.shape[1])
                s = torch.stack([s1.view(-1, 8, s1.shape[1]), s3.view(-1, 8, s3.shape[1])], 1).reshape(-1, s1.shape[1])
            else:
                q = torch.cat([a for a, _ in qs]) if len(qs) > 1 else qs[0][0]
                s = torch.cat([b for _, b in qs]) if len(qs) > 1 else qs[0][1]
            return i4.tile_int4(q.contiguous(), s.contiguous(), None, g)

        def vec(name: str) -> Tensor:
            return get(name).to(dev, torch.bfloat16).contiguous()

        layers = []
        for i in range(cfg.n_layers):
            p = f"blocks.{i}."
            layers.append(_Layer(
                attn_norm=vec(p + "attn_norm.weight"),
                wqkv=qw(p + "attn.q_proj.weight", p + "attn.k_proj.weight", p + "attn.v_proj.weight"),
                wo=qw(p + "attn.o_proj.weight"),
                ffn_norm=vec(p + "ffn_norm.weight"),
                w13=qw(p + "ffn.w1.weight", p + "ffn.w3.weight", pairs8=True),
                w2=qw(p + "ffn.w2.weight"),
            ))
        embed = get("token_emb.weight").to(dev, torch.bfloat16).contiguous()
        return cls(cfg, embed, layers, vec("final_norm.weight"), qw("lm_head.weight"))

    @classmethod
    def random_init(cls, cfg: DecodeConfig, device: torch.device | str, seed: int = 0, std: float = 0.02) -> "Int4DecodeLM":
        """Synthetic weights of the configured shape: linears ~N(0, std) in fp32, generated and
        quantized one at a time on the device; embedding ~N(0, 1); norm gains 1 (model.py:153)."""
        dev = torch.device(device)
        gen = torch.Generator(device=dev)
        gen.manual_seed(seed)
        hd = cfg.head_dim
        shapes = {
            "attn.q_proj.weight": (cfg.n_heads * hd, cfg.d_model),
            "attn.k_proj.weight": (cfg.n_kv_heads * hd, cfg.d_model),
            "attn.v_proj.weight": (cfg.n_kv_heads * hd, cfg.d_model),
            "attn.o_proj.weight": (cfg.d_model, cfg.n_heads * hd),
            "ffn.w1.weight": (cfg.d_ff, cfg.d_model),
            "ffn.w3.weight": (cfg.d_ff, cfg.d_model),
            "ffn.w2.weight": (cfg.d_model, cfg.d_ff),
        }

        def get(name: str) -> Tensor:
            if name.endswith("norm.weight"):
                return torch.ones(cfg.d_model, device=dev)
            if name == "token_emb.weight":
                return torch.randn(cfg.vocab_size, cfg.d_model, device=dev, generator=gen)
            if name == "lm_head.weight":
                return torch.randn(cfg.vocab_size, cfg.d_model, device=dev, generator=gen) * std
            return torch.randn(shapes[name.split(".", 2)[2]], device=dev, generator=gen) * std

        return cls.from_state_dict(cfg, get, dev)

    # ------------------------------------------------------------------ queries
    def linears(self) -> list[i4.Int4Tiled]:
        out = []
        for ly in self.layers:
            out += [ly.wqkv, ly.wo, ly.w13, ly.w2]
        return out + [self.lm_head]

    def weight_bytes(self) -> int:
        """HBM bytes one step streams for weights (tiled codes, scales, norm gains)."""
        return sum(tw.nbytes for tw in self.linears()) + sum(
            ly.attn_norm.numel() * 2 + ly.ffn_norm.numel() * 2 for ly in self.layers
        ) + self.final_norm.numel() * 2

    def new_state(self, batch: int, max_ctx: int | None = None, kv_dtype: str = "bf16", kv_block_size: int = 64) -> DecodeState:
        return DecodeState(self, batch, self.cfg.context_length if max_ctx is None else max_ctx, kv_dtype, kv_block_size)

    # ------------------------------------------------------------------ the step
    def _linear(self, st: DecodeState, tw: i4.Int4Tiled, x: Tensor, y: Tensor, stream: int) -> None:
        lib = _lib.load()
        m = st.batch
        if 2 <= m <= _SKINNY_MAX_M:  # the library picks the GEMV or a decode-regime kernel by shape
            rc = lib.sqx_int4_skinny(
                tw.wt.data_ptr(), tw.st.data_ptr(), None, _lib.DTYPE_F32, x.data_ptr(), _lib.DTYPE_BF16,
                y.data_ptr(), None, m, tw.rows, tw.cols, tw.group_size, -1, 0, 0, 0, *_lib.ws_args(st.gemm_ws),
                stream,
            )
        elif m > _SKINNY_MAX_M:
            rc = lib.sqx_int4_gemm(
                tw.wt.data_ptr(), tw.st.data_ptr(), None, _lib.DTYPE_F32, x.data_ptr(), _lib.DTYPE_BF16,
                y.data_ptr(), None, m, tw.rows, tw.cols, tw.group_size, *_lib.ws_args(st.gemm_ws), stream,
            )
        else:
            rc = lib.sqx_int4_linear(
                tw.wt.data_ptr(), tw.st.data_ptr(), None, _lib.DTYPE_F32, x.data_ptr(), _lib.DTYPE_BF16,
                y.data_ptr(), None, m, tw.rows, tw.cols, tw.group_size, 0, stream,
            )
        _lib.check(rc, "int4 linear")

    def _delta_linear(self, st: DecodeState, tw: i4.Int4Tiled, x: Tensor, stream: int) -> tuple[int, int]:
        """A linear whose output is the residual delta: ``(pointer, 0)`` to the bf16 delta, or
        ``(workspace, S)`` when its launch splits K into S fp32 partials left for the norm to add."""
        lib, B = _lib.load(), st.batch
        if self.fuse_split_norm and 2 <= B <= _SKINNY_MAX_M:
            S = lib.sqx_int4_skinny_default_splits(B, tw.rows, tw.cols)
            if S >= 2:
                _lib.check(lib.sqx_int4_skinny_partials(
                    tw.wt.data_ptr(), tw.st.data_ptr(), None, _lib.DTYPE_F32, x.data_ptr(), _lib.DTYPE_BF16, B,
                    tw.rows, tw.cols, tw.group_size, *_lib.ws_args(st.gemm_ws), stream), "int4 linear (partials)")
                return st.gemm_ws.data_ptr(), S
        self._linear(st, tw, x, st.delta, stream)
        return st.delta.data_ptr(), 0

    def _norm_linear(self, st: DecodeState, cur: int, delta: int | None, gain: Tensor, tw: i4.Int4Tiled, y: Tensor,
                     stream: int, splits: int = 0, swiglu: bool = False, parts: bool = False) -> int:
        """RMSNorm of the residual stream (after adding ``delta`` when given: a bf16 row, or with
        ``splits`` >= 2 the fp32 partials of a K-split linear) feeding ``tw``; returns the index of the
        buffer that holds the residual stream afterwards. Small batches run it as one kernel when
        ``fuse_norm`` is set (the norm computed in the linear's LDS copy of the activations), otherwise
        as two. ``swiglu``: ``tw`` is the fused gate|up weight and ``y`` [B, d_ff] receives
        bf16(silu(g) * u), formed in the linear's epilogue up to 64 rows. ``parts``: the linear splits K
        and leaves its fp32 partials in ``st.gemm_ws`` for the next kernel to add (``y`` unused)."""
        cfg, lib, B, d = self.cfg, _lib.load(), st.batch, self.cfg.d_model
        nxt = cur if delta is None else 1 - cur
        h_out = None if delta is None else st.x[nxt].data_ptr()
        lin_out = st.gu if swiglu else y
        if self.fuse_norm and splits < 2 and not parts and lib.sqx_int4_prologue_fits(B, d):
            _lib.check(lib.sqx_int4_linear_rmsnorm(
                tw.wt.data_ptr(), tw.st.data_ptr(), st.x[cur].data_ptr(), delta, gain.data_ptr(), cfg.norm_eps, h_out,
                lin_out.data_ptr(), B, tw.rows, tw.cols, tw.group_size, 0, stream), "rmsnorm + int4 linear")
        else:
            if splits >= 2:
                _lib.check(lib.sqx_rmsnorm_partials(st.x[cur].data_ptr(), delta, splits, gain.data_ptr(), cfg.norm_eps,
                                                    B, d, h_out, st.h.data_ptr(), stream), "rmsnorm (partials)")
            else:
                _lib.check(lib.sqx_rmsnorm(st.x[cur].data_ptr(), delta, gain.data_ptr(), cfg.norm_eps, B, d, h_out,
                                           st.h.data_ptr(), stream), "rmsnorm")
            if swiglu and B <= _SKINNY_MAX_M:
                _lib.check(lib.sqx_int4_linear_swiglu(tw.wt.data_ptr(), tw.st.data_ptr(), st.h.data_ptr(), y.data_ptr(),
                                                      B, tw.rows, tw.cols, tw.group_size, stream), "gate|up + silu * up")
                return nxt
            if parts:
                _lib.check(lib.sqx_int4_skinny_partials(
                    tw.wt.data_ptr(), tw.st.data_ptr(), None, _lib.DTYPE_F32, st.h.data_ptr(), _lib.DTYPE_BF16, B,
                    tw.rows, tw.cols, tw.group_size, *_lib.ws_args(st.gemm_ws), stream), "int4 linear (partials)")
                return nxt
            self._linear(st, tw, st.h, lin_out, stream)
        if swiglu:
            _lib.check(lib.sqx_silu_mul_pairs8(st.gu.data_ptr(), B, cfg.d_ff, y.data_ptr(), stream), "silu_mul")
        return nxt

    def _norm_sums_linear(self, st: DecodeState, tw: i4.Int4Tiled, y: Tensor, stream: int) -> None:
        """``tw`` applied to RMSNorm(h) as ``r * (bf16(h * gain) @ W^T)`` per row: ``st.h`` holds
        bf16(h * gain) and ``st.ss`` the sums of squares of h, both left by the residual epilogue of
        the linear that wrote h; the row factor r is formed from the sums in the linear's epilogue."""
        lib = _lib.load()
        _lib.check(lib.sqx_int4_linear_rowscale_sumsq(
            tw.wt.data_ptr(), tw.st.data_ptr(), st.h.data_ptr(), st.ss.data_ptr(), st.nss, self.cfg.norm_eps,
            y.data_ptr(), st.batch, tw.rows, tw.cols, tw.group_size, 0, stream), "rmsnorm (row factor) + int4 linear")

    def _norm_sums_swiglu(self, st: DecodeState, tw: i4.Int4Tiled, y: Tensor, stream: int) -> None:
        """:meth:`_norm_sums_linear` for the fused gate|up weight (gate and up rows alternating in groups
        of 8) with SwiGLU's product in the epilogue: ``y`` [B, d_ff] = bf16(silu(g) * u)."""
        lib = _lib.load()
        _lib.check(lib.sqx_int4_linear_rowscale_swiglu(
            tw.wt.data_ptr(), tw.st.data_ptr(), st.h.data_ptr(), st.ss.data_ptr(), st.nss, self.cfg.norm_eps,
            y.data_ptr(), st.batch, tw.rows, tw.cols, tw.group_size, 0, stream),
            "rmsnorm (row factor) + gate|up + silu * up")

    STEP_KINDS = ("qkv", "attention", "o", "gate_up", "down", "lm_head", "other")

    def step(self, st: DecodeState, tokens=None, only: str | None = None) -> Tensor:
        """Decode one token per row: logits of ``st.tokens`` (or ``tokens``) at each row's position,
        written to ``st.logits``; the greedy picks replace ``st.tokens``; active rows advance. Returns
        ``st.tokens``. Only device work is issued (no host synchronisation).

        ``only`` (one of ``STEP_KINDS``) issues just the launches of that kind, with the arguments the
        full step gives them, for timing each kind's share of the step; the results are then
        meaningless. A norm that runs as a kernel of its own before a linear counts with the linear."""
        cfg, lib = self.cfg, _lib.load()
        if only is not None and only not in self.STEP_KINDS:
            raise ValueError(f"only must be one of {self.STEP_KINDS}, got {only!r}")
        if tokens is not None:
            st.set_tokens(tokens, cfg.vocab_size)
        if st.block_kv:
            st.check_rows("Int4DecodeLM.step")
        _lib.require_device(st.tokens, self.embed, fn="Int4DecodeLM.step")
        B, d, H, Hkv, hd, T = st.batch, cfg.d_model, cfg.n_heads, cfg.n_kv_heads, cfg.head_dim, st.max_ctx
        s = _lib.stream_ptr(self.device)
        ck = _lib.check

        def go(kind: str) -> bool:
            return only is None or only == kind

        # no norm launches: each residual add ends a linear and leaves the sums of squares its norm needs,
        # and the linear after the norm applies the row factor (one row: the one-row GEMV; 2..8 rows:
        # the multi-row GEMV, where it takes every linear of the step)
        qkv_rows = (H + 2 * Hkv) * hd
        if B == 1:
            sums = (self.fuse_norm_sums and d <= 8192 and lib.sqx_int4_prologue_fits(1, d)
                    and lib.sqx_int4_prologue_fits(1, cfg.d_ff))
        else:
            rf = lib.sqx_int4_rows_fits
            sums = (self.fuse_norm_sums and d <= 8192 and d % 64 == 0 and rf(B, qkv_rows, d, 1) and rf(B, d, d, 0)
                    and rf(B, 2 * cfg.d_ff, d, 1) and rf(B, d, cfg.d_ff, 0) and rf(B, cfg.vocab_size, d, 1))
        # with a bf16 cache: RoPE and the cache write run in the q|k|v projection's epilogue (the one-row
        # form takes fewer than 1024 row tiles of 16; wider projections keep the separate RoPE)
        rope_in_qkv = sums and st.kv_dtype == "bf16" and (B > 1 or qkv_rows // 16 < 1024)
        # one row: the attention combine runs in the o projection's activation load (two 128-column
        # k-blocks per wave)
        kb_o = d // 128
        merge = (self.fuse_attn_merge and sums and B == 1 and not st.block_kv and d % 256 == 0 and kb_o // 2 <= 16 and H * hd == d)
        # a K-split q|k|v projection (the general step, B >= 48 at Llama-3-8B shapes) leaves its fp32
        # partials and the attention kernel adds them as the projection's reduce would (no reduce launch)
        qkv_split = 0
        if not sums and self.fuse_qkv_parts and not st.block_kv and 2 <= B <= _SKINNY_MAX_M:
            S = lib.sqx_int4_skinny_default_splits(B, qkv_rows, d)
            qkv_split = S if S >= 2 else 0
        with torch.cuda.device(self.device):
            if st.block_kv and go("attention"):
                st.counts.copy_(st.active)  # the flags may change between replays of a captured step
            if go("other"):
                ck(lib.sqx_embed(self.embed.data_ptr(), cfg.vocab_size, st.tokens.data_ptr(), B, d,
                                 st.x[0].data_ptr(), s), "embed")
            cur, delta, dsplit, have_ss = 0, None, 0, False
            for li, ly in enumerate(self.layers):
                # ---- q|k|v (with the attention norm)
                if rope_in_qkv:
                    if not have_ss and go("qkv"):  # layer 0: the norm of the embedding row on its own
                        ck(lib.sqx_rmsnorm(st.x[cur].data_ptr(), None, ly.attn_norm.data_ptr(), cfg.norm_eps, B, d,
                                           None, st.h.data_ptr(), s), "rmsnorm")
                    if go("qkv"):
                        ck(lib.sqx_int4_linear_rope_kv(
                            ly.wqkv.wt.data_ptr(), ly.wqkv.st.data_ptr(), st.h.data_ptr(),
                            st.ss.data_ptr() if have_ss else None, st.nss, cfg.norm_eps,
                            st.lengths.data_ptr(), self.cos.data_ptr(), self.sin.data_ptr(), cfg.context_length, H,
                            Hkv, T, st.q.data_ptr(), st.k[li].data_ptr(), st.v[li].data_ptr(), B, ly.wqkv.rows,
                            ly.wqkv.cols, ly.wqkv.group_size, 0, s), "qkv + rope + cache write")
                elif have_ss:
                    if go("qkv"):
                        self._norm_sums_linear(st, ly.wqkv, st.qkv, s)
                elif go("qkv"):
                    cur = self._norm_linear(st, cur, delta, ly.attn_norm, ly.wqkv, st.qkv, s, dsplit,
                                            parts=qkv_split > 0)
                else:  # the residual stream advances as the norm's launch would have left it
                    cur = cur if delta is None else 1 - cur
                # ---- attention over the cache
                if not go("attention"):
                    pass
                elif st.block_kv:
                    self._block_attention(st, li, st.qkv, st.q, st.attn, B, 1, st.counts, st.attn_ws, s)
                elif merge:  # the partials only; the o projection merges them
                    fp8 = st.kv_dtype == "fp8"
                    ck(lib.sqx_decode_attention_partials(
                        st.q.data_ptr() if rope_in_qkv else st.qkv.data_ptr(), st.lengths.data_ptr(),
                        None if rope_in_qkv else self.cos.data_ptr(), None if rope_in_qkv else self.sin.data_ptr(),
                        cfg.context_length, st.k[li].data_ptr(), st.v[li].data_ptr(),
                        st.k_scale[li].data_ptr() if fp8 else None, st.v_scale[li].data_ptr() if fp8 else None,
                        B, H, Hkv, hd, T, st.attn_ws.data_ptr(), st.attn_ws.numel() * 4, s), "attention partials")
                elif rope_in_qkv:
                    ck(lib.sqx_decode_attention(st.q.data_ptr(), st.k[li].data_ptr(), st.v[li].data_ptr(),
                                                st.lengths.data_ptr(), B, H, Hkv, hd, T, st.attn.data_ptr(),
                                                st.attn_ws.data_ptr(), st.attn_ws.numel() * 4, s), "attention")
                elif qkv_split:
                    fp8 = st.kv_dtype == "fp8"
                    ck(lib.sqx_decode_attention_rope_parts(
                        st.gemm_ws.data_ptr(), qkv_split, st.lengths.data_ptr(), self.cos.data_ptr(),
                        self.sin.data_ptr(), cfg.context_length, st.k[li].data_ptr(), st.v[li].data_ptr(),
                        st.k_scale[li].data_ptr() if fp8 else None, st.v_scale[li].data_ptr() if fp8 else None,
                        B, H, Hkv, hd, T, st.attn.data_ptr(), st.attn_ws.data_ptr(), st.attn_ws.numel() * 4, s),
                       "attention (q|k|v partials)")
                elif st.kv_dtype == "fp8":
                    ck(lib.sqx_decode_attention_rope_fp8kv(
                        st.qkv.data_ptr(), st.lengths.data_ptr(), self.cos.data_ptr(), self.sin.data_ptr(),
                        cfg.context_length, st.k[li].data_ptr(), st.v[li].data_ptr(), st.k_scale[li].data_ptr(),
                        st.v_scale[li].data_ptr(), B, H, Hkv, hd, T, st.attn.data_ptr(), st.attn_ws.data_ptr(),
                        st.attn_ws.numel() * 4, s), "attention")
                else:
                    ck(lib.sqx_decode_attention_rope(
                        st.qkv.data_ptr(), st.lengths.data_ptr(), self.cos.data_ptr(), self.sin.data_ptr(),
                        cfg.context_length, st.k[li].data_ptr(), st.v[li].data_ptr(), B, H, Hkv, hd, T,
                        st.attn.data_ptr(), st.attn_ws.data_ptr(), st.attn_ws.numel() * 4, s), "attention")
                if sums:
                    # o and down end in the residual add and leave bf16(h * gain) of the next norm with
                    # the sums of squares of h; the linear after each norm applies its row factor
                    gain_next = self.layers[li + 1].attn_norm if li + 1 < len(self.layers) else self.final_norm
                    if go("o") and merge:
                        ck(lib.sqx_int4_linear_attn_residual(
                            ly.wo.wt.data_ptr(), ly.wo.st.data_ptr(), st.attn_ws.data_ptr(), st.lengths.data_ptr(), T,
                            st.x[cur].data_ptr(), st.x[1 - cur].data_ptr(), st.ss.data_ptr(), ly.ffn_norm.data_ptr(),
                            st.h.data_ptr(), 1, ly.wo.rows, ly.wo.cols, ly.wo.group_size, kb_o // 2, s),
                           "attention merge + o + residual")
                    elif go("o"):
                        ck(lib.sqx_int4_linear_residual(
                            ly.wo.wt.data_ptr(), ly.wo.st.data_ptr(), st.attn.data_ptr(), st.x[cur].data_ptr(),
                            st.x[1 - cur].data_ptr(), st.ss.data_ptr(), ly.ffn_norm.data_ptr(), st.h.data_ptr(), B,
                            ly.wo.rows, ly.wo.cols, ly.wo.group_size, 0, s), "o + residual")
                    cur = 1 - cur
                    if go("gate_up"):
                        self._norm_sums_swiglu(st, ly.w13, st.act, s)
                    if go("down"):
                        ck(lib.sqx_int4_linear_residual(
                            ly.w2.wt.data_ptr(), ly.w2.st.data_ptr(), st.act.data_ptr(), st.x[cur].data_ptr(),
                            st.x[1 - cur].data_ptr(), st.ss.data_ptr(), gain_next.data_ptr(), st.h.data_ptr(), B,
                            ly.w2.rows, ly.w2.cols, ly.w2.group_size, 0, s), "down + residual")
                    cur, have_ss = 1 - cur, True
                    continue
                if go("o"):
                    delta, dsplit = self._delta_linear(st, ly.wo, st.attn, s)
                else:
                    delta, dsplit = self._delta_plan(st, ly.wo)
                if go("gate_up"):
                    cur = self._norm_linear(st, cur, delta, ly.ffn_norm, ly.w13, st.act, s, dsplit, swiglu=True)
                else:
                    cur = cur if delta is None else 1 - cur
                if go("down"):
                    delta, dsplit = self._delta_linear(st, ly.w2, st.act, s)
                else:
                    delta, dsplit = self._delta_plan(st, ly.w2)
            if not go("lm_head"):
                pass
            elif have_ss:  # the last down projection left bf16(h * final gain) and the sums of squares
                self._norm_sums_linear(st, self.lm_head, st.logits, s)
            else:
                self._norm_linear(st, cur, delta, self.final_norm, self.lm_head, st.logits, s, dsplit)
            if go("other"):
                ck(lib.sqx_argmax(st.logits.data_ptr(), B, cfg.vocab_size, st.tokens.data_ptr(),
                                  st.argmax_ws.data_ptr(), st.argmax_ws.numel() * 4, s), "argmax")
                ck(lib.sqx_advance(st.lengths.data_ptr(), st.active.data_ptr(), B, s), "advance")
        return st.tokens

    def _block_attention(self, st: DecodeState, li: int, qkv: Tensor, q: Tensor, attn: Tensor, batch: int, t: int,
                         counts: Tensor, ws: Tensor, stream: int) -> None:
        """RoPE, the cache write and attention of ``t`` tokens a row over layer ``li`` of a block-scaled cache: ``qkv``
        [batch * t, (H + 2 Hkv) hd] as the fused projection leaves it, ``q`` the rotated queries, ``attn`` the output (rows
        past their count stay as they are)."""
        cfg, lib = self.cfg, _lib.load()
        H, Hkv, hd = cfg.n_heads, cfg.n_kv_heads, cfg.head_dim
        row = (H + 2 * Hkv) * hd
        at = qkv.data_ptr()
        k, v, ks, vs = st.kv_layer(li)
        fmt = _lib.KV_INT8 if k.dtype == torch.int8 else _lib.KV_E4M3
        pages, _, block, _ = k.shape
        width = st.block_table.shape[1]
        cache = (k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), st.block_table.data_ptr(), st.lengths.data_ptr(),
                 counts.data_ptr(), batch, t, H, Hkv, hd, block, pages, width)
        _lib.check(lib.sqx_kvblock_write(
            at + 2 * H * hd, at + 2 * (H + Hkv) * hd, _lib.DTYPE_BF16, t * row, row, hd, t * row, row, hd, at, t * row, row, hd,
            q.data_ptr(), self.cos.data_ptr(), self.sin.data_ptr(), cfg.context_length, hd, 1, fmt, *cache, stream),
            "rope + cache write")
        _lib.check(lib.sqx_kvblock_attention(
            q.data_ptr(), _lib.DTYPE_BF16, t * H * hd, H * hd, hd, fmt, *cache, 1.0 / math.sqrt(hd), attn.data_ptr(),
            ws.data_ptr(), ws.numel() * 4, stream), "attention")

    # ------------------------------------------------------------------ several tokens a row
    @torch.no_grad()
    def extend(self, st: DecodeState, tokens: Tensor, counts: Tensor | None = None, *, last_only: bool = False,
               advance: bool = True) -> Tensor:
        """Score ``tokens`` [B, T] (int32, on the device) of every row after its ``st.lengths`` tokens, on a block-scaled
        cache: their keys and values are stored, and bf16 logits [B, T, vocab] come back; ``last_only``: [B, vocab] of each
        row's last token. ``counts`` (int32 [B]; default T) is how many of a row's tokens are real; logits past them
        mean nothing (for a count of 0 none do). Rows that are not active store nothing. ``advance`` adds the counts
        of active rows to ``st.lengths``. Chunks follow one another, each of fewer than 2^30 / d_ff tokens over all rows; T = 1 is a
        decode step without the pick. A chunk is attended over a cache that holds all of it, and a block's scale goes by all
        of its tokens: scores depend on the later tokens of their blocks by that much, up to a step of the codes. Only
        device work is issued."""
        if not st.block_kv:
            raise ValueError(f"extend needs a block-scaled cache (kv_dtype 'int8_block' or 'fp8_block'), got {st.kv_dtype!r}")
        if tokens.ndim != 2 or tokens.shape[0] != st.batch or tokens.shape[1] < 1 or tokens.dtype != torch.int32:
            raise ValueError(f"tokens must be int32 [{st.batch}, T], got {tuple(tokens.shape)} of {tokens.dtype}")
        if counts is not None and (tuple(counts.shape) != (st.batch,) or counts.dtype != torch.int32):
            raise ValueError(f"counts must be int32 [{st.batch}], got {tuple(counts.shape)} of {counts.dtype}")
        self._check_pass(*tokens.shape, "Int4DecodeLM.extend")
        st.check_rows("Int4DecodeLM.extend")
        _lib.require_device(tokens, counts, self.embed, st.lengths, fn="Int4DecodeLM.extend")
        stored = self._stored(st, tokens.shape[1], counts)
        logits, _ = self._pass(st, tokens.contiguous(), stored, last_only)
        if advance:
            st.lengths.add_(stored)
        return logits

    def _check_pass(self, b: int, t: int, fn: str) -> None:
        """Refuses a pass that a kernel would refuse behind others that have stored a layer's keys and values already."""
        cfg = self.cfg
        most = ((1 << 31) - 1) // (2 * max(cfg.d_model, cfg.n_heads * cfg.head_dim, cfg.d_ff))
        if b * t > max(most, _SKINNY_MAX_M):
            raise ValueError(f"{fn}: {b} rows of {t} tokens, at most {most} of this model in one pass (2 GiB of activations a linear): "
                             "take smaller chunks")
        if t >= 1 << 24 or -(-t * (cfg.n_heads // cfg.n_kv_heads) // 256) >= 1 << 16:
            raise ValueError(f"{fn}: {t} tokens a row are too many for one pass: take smaller chunks")

    @staticmethod
    def _stored(st: DecodeState, t: int, counts: Tensor | None) -> Tensor:
        """How many of its t tokens each row stores: its count, none where it is not active."""
        n = torch.full((st.batch,), t, dtype=torch.int32, device=st.lengths.device) if counts is None else counts.clamp(0, t)
        return n * (st.active != 0)

    def _pass(self, st: DecodeState, tokens: Tensor, stored: Tensor, last_only: bool = False,
              each_qkv: bool = False) -> tuple[Tensor, Tensor]:
        """The layers over ``tokens`` [B, T], of which the cache keeps ``stored`` a row: the logits, and the fused projections
        q|k|v [layers, B * T, (H + 2 Hkv) hd] of every layer (``each_qkv``), else the last one's."""
        cfg, lib, dev = self.cfg, _lib.load(), st.lengths.device
        B, T = tokens.shape
        rows = _Rows(self, B * T, each_qkv=each_qkv)
        nb = int(lib.sqx_kvblock_attention_workspace_bytes(B, T, cfg.n_heads, cfg.n_kv_heads, cfg.head_dim, st.k.shape[3],
                                                           st.block_table.shape[1]))
        ws = torch.empty(max(nb // 4, 4), dtype=torch.float32, device=dev)
        with torch.cuda.device(dev):
            s = _lib.stream_ptr(dev)
            _lib.check(lib.sqx_embed(self.embed.data_ptr(), cfg.vocab_size, tokens.data_ptr(), B * T, cfg.d_model,
                                     rows.x[0].data_ptr(), s), "embed")
            cur, delta, dsplit = 0, None, 0
            for li, ly in enumerate(self.layers):
                qkv = rows.qkv[li if each_qkv else 0]
                cur = self._norm_linear(rows, cur, delta, ly.attn_norm, ly.wqkv, qkv, s, dsplit)
                self._block_attention(st, li, qkv, rows.q, rows.attn, B, T, stored, ws, s)
                delta, dsplit = self._delta_linear(rows, ly.wo, rows.attn, s)
                cur = self._norm_linear(rows, cur, delta, ly.ffn_norm, ly.w13, rows.act, s, dsplit, swiglu=True)
                delta, dsplit = self._delta_linear(rows, ly.w2, rows.act, s)
            if last_only:
                # the final norm of all rows (it also adds the last delta), then the head of each row's last token
                self._final_norm(rows, cur, delta, dsplit, s)
                at = torch.arange(B, device=dev) * T + (stored.long() - 1).clamp_min(0)
                last = _Rows(self, B, head_only=True)
                last.h.copy_(rows.h[at])
                logits = torch.empty(B, cfg.vocab_size, dtype=torch.bfloat16, device=dev)
                self._linear(last, self.lm_head, last.h, logits, s)
            else:
                logits = torch.empty(B, T, cfg.vocab_size, dtype=torch.bfloat16, device=dev)
                self._norm_linear(rows, cur, delta, self.final_norm, self.lm_head, logits, s, dsplit)
        return logits, rows.qkv

    def _open_blocks(self, st: DecodeState, rows: Tensor, saved: Tensor | None = None) -> Tensor:
        """A copy of the blocks that the rows with ``rows`` not zero are in the middle of, in all layers; with ``saved`` they
        are put back from it."""
        cfg, lib, dev = self.cfg, _lib.load(), st.lengths.device
        hkv, hd, pages, block = cfg.n_kv_heads, cfg.head_dim, st.k.shape[1], st.k.shape[3]
        back = saved is not None
        if saved is None:
            saved = torch.empty(int(lib.sqx_kvblock_open_bytes(cfg.n_layers, st.batch, hkv, hd, block)), dtype=torch.uint8, device=dev)
        with torch.cuda.device(dev):
            _lib.check(lib.sqx_kvblock_open(
                back, st.k.data_ptr(), st.v.data_ptr(), st.k_scale.data_ptr(), st.v_scale.data_ptr(), st.block_table.data_ptr(),
                st.lengths.data_ptr(), rows.data_ptr(), cfg.n_layers, st.batch, hkv, hd, block, pages, st.block_table.shape[1],
                saved.data_ptr(), saved.numel(), _lib.stream_ptr(dev)), "open blocks")
        return saved

    def _write_again(self, st: DecodeState, qkv: Tensor, t: int, counts: Tensor) -> None:
        """Store the keys and values of ``counts`` of each row's t tokens in all layers from what a pass projected. The layers
        are rows of one write: layer l's page p is page l * pages + p of the whole cache."""
        cfg, lib, dev, B = self.cfg, _lib.load(), st.lengths.device, st.batch
        H, hkv, hd = cfg.n_heads, cfg.n_kv_heads, cfg.head_dim
        pages, block, width = st.k.shape[1], st.k.shape[3], st.block_table.shape[1]
        fmt = _lib.KV_INT8 if st.k.dtype == torch.int8 else _lib.KV_E4M3
        row = (H + 2 * hkv) * hd
        on = (st.block_table >= 0) & (st.block_table < pages)
        each = max(1, min(cfg.n_layers, _WRITE_ROWS // B))  # layers of a call
        first = torch.arange(each, dtype=torch.int32, device=dev)[:, None, None] * pages
        table = torch.where(on, st.block_table + first, -1)
        starts, counts = st.lengths.repeat(each), counts.repeat(each)
        with torch.cuda.device(dev):
            s = _lib.stream_ptr(dev)
            for l in range(0, cfg.n_layers, each):
                n = min(each, cfg.n_layers - l)
                at = qkv[l].data_ptr()
                _lib.check(lib.sqx_kvblock_write(
                    at + 2 * H * hd, at + 2 * (H + hkv) * hd, _lib.DTYPE_BF16, t * row, row, hd, t * row, row, hd, None, 0, 0, 0,
                    None, self.cos.data_ptr(), self.sin.data_ptr(), cfg.context_length, hd, 1, fmt, st.k[l].data_ptr(),
                    st.v[l].data_ptr(), st.k_scale[l].data_ptr(), st.v_scale[l].data_ptr(), table.data_ptr(), starts.data_ptr(),
                    counts.data_ptr(), n * B, t, H, hkv, hd, block, n * pages, width, s), "cache write")

    def _final_norm(self, rows: "_Rows", cur: int, delta: int | None, splits: int, stream: int) -> None:
        cfg, lib = self.cfg, _lib.load()
        a = (self.final_norm.data_ptr(), cfg.norm_eps, rows.batch, cfg.d_model, rows.x[1 - cur].data_ptr(), rows.h.data_ptr(), stream)
        if splits >= 2:
            _lib.check(lib.sqx_rmsnorm_partials(rows.x[cur].data_ptr(), delta, splits, *a), "rmsnorm (partials)")
        else:
            _lib.check(lib.sqx_rmsnorm(rows.x[cur].data_ptr(), delta, *a), "rmsnorm")

    @torch.no_grad()
    def verify(self, st: DecodeState, draft: Tensor, u: Tensor | None, r: Tensor | None, *, draft_probs: Tensor | None = None,
               counts: Tensor | None = None, temperature: float = 1.0) -> tuple[Tensor, Tensor]:
        """One step of speculative decoding: score ``st.tokens`` and the drafted tokens ``draft`` [B, T] behind them in one
        pass, keep what :func:`scratch_llm_amd.speculative.verify_draft` accepts, and continue from there. Returns its
        ``(n_accepted, tokens)``; ``st.lengths`` grows by the accepted tokens and one, and ``st.tokens`` becomes the token
        that follows them (rows that are not active keep both, and give what the arguments say without meaning). Where no
        token follows, because the row of logits behind the kept ones is no distribution (-1 in ``tokens``), the row stays
        before it: ``st.tokens`` is its last kept token and ``st.lengths`` grows by one less, so that the next pass scores
        that token anew.
        ``counts`` is how many drafts a row has (default T). Rejected drafts leave no trace before the new length: the blocks
        that they shared with older or kept tokens are put back and the kept tokens stored again without them, as a chunk
        of those alone would be. Only the scores have seen them, as those of :meth:`extend` see a chunk."""
        fn = "Int4DecodeLM.verify"
        if draft.ndim != 2 or draft.shape[0] != st.batch or draft.dtype != torch.int32:
            raise ValueError(f"draft must be int32 [{st.batch}, T], got {tuple(draft.shape)} of {draft.dtype}")
        t = draft.shape[1]
        if not st.block_kv:
            raise ValueError(f"verify needs a block-scaled cache (kv_dtype 'int8_block' or 'fp8_block'), got {st.kv_dtype!r}")
        # all of it before the pass, which writes into the cache
        st.check_rows(fn)
        self._check_pass(st.batch, t + 1, fn)
        temperature, u, r, draft_probs = speculative.check_arguments(fn, st.batch, t, self.cfg.vocab_size, draft, u, r, draft_probs,
                                                                     counts, temperature)
        _lib.require_device(draft, u, r, draft_probs, counts, self.embed, st.lengths, fn=fn)
        ids = torch.cat((st.tokens[:, None], draft), 1)
        stored = self._stored(st, t + 1, None if counts is None else counts.clamp(0, t) + 1)
        saved = self._open_blocks(st, stored)
        logits, qkv = self._pass(st, ids, stored, each_qkv=True)
        n, tokens = speculative.verify_draft(logits, draft, u, r, draft_probs=draft_probs, counts=counts, temperature=temperature)
        live = st.active != 0
        at = n.long()[:, None]
        nxt = tokens.gather(1, at)[:, 0]
        nxt_ok = nxt >= 0
        kept = (n + nxt_ok) * live
        # rows that keep fewer tokens than the pass stored: as it was before, then the kept ones
        less = (kept < stored).to(torch.int32)
        self._open_blocks(st, less, saved)
        self._write_again(st, qkv, t + 1, kept * less)
        st.lengths.add_(kept)
        st.tokens.copy_(torch.where(live, torch.where(nxt_ok, nxt, ids.gather(1, at)[:, 0]), st.tokens))
        return n, tokens

    def _delta_plan(self, st: DecodeState, tw: i4.Int4Tiled) -> tuple[int, int]:
        """What :meth:`_delta_linear` would return for ``tw``, without launching it."""
        lib, B = _lib.load(), st.batch
        if self.fuse_split_norm and 2 <= B <= _SKINNY_MAX_M:
            S = lib.sqx_int4_skinny_default_splits(B, tw.rows, tw.cols)
            if S >= 2:
                return st.gemm_ws.data_ptr(), S
        return st.delta.data_ptr(), 0

    def capture(self, st: DecodeState) -> torch.cuda.CUDAGraph:
        """Record one :meth:`step` on ``st`` in a HIP graph. Each ``replay()`` decodes the next token
        from ``st.tokens`` and the cache as they are at that moment. Capturing runs nothing, so ``st``
        is unchanged."""
        torch.cuda.synchronize(self.device)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.device(self.device), torch.cuda.graph(g):
            self.step(st)
        return g
