"""Llama-3-architecture decoder on connex_b200's own sm_100a kernels.

Weights are random-init N(0, 0.02) from a seed (there is no checkpoint to
load); the architecture is Llama-3-8B's by default (32 layers, hidden 4096,
32 q heads / 8 kv heads of 128, FFN 14336, vocab 128256, RoPE theta 5e5).

Storage layout, chosen for the kernels rather than for checkpoint parity:

* ``wqkv``  [(Hq + 2 Hkv) * 128, H]  -- q, k, v projections stacked (fused QKV GEMM)
* ``w13``   [2 F, H]                 -- gate/up interleaved per 256-row tile so the
                                        GEMM epilogue emits SiLU(gate) * up directly
* ``wo``, ``w2``                     -- consumed with the residual-add epilogue
* paged KV cache [L, 2, blocks, Hkv, 16, 128]: one head of one block is a
  contiguous 4 KB slice, the unit the PD push kernel moves.  With
  ``dtype=torch.float8_e4m3fn`` it holds 8-bit values and one power-of-two
  scale per (block, KV head), with ``dtype=torch.uint8`` 4-bit codes with a scale
  and a minimum per half of a token's head ([.., 16, 72] bytes); attention then
  reads K and V from the cache in prefill steps too, so a prompt split at block
  boundaries attends to the same keys and values as a whole one.
* projections may be :class:`Fp8Weight` (e4m3 with a scale per 128 x 128 block):
  their inputs are then quantised per row and 128 columns, by the norm before
  them or by the SiLU-mul product itself

The forward passes launch only this package's kernels (tcgen05 GEMM,
RMSNorm, RoPE + cache write, attention, argmax); a per-layer hook lets the
PD path launch the KV push of layer l while layers l+1.. still compute.
"""
from __future__ import annotations

import math
from collections import Counter
from dataclasses import dataclass, field
from typing import Callable, List, Optional, Sequence

import torch

from connex_b200 import ops
from connex_b200.utils import nvtx


@dataclass(frozen=True)
class LlamaConfig:
    vocab_size: int = 128256
    hidden: int = 4096
    layers: int = 32
    heads: int = 32
    kv_heads: int = 8
    head_dim: int = 128
    ffn: int = 14336
    rope_theta: float = 500000.0
    eps: float = 1e-5
    max_pos: int = 8192 + 512
    block_size: int = 16
    rope_scaling: Optional[tuple] = None     # (factor, low_freq_factor, high_freq_factor, original_max_pos)

    @classmethod
    def llama3_8b(cls) -> "LlamaConfig":
        return cls()

    @classmethod
    def llama31_8b(cls) -> "LlamaConfig":
        """Llama-3.1-8B: the 8B geometry with 128k positions and Llama 3.1 RoPE scaling."""
        return cls(max_pos=131072, rope_scaling=(8.0, 1.0, 4.0, 8192))

    @classmethod
    def tiny(cls, layers: int = 2) -> "LlamaConfig":
        """A small config with the same head geometry (for tests / smoke)."""
        return cls(vocab_size=1024, hidden=512, layers=layers, heads=8, kv_heads=2, ffn=1024,
                   max_pos=2048)

    @property
    def qkv_dim(self) -> int:
        return (self.heads + 2 * self.kv_heads) * self.head_dim

    @property
    def kv_bytes_per_token(self) -> int:
        return 2 * self.layers * self.kv_heads * self.head_dim * 2

    def num_params(self) -> int:
        per_layer = self.qkv_dim * self.hidden + self.hidden * self.heads * self.head_dim \
            + 3 * self.ffn * self.hidden + 2 * self.hidden
        return self.layers * per_layer + 2 * self.vocab_size * self.hidden + self.hidden


@dataclass
class Fp8Weight:
    """A projection [N, K] in e4m3, ``q``, with fp32 ``scale`` [ceil(N / 128),
    ceil(K / 128)]: an element stands for value * its block's scale."""
    q: torch.Tensor
    scale: torch.Tensor

    @classmethod
    def of(cls, w: torch.Tensor) -> "Fp8Weight":
        """A bf16 weight, quantised on its GPU."""
        return cls(*ops.quantize_weight_fp8(w))

    @property
    def shape(self) -> torch.Size:
        return self.q.shape

    @property
    def device(self) -> torch.device:
        return self.q.device

    def float(self) -> torch.Tensor:
        """fp32 [N, K] of the values."""
        s = self.scale.repeat_interleave(128, 0)[:self.q.shape[0]].repeat_interleave(128, 1)[:, :self.q.shape[1]]
        return self.q.float() * s

    def to(self, device) -> "Fp8Weight":
        return Fp8Weight(self.q.to(device), self.scale.to(device))


PROJECTIONS = ("wqkv", "wo", "w13", "w2")


@dataclass
class LayerWeights:
    attn_norm: torch.Tensor
    wqkv: torch.Tensor              # the projections: bf16 tensors or Fp8Weight
    wo: torch.Tensor
    mlp_norm: torch.Tensor
    w13: torch.Tensor
    w2: torch.Tensor

    def to_fp8(self) -> "LayerWeights":
        """The same layer with its projections in e4m3 (those that are already stay as they are)."""
        return LayerWeights(**{n: Fp8Weight.of(t) if n in PROJECTIONS and not isinstance(t, Fp8Weight) else t
                               for n, t in self.__dict__.items()})


@dataclass
class LlamaWeights:
    cfg: LlamaConfig
    embed: torch.Tensor
    layers: List[LayerWeights]
    final_norm: torch.Tensor
    lm_head: torch.Tensor

    @classmethod
    def random(cls, cfg: LlamaConfig, device, seed: int = 0, std: float = 0.02) -> "LlamaWeights":
        g = torch.Generator(device=device)
        g.manual_seed(seed)

        def rnd(*shape):
            t = torch.empty(*shape, dtype=torch.bfloat16, device=device)
            t.normal_(0.0, std, generator=g)
            return t

        def ones(n):
            return torch.ones(n, dtype=torch.bfloat16, device=device)

        layers = []
        for _ in range(cfg.layers):
            gate, up = rnd(cfg.ffn, cfg.hidden), rnd(cfg.ffn, cfg.hidden)
            layers.append(LayerWeights(
                attn_norm=ones(cfg.hidden),
                wqkv=rnd(cfg.qkv_dim, cfg.hidden),
                wo=rnd(cfg.hidden, cfg.heads * cfg.head_dim),
                mlp_norm=ones(cfg.hidden),
                w13=ops.interleave_gate_up(gate, up),
                w2=rnd(cfg.hidden, cfg.ffn),
            ))
            del gate, up
        return cls(cfg=cfg, embed=rnd(cfg.vocab_size, cfg.hidden), layers=layers,
                   final_norm=ones(cfg.hidden), lm_head=rnd(cfg.vocab_size, cfg.hidden))

    def to_fp8(self) -> "LlamaWeights":
        """Quantises the layers' projections, one layer at a time in place:
        embedding, norms and head stay bf16."""
        for i, lw in enumerate(self.layers):
            self.layers[i] = lw.to_fp8()
        return self

    @staticmethod
    def layout(cfg: LlamaConfig):
        """``(name, shape)`` of every engine tensor, in :meth:`named_tensors` order."""
        yield "model.embed_tokens.weight", (cfg.vocab_size, cfg.hidden)
        for i in range(cfg.layers):
            p = f"model.layers.{i}."
            yield p + "input_layernorm.weight", (cfg.hidden,)
            yield p + "self_attn.qkv_proj.weight", (cfg.qkv_dim, cfg.hidden)
            yield p + "self_attn.o_proj.weight", (cfg.hidden, cfg.heads * cfg.head_dim)
            yield p + "post_attention_layernorm.weight", (cfg.hidden,)
            yield p + "mlp.gate_up_proj.weight", (2 * cfg.ffn, cfg.hidden)
            yield p + "mlp.down_proj.weight", (cfg.hidden, cfg.ffn)
        yield "model.norm.weight", (cfg.hidden,)
        yield "lm_head.weight", (cfg.vocab_size, cfg.hidden)

    @classmethod
    def from_arena(cls, cfg: LlamaConfig, arena: torch.Tensor, manifest) -> "LlamaWeights":
        """Weights as views into one uint8 arena laid out by ``manifest``
        (a ``connex.rl.weights.WeightManifest`` of :meth:`layout`)."""
        t = {e.name: arena[e.offset:e.offset + e.nbytes].view(torch.bfloat16).view(e.shape)
             for e in manifest.entries}
        layers = []
        for i in range(cfg.layers):
            p = f"model.layers.{i}."
            layers.append(LayerWeights(attn_norm=t[p + "input_layernorm.weight"],
                                       wqkv=t[p + "self_attn.qkv_proj.weight"], wo=t[p + "self_attn.o_proj.weight"],
                                       mlp_norm=t[p + "post_attention_layernorm.weight"],
                                       w13=t[p + "mlp.gate_up_proj.weight"], w2=t[p + "mlp.down_proj.weight"]))
        return cls(cfg=cfg, embed=t["model.embed_tokens.weight"], layers=layers, final_norm=t["model.norm.weight"],
                   lm_head=t["lm_head.weight"])

    def named_tensors(self):
        """(name, tensor) in HF-style naming with fused qkv / gate_up tensors; the
        scales of an :class:`Fp8Weight` follow it as ``<name>_scale_inv``."""
        def both(name, w):
            if isinstance(w, Fp8Weight):
                yield name, w.q
                yield name + "_scale_inv", w.scale
            else:
                yield name, w
        yield "model.embed_tokens.weight", self.embed
        for i, lw in enumerate(self.layers):
            p = f"model.layers.{i}."
            yield p + "input_layernorm.weight", lw.attn_norm
            yield from both(p + "self_attn.qkv_proj.weight", lw.wqkv)
            yield from both(p + "self_attn.o_proj.weight", lw.wo)
            yield p + "post_attention_layernorm.weight", lw.mlp_norm
            yield from both(p + "mlp.gate_up_proj.weight", lw.w13)
            yield from both(p + "mlp.down_proj.weight", lw.w2)
        yield "model.norm.weight", self.final_norm
        yield "lm_head.weight", self.lm_head


def trainer_layout(cfg: LlamaConfig):
    """``(name, shape)`` of the unfused HF checkpoint tensors a trainer holds."""
    yield "model.embed_tokens.weight", (cfg.vocab_size, cfg.hidden)
    for i in range(cfg.layers):
        p = f"model.layers.{i}."
        yield p + "input_layernorm.weight", (cfg.hidden,)
        yield p + "self_attn.q_proj.weight", (cfg.heads * cfg.head_dim, cfg.hidden)
        yield p + "self_attn.k_proj.weight", (cfg.kv_heads * cfg.head_dim, cfg.hidden)
        yield p + "self_attn.v_proj.weight", (cfg.kv_heads * cfg.head_dim, cfg.hidden)
        yield p + "self_attn.o_proj.weight", (cfg.hidden, cfg.heads * cfg.head_dim)
        yield p + "post_attention_layernorm.weight", (cfg.hidden,)
        yield p + "mlp.gate_proj.weight", (cfg.ffn, cfg.hidden)
        yield p + "mlp.up_proj.weight", (cfg.ffn, cfg.hidden)
        yield p + "mlp.down_proj.weight", (cfg.hidden, cfg.ffn)
    yield "model.norm.weight", (cfg.hidden,)
    yield "lm_head.weight", (cfg.vocab_size, cfg.hidden)


def random_trainer_weights(cfg: LlamaConfig, device, dtype=torch.float32, seed: int = 0, std: float = 0.02):
    """Random unfused HF-named weights (e.g. a trainer's fp32 master copy)."""
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    out = {}
    for name, shape in trainer_layout(cfg):
        t = torch.empty(shape, dtype=dtype, device=device)
        if "norm" in name:
            t.uniform_(0.5, 1.5, generator=g)
        else:
            t.normal_(0.0, std, generator=g)
        out[name] = t
    return out


class PagedKVCache:
    """Paged KV cache [L, 2, blocks, Hkv, BS, D] with a free-block allocator.

    ``dtype=torch.float8_e4m3fn``: an 8-bit cache; ``scales`` [L, 2, blocks,
    Hkv] fp32 then belong to it (see :func:`connex_b200.ops.rope_cache_fp8`),
    otherwise ``scales`` is None.  ``dtype=torch.uint8``: a 4-bit cache [L, 2,
    blocks, Hkv, BS, 72], whose rows hold their scales and minima themselves
    (see :func:`connex_b200.ops.rope_cache_int4`).

    Blocks can be shared: :meth:`fork` gives sequences that continue another
    one tables on its full blocks, and :meth:`free` returns a block to the
    pool with its last owner.  Shared blocks are only read: a sequence appends
    behind its last full block, and :meth:`own` comes before a write to any
    earlier one."""

    def __init__(self, cfg: LlamaConfig, num_blocks: int, device, dtype=torch.bfloat16,
                 storage: Optional[torch.Tensor] = None):
        self.cfg = cfg
        self.num_blocks = num_blocks
        four = (storage.dtype if storage is not None else dtype) == torch.uint8
        shape = (cfg.layers, 2, num_blocks, cfg.kv_heads, cfg.block_size, ops.KV_INT4_ROW if four else cfg.head_dim)
        self.kv = storage.view(shape) if storage is not None else torch.empty(shape, dtype=dtype, device=device)
        self.scales = None
        if self.kv.dtype == torch.float8_e4m3fn:
            self.scales = torch.ones(shape[:4], dtype=torch.float32, device=self.kv.device)
        self._free = list(range(num_blocks - 1, -1, -1))
        self._shared = {}              # block -> owners beyond the first

    @property
    def kind(self) -> str:
        """``bf16``, ``fp8`` or ``int4``."""
        return {torch.float8_e4m3fn: "fp8", torch.uint8: "int4"}.get(self.kv.dtype, "bf16")

    def k(self, layer: int) -> torch.Tensor:
        return self.kv[layer, 0]

    def v(self, layer: int) -> torch.Tensor:
        return self.kv[layer, 1]

    def k_scale(self, layer: int) -> torch.Tensor:
        return self.scales[layer, 0]

    def v_scale(self, layer: int) -> torch.Tensor:
        return self.scales[layer, 1]

    def values(self, layer: int, blocks: Sequence[int]):
        """What K and V of ``blocks`` stand for, bf16 [n, Hkv, BS, D] each (of
        any kind of cache; 4-bit values are rounded to bf16)."""
        at = torch.tensor(list(blocks), dtype=torch.long, device=self.kv.device)
        out = []
        for i in range(2):
            if self.kind == "fp8":
                x = self.kv[layer, i].view(torch.uint8)[at].view(self.kv.dtype)
                out.append((x.float() * self.scales[layer, i][at][..., None, None]).to(torch.bfloat16))
            elif self.kind == "int4":
                out.append(ops.kv_values_int4(self.kv[layer, i][at]))
            else:
                out.append(self.kv[layer, i][at])
        return tuple(out)

    @property
    def head_slice_bytes(self) -> int:
        return self.kv.shape[-2] * self.kv.shape[-1] * self.kv.element_size()

    @property
    def layer_stride_bytes(self) -> int:
        return self.kv.stride(0) * self.kv.element_size()

    @property
    def kv_stride_bytes(self) -> int:
        return self.kv.stride(1) * self.kv.element_size()

    def blocks_needed(self, n_tokens: int) -> int:
        return (n_tokens + self.cfg.block_size - 1) // self.cfg.block_size

    def allocate(self, n_blocks: int) -> List[int]:
        if n_blocks > len(self._free):
            raise MemoryError(f"KV cache exhausted: need {n_blocks}, have {len(self._free)}")
        return [self._free.pop() for _ in range(n_blocks)]

    def free(self, blocks: Sequence[int]) -> None:
        """One owner gives the blocks up; shared ones stay with the others."""
        if not self._shared:
            self._free.extend(reversed(list(blocks)))
            return
        for b in reversed(list(blocks)):
            left = self._shared.get(b, 0)
            if left == 0:
                self._free.append(b)
            elif left == 1:
                del self._shared[b]
            else:
                self._shared[b] = left - 1

    def copy_blocks(self, pairs: Sequence[Sequence[int]]) -> None:
        """Copy whole blocks (source, destination) in every layer, scales
        included, in order with the current stream."""
        pairs = [(int(s), int(d)) for s, d in pairs]
        dst = {d for _, d in pairs}
        if len(dst) != len(pairs) or any(s in dst for s, _ in pairs):
            raise ValueError("copy_blocks: a destination may be neither a source nor another pair's destination")
        if any(not 0 <= b < self.num_blocks for p in pairs for b in p):
            raise ValueError(f"copy_blocks: block ids must lie in [0, {self.num_blocks})")
        if not pairs:
            return
        t = torch.tensor(pairs, dtype=torch.int32)
        if self.kv.is_cuda:
            ops.kv_copy_blocks(self.kv, t.pin_memory().to(self.kv.device, non_blocking=True), self.scales)
            return
        from connex_b200.ops import reference as R
        R.kv_copy_blocks(self.kv, t, self.scales)

    def fork(self, blocks: Sequence[int], n_tokens: int, n: int = 1) -> List[List[int]]:
        """Block tables of ``n`` sequences that go on from the first
        ``n_tokens`` of the one with table ``blocks``: its full blocks are
        shared, a partly filled last one is copied (one launch for all)."""
        bs = self.cfg.block_size
        full, rest = divmod(n_tokens, bs)
        if n_tokens < 0 or self.blocks_needed(n_tokens) > len(blocks):
            raise ValueError(f"fork: {n_tokens} tokens do not lie in {len(blocks)} blocks")
        if n < 0:
            raise ValueError("fork: n must not be negative")
        if any(not 0 <= b < self.num_blocks for b in blocks[:self.blocks_needed(n_tokens)]):
            raise ValueError(f"fork: block ids must lie in [0, {self.num_blocks})")
        tails = self.allocate(n) if rest else []
        self.copy_blocks([(blocks[full], t) for t in tails])
        if n:
            for b in blocks[:full]:
                self._shared[b] = self._shared.get(b, 0) + n
        return [list(blocks[:full]) + tails[i:i + 1] for i in range(n)]

    def own(self, blocks: List[int], start: int, stop: int) -> None:
        """Before the sequence with table ``blocks`` (changed in place) writes its
        tokens [start, stop): shared blocks that they fall into give way to
        blocks of its own, the first of which keeps the tokens before ``start``."""
        if not self._shared:
            return
        bs = self.cfg.block_size
        at = [i for i in range(start // bs, min(len(blocks), -(-stop // bs))) if blocks[i] in self._shared]
        mine = self.allocate(len(at))
        if at and start > at[0] * bs:
            self.copy_blocks([(blocks[at[0]], mine[0])])
        for i, b in zip(at, mine):
            self.free([blocks[i]])
            blocks[i] = b

    def compact(self, tables) -> int:
        """Move the blocks of ``tables`` (the block lists of the live
        sequences, changed in place) down so that the pool's used blocks are
        its lowest ones; blocks in none of them, and shared ones with an owner
        beside them, stay where they are.  Returns the number of blocks moved."""
        tables = list({id(t): t for t in tables}.values())
        used = self.num_blocks - len(self._free)
        holes = sorted(b for b in self._free if b < used)
        owners = Counter(b for t in tables for b in set(t))
        high = sorted((b for b, n in owners.items() if b >= used and n > self._shared.get(b, 0)), reverse=True)
        moves = dict(zip(high, holes))
        if not moves:
            return 0
        self.copy_blocks(list(moves.items()))
        for t in tables:
            t[:] = [moves.get(b, b) for b in t]
        for s, d in moves.items():
            if s in self._shared:
                self._shared[d] = self._shared.pop(s)
        taken = set(moves.values())
        self._free = sorted([b for b in self._free if b not in taken] + list(moves), reverse=True)
        return len(moves)

    @property
    def free_blocks(self) -> int:
        return len(self._free)


def slot_mapping(block_ids: Sequence[int], start: int, n: int, block_size: int) -> List[int]:
    return [block_ids[(start + i) // block_size] * block_size + (start + i) % block_size for i in range(n)]


LayerHook = Callable[[int], None]


class LlamaModel:
    """Forward passes of the Llama decoder over a :class:`PagedKVCache`."""

    def __init__(self, weights: LlamaWeights, cache: PagedKVCache, max_tokens: int, max_batch: int = 256,
                 tp=None):
        """``tp``: a :class:`connex_b200.parallel.tp.TPGroup` when ``weights``
        are one rank's shard (``shard_llama``); the residual stream is then
        all-reduced after the o- and down-projections."""
        self.w = weights
        self.tp = tp
        self.cfg = weights.cfg
        self.cache = cache
        cfg = self.cfg
        dev = weights.embed.device
        self.device = dev
        self.cos_sin = ops.rope_cos_sin(cfg.max_pos, cfg.head_dim, cfg.rope_theta, dev, cfg.rope_scaling)
        self.status = ops.new_status(dev)
        self.max_tokens = max_tokens
        bf = dict(dtype=torch.bfloat16, device=dev)
        self.x = torch.empty(max_tokens, cfg.hidden, **bf)
        self.h = torch.empty(max_tokens, cfg.hidden, **bf)
        self.qkv = torch.empty(max_tokens, cfg.qkv_dim, **bf)
        self.attn = torch.empty(max_tokens, cfg.heads * cfg.head_dim, **bf)
        self.mid = torch.empty(max_tokens, cfg.ffn, **bf)
        self.last = torch.empty(max_batch, cfg.hidden, **bf)
        self.logits = torch.empty(max_batch, cfg.vocab_size, **bf)
        self.next_ids = torch.empty(max_batch, dtype=torch.int32, device=dev)
        self.max_batch = max_batch
        # e4m3 inputs of Fp8Weight projections, with their scales: the normed rows, the attention's, the MLP's
        self.q8 = {}
        if any(isinstance(getattr(lw, n), Fp8Weight) for lw in weights.layers for n in PROJECTIONS):
            for name, width in (("h", cfg.hidden), ("attn", cfg.heads * cfg.head_dim), ("mid", cfg.ffn)):
                self.q8[name] = (torch.empty(max_tokens, width, dtype=torch.float8_e4m3fn, device=dev),
                                 torch.empty(max_tokens * -(-width // ops.FP8_BLOCK), dtype=torch.float32, device=dev))

    # ------------------------------------------------------------ layers
    def _q8(self, name: str, T: int):
        """The first ``T`` rows of an e4m3 buffer and of its scales."""
        q, s = self.q8[name]
        return q[:T], s[:T * -(-q.shape[1] // ops.FP8_BLOCK)].view(-1, T).t()

    def _norm(self, x: torch.Tensor, norm: torch.Tensor, w, T: int) -> None:
        """RMSNorm of ``x`` as the input of the projection ``w`` (None: the head's)."""
        if isinstance(w, Fp8Weight):
            q, s = self._q8("h", T)
            ops.quantize_fp8(x, norm=norm, eps=self.cfg.eps, out=q, scale=s)
        else:
            ops.rmsnorm(x, norm, self.cfg.eps, out=self.h[:T])

    def _qkv(self, lw: LayerWeights, T: int) -> torch.Tensor:
        """The fused projection of the rows that :meth:`_norm` left."""
        qkv = self.qkv[:T]
        if isinstance(lw.wqkv, Fp8Weight):
            ops.gemm_fp8(*self._q8("h", T), lw.wqkv.q, lw.wqkv.scale, out=qkv, status=self.status)
        else:
            ops.gemm(self.h[:T], lw.wqkv, qkv, status=self.status)
        return qkv

    def _mlp(self, lw: LayerWeights, T: int, x: torch.Tensor) -> None:
        """x += down(SiLU(gate) * up) of the rows that :meth:`_norm` left."""
        q13, q2 = isinstance(lw.w13, Fp8Weight), isinstance(lw.w2, Fp8Weight)
        mid = self.mid[:T]
        if q13:
            q, s = self._q8("mid", T)
            out, scale = (q, s) if q2 else (mid, None)
            ops.gemm_fp8(*self._q8("h", T), lw.w13.q, lw.w13.scale, out=out, out_scale=scale, silu_mul=True,
                         status=self.status)
        else:
            ops.gemm(self.h[:T], lw.w13, mid, silu_mul=True, status=self.status)
        self._residual_gemm(mid, lw.w2, x, "mid", quantised=q13 and q2)

    def _residual_gemm(self, a: torch.Tensor, w, x: torch.Tensor, name: str = "attn", quantised: bool = False) -> None:
        """x += a @ w^T; under tensor parallelism summed over the group: rank 0
        adds its partial to x in the epilogue, the others store theirs into
        x, and an all-reduce of x adds them up.  ``name``: the buffer that
        ``a`` is quantised into for an Fp8Weight; it holds it already if
        ``quantised``."""
        tp = self.tp
        alone = tp is None or tp.world == 1
        residual = x if alone or tp.rank == 0 else None
        if isinstance(w, Fp8Weight):
            q, s = self._q8(name, x.shape[0])
            if not quantised:
                ops.quantize_fp8(a, out=q, scale=s)
            ops.gemm_fp8(q, s, w.q, w.scale, out=x, residual=residual, status=self.status)
        else:
            ops.gemm(a, w, x, residual=residual, status=self.status)
        if not alone:
            tp.all_reduce(x)

    def _rotate_and_cache(self, i: int, qkv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
                          **norms) -> torch.Tensor:
        """Rotate q (in place) and write the rows' K and V to layer ``i`` of the
        cache; returns what the attention reads its queries from."""
        cfg, c = self.cfg, self.cache
        if c.kind == "bf16":
            ops.rope_cache(qkv, positions, self.cos_sin, cfg.heads, cfg.kv_heads, slots, c.k(i), c.v(i),
                           status=self.status, **norms)
            return qkv
        if c.kind == "int4":
            return ops.rope_cache_int4(qkv, positions, self.cos_sin, cfg.heads, cfg.kv_heads, slots, c.k(i), c.v(i),
                                       out=qkv[:, :cfg.heads * cfg.head_dim], status=self.status, **norms)
        return ops.rope_cache_fp8(qkv, positions, self.cos_sin, cfg.heads, cfg.kv_heads, slots, c.k(i), c.v(i),
                                  c.k_scale(i), c.v_scale(i), out=qkv[:, :cfg.heads * cfg.head_dim],
                                  status=self.status, **norms)

    def _decode_attention(self, i: int, q: torch.Tensor, block_tables: torch.Tensor, ctx_lens: torch.Tensor,
                          max_ctx: int, workspace: torch.Tensor, out: torch.Tensor) -> None:
        cfg, c = self.cfg, self.cache
        if c.kind == "int4":
            ops.decode_attention_int4(q, c.k(i), c.v(i), block_tables, ctx_lens, cfg.heads, workspace, out=out,
                                      status=self.status)
        elif c.kind == "bf16":
            ops.decode_attention(q, c.k(i), c.v(i), block_tables, ctx_lens, cfg.heads, max_ctx, workspace, out=out)
        else:
            ops.decode_attention_fp8(q, c.k(i), c.v(i), c.k_scale(i), c.v_scale(i), block_tables, ctx_lens, cfg.heads,
                                     workspace, out=out, status=self.status)

    def _chunk_attention(self, i: int, q: torch.Tensor, block_tables: torch.Tensor, tile_info: torch.Tensor,
                         out: torch.Tensor, n_blocks: Optional[int] = None) -> None:
        cfg, c = self.cfg, self.cache
        if c.kind == "int4":
            ops.prefill_attention_paged_int4(q, c.k(i), c.v(i), block_tables, tile_info, cfg.heads, cfg.kv_heads, out=out,
                                             status=self.status, n_blocks=n_blocks)
        elif c.kind == "bf16":
            ops.prefill_attention_paged(q, c.k(i), c.v(i), block_tables, tile_info, cfg.heads, cfg.kv_heads, out=out,
                                        status=self.status)
        else:
            ops.prefill_attention_paged_fp8(q, c.k(i), c.v(i), c.k_scale(i), c.v_scale(i), block_tables, tile_info,
                                            cfg.heads, cfg.kv_heads, out=out, status=self.status, n_blocks=n_blocks)

    def decode_workspace(self, max_batch: int, max_ctx: int) -> torch.Tensor:
        """The decode attention's workspace for this model's cache."""
        cfg = self.cfg
        if self.cache.kind == "bf16":
            return ops.decode_workspace(max_batch, cfg.heads, max_ctx, self.device)
        if self.cache.kind == "int4":
            return ops.decode_workspace_int4(max_batch, cfg.heads, cfg.kv_heads, self.device)
        return ops.decode_workspace_fp8(max_batch, cfg.heads, cfg.kv_heads, self.device)

    def _layer_tail(self, l: int, T: int):
        layers, lw, x = self.w.layers, self.w.layers[l], self.x[:T]
        self._residual_gemm(self.attn[:T], lw.wo, x)
        self._norm(x, lw.mlp_norm, lw.w13, T)
        self._mlp(lw, T, x)
        if l + 1 < len(layers):
            self._norm(x, layers[l + 1].attn_norm, layers[l + 1].wqkv, T)
        else:
            self._norm(x, self.w.final_norm, None, T)

    def _head(self, rows: torch.Tensor, B: int) -> torch.Tensor:
        last = self.last[:B]
        ops.gather_rows(self.h, rows, last)
        logits = self.logits[:B]
        ops.gemm(last, self.w.lm_head, logits, status=self.status)
        return ops.argmax(logits, self.next_ids[:B])

    def prefill(self, ids: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
                seq_lens: Sequence[int], last_rows: torch.Tensor, tile_info: torch.Tensor,
                layer_hook: Optional[LayerHook] = None, hook_after_attention: bool = False,
                block_tables: Optional[torch.Tensor] = None, n_blocks: Optional[int] = None) -> torch.Tensor:
        """Prefill a packed batch; returns the greedy next token of each sequence.

        With an 8-bit or a 4-bit cache the attention reads it: ``block_tables`` [B,
        max_blocks] is then needed, and ``tile_info`` from
        ``prefill_tile_info(seq_lens, device, ctx)``; ``n_blocks``, the blocks
        that the sequences have together, bounds the workspace (by default the
        tables' size, as much as the longest sequence takes for each of them).

        ``layer_hook(l)`` runs (on the host, in stream order) right after layer
        l's K/V are in the paged cache: the PD path launches its push there.
        With ``hook_after_attention`` it runs after layer l's attention has
        been enqueued instead (the push then overlaps the layer's GEMMs rather
        than its attention kernel)."""
        cfg, T = self.cfg, ids.numel()
        assert T <= self.max_tokens
        if self.cache.kind != "bf16" and block_tables is None:
            raise ValueError("prefill over an 8-bit cache, or one of 4 bits, needs block_tables")
        nvtx.push(f"prefill T={T}")
        ops.embedding(ids, self.w.embed, self.x[:T], status=self.status)
        self._norm(self.x[:T], self.w.layers[0].attn_norm, self.w.layers[0].wqkv, T)
        for l, lw in enumerate(self.w.layers):
            nvtx.push(f"layer {l}")
            qkv = self._qkv(lw, T)
            q = self._rotate_and_cache(l, qkv, positions, slots)
            if layer_hook is not None and not hook_after_attention:
                layer_hook(l)
            if self.cache.kind == "bf16":
                ops.prefill_attention(qkv, tile_info, cfg.heads, cfg.kv_heads, out=self.attn[:T])
            else:
                self._chunk_attention(l, q, block_tables, tile_info, self.attn[:T], n_blocks)
            if layer_hook is not None and hook_after_attention:
                layer_hook(l)
            self._layer_tail(l, T)
            nvtx.pop()
        out = self._head(last_rows, len(seq_lens))
        nvtx.pop()
        return out

    def decode(self, ids: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
               block_tables: torch.Tensor, ctx_lens: torch.Tensor, max_ctx: int,
               workspace: torch.Tensor, rows: torch.Tensor) -> torch.Tensor:
        """One decode step for B sequences (ctx_lens include the new token);
        ``workspace`` from :meth:`decode_workspace`."""
        cfg, B = self.cfg, ids.numel()
        nvtx.push(f"decode B={B}")
        ops.embedding(ids, self.w.embed, self.x[:B], status=self.status)
        self._norm(self.x[:B], self.w.layers[0].attn_norm, self.w.layers[0].wqkv, B)
        for l, lw in enumerate(self.w.layers):
            qkv = self._qkv(lw, B)
            q = self._rotate_and_cache(l, qkv, positions, slots)
            self._decode_attention(l, q, block_tables, ctx_lens, max_ctx, workspace, self.attn[:B])
            self._layer_tail(l, B)
        out = self._head(rows, B)
        nvtx.pop()
        return out


# ------------------------------------------------------------- oracle
def reference_forward(weights: LlamaWeights, seqs: Sequence[Sequence[int]]) -> List[torch.Tensor]:
    """fp32 PyTorch forward (no cache) returning last-position logits per sequence."""
    from connex_b200.ops import reference as R

    def plain(w):
        return w.float() if isinstance(w, Fp8Weight) else w
    cfg = weights.cfg
    cos_sin = ops.rope_cos_sin(cfg.max_pos, cfg.head_dim, cfg.rope_theta, weights.embed.device,
                               cfg.rope_scaling)
    outs = []
    for seq in seqs:
        ids = torch.tensor(seq, device=weights.embed.device)
        n = len(seq)
        pos = torch.arange(n, device=ids.device)
        x = weights.embed[ids].float()
        for lw in weights.layers:
            h = R.rmsnorm(x, lw.attn_norm, cfg.eps)
            qkv = h @ lw.wqkv.float().t()
            q = qkv[:, :cfg.heads * 128].view(n, cfg.heads, 128)
            k = qkv[:, cfg.heads * 128:(cfg.heads + cfg.kv_heads) * 128].view(n, cfg.kv_heads, 128)
            v = qkv[:, (cfg.heads + cfg.kv_heads) * 128:].view(n, cfg.kv_heads, 128)
            q, k = R.rope(q, pos, cos_sin), R.rope(k, pos, cos_sin)
            a = R.causal_attention(q, k, v, [n]).reshape(n, -1)
            x = x + a @ lw.wo.float().t()
            h = R.rmsnorm(x, lw.mlp_norm, cfg.eps)
            x = x + R.silu_mul_gemm(h, plain(lw.w13)) @ lw.w2.float().t()
        h = R.rmsnorm(x[-1:], weights.final_norm, cfg.eps)
        outs.append((h @ weights.lm_head.float().t())[0])
    return outs
