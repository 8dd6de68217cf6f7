"""Block-scaled fp8 projections and the 4-bit KV cache together on the GPU: steps
captured and replayed, calls on two streams, far offsets, and the runtimes that
serve with them."""
import pytest
import torch

pytestmark = pytest.mark.gpu

D, BS, ROW = 128, 16, 72
U_BF16, U_E4M3 = 2.0 ** -8, 2.0 ** -4


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def _g(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _weight(n, k, dev, seed):
    from connex_b200.models.llama import Fp8Weight
    return Fp8Weight.of((torch.randn(n, k, generator=_g(dev, seed), device=dev) * 0.05).to(torch.bfloat16))


def test_layer_in_a_graph(dev):
    """A layer's operators in their order, captured and replayed while the lengths grow, next to the same steps run
    eagerly; two graphs with a workspace each, replayed on two streams."""
    from connex_b200 import ops
    hq, hkv, B, width, H, F = 8, 2, 5, 8, 512, 768
    nb = B * width + 1
    table = torch.arange(1, nb, dtype=torch.int32, device=dev).view(B, width)
    cs = ops.rope_cos_sin(256, D, 1e4, dev)
    norm = (torch.rand(H, generator=_g(dev, 1), device=dev) + 0.5).to(torch.bfloat16)
    wqkv, wo = _weight((hq + 2 * hkv) * D, H, dev, 2), _weight(H, hq * D, dev, 3)
    w13, w2 = _weight(2 * F, H, dev, 4), _weight(H, F, dev, 5)

    def make():
        return dict(k=torch.zeros(nb, hkv, BS, ROW, dtype=torch.uint8, device=dev),
                    v=torch.zeros(nb, hkv, BS, ROW, dtype=torch.uint8, device=dev),
                    x=torch.zeros(B, H, dtype=torch.bfloat16, device=dev), pos=torch.zeros(B, dtype=torch.int32, device=dev),
                    slots=torch.full((B,), -1, dtype=torch.int64, device=dev),
                    lens=torch.ones(B, dtype=torch.int32, device=dev), ws=ops.decode_workspace_int4(B, hq, hkv, dev),
                    st=ops.new_status(dev))

    def step(s):
        st = s["st"]
        qkv = ops.gemm_fp8(*ops.quantize_fp8(s["x"], norm=norm), wqkv.q, wqkv.scale, status=st)
        q = ops.rope_cache_int4(qkv, s["pos"], cs, hq, hkv, s["slots"], s["k"], s["v"], status=st)
        a = ops.decode_attention_int4(q, s["k"], s["v"], table, s["lens"], hq, s["ws"], status=st)
        y = ops.gemm_fp8(*ops.quantize_fp8(a), wo.q, wo.scale, residual=s["x"], status=st)
        mid = ops.gemm_fp8(*ops.quantize_fp8(y, norm=norm), w13.q, w13.scale, silu_mul=True, status=st)
        return ops.gemm_fp8(*mid, w2.q, w2.scale, residual=y, status=st)
    sides = [make() for _ in range(3)]
    graphs = []
    for s in sides[:2]:
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            step(s)
        stream.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(s)
        graphs.append((g, out, stream))
    for s in sides[:2]:
        s["k"].zero_(), s["v"].zero_()
    for t in range(40):
        x = (torch.randn(B, H, generator=_g(dev, 200 + t), device=dev) * (1 + t % 7)).to(torch.bfloat16)
        pos = torch.tensor([(t + 3 * b) % 100 for b in range(B)], dtype=torch.int32, device=dev)
        for s in sides:
            s["x"].copy_(x)
            s["pos"].copy_(pos)
            s["slots"].copy_(table.gather(1, (pos.long() // BS)[:, None])[:, 0].long() * BS + pos.long() % BS)
            s["lens"].copy_(pos + 1)
        torch.cuda.synchronize()
        for g, _, stream in graphs:
            with torch.cuda.stream(stream):
                g.replay()
        eager = step(sides[2])
        torch.cuda.synchronize()
        for (_, out, _), s in zip(graphs, sides):
            assert torch.equal(out.view(torch.int16), eager.view(torch.int16)), t
            assert torch.equal(s["k"], sides[2]["k"]) and torch.equal(s["v"], sides[2]["v"])
    for s in sides:
        ops.check_status(s["st"])


def test_two_streams_at_once(dev):
    """Calls on two streams, each with a workspace of its own, give the bits of calls one after another."""
    from connex_b200 import ops
    from connex_b200.ops import reference as R
    hq, hkv = 16, 4
    sides = []
    for i, (lens, m) in enumerate((([3000, 17, 900], 40), ([64, 5000, 1, 333], 700))):
        nb = [-(-n // BS) for n in lens]
        table = torch.zeros(len(lens), max(nb), dtype=torch.int32, device=dev)
        for b, n in enumerate(nb):
            table[b, :n] = torch.arange(n, device=dev) + sum(nb[:b])
        k, v = (R.int4_rows(torch.randn(sum(nb), hkv, BS, D, generator=_g(dev, 10 + 2 * i + j), device=dev).to(torch.bfloat16))
                for j in range(2))
        new = [min(n, 70) for n in lens]
        q = torch.randn(sum(new), hq * D, generator=_g(dev, 20 + i), device=dev).to(torch.bfloat16)
        x = torch.randn(m, 2048, generator=_g(dev, 30 + i), device=dev).to(torch.bfloat16)
        sides.append(((k, v, table), q, torch.tensor(lens, dtype=torch.int32, device=dev),
                      ops.prefill_tile_info(new, dev, ctx=[n - c for n, c in zip(lens, new)]),
                      ops.decode_workspace_int4(len(lens), hq, hkv, dev), x, _weight(1536, 2048, dev, 40 + i)))

    def run(side):
        cache, q, lens, ti, ws, x, w = side
        a, s = ops.quantize_fp8(x)
        return (ops.decode_attention_int4(q[:len(lens)], *cache, lens, hq, ws),
                ops.prefill_attention_paged_int4(q, *cache, ti, hq, hkv), ops.gemm_fp8(a, s, w.q, w.scale),
                *(t.view(torch.uint8) if t.element_size() == 1 else t
                  for t in ops.gemm_fp8(a, s, w.q, w.scale, silu_mul=True)))
    want = [run(side) for side in sides]
    streams = [torch.cuda.Stream(dev) for _ in sides]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (side, stream) in enumerate(zip(sides, streams)):
            with torch.cuda.stream(stream):
                got[i].append(run(side))
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        assert all(torch.equal(x, y) for r in runs for x, y in zip(r, w))


def test_offsets_past_32_bits(dev):
    """Blocks that lie more than 4 GB into the cache give the bits of the same blocks at its start, and so do rows of a
    product whose result is larger than that."""
    from connex_b200 import ops
    hq, hkv, far = 16, 8, 470000
    assert far * hkv * BS * ROW > 2 ** 32
    n, T = 40, 600
    big = torch.zeros(2, far + n, hkv, BS, ROW, dtype=torch.uint8, device=dev)
    qkv = torch.randn(T, (hq + 2 * hkv) * D, generator=_g(dev, 141), device=dev).to(torch.bfloat16)
    cs = ops.rope_cos_sin(T, D, 5e5, dev)
    pos = torch.arange(T, dtype=torch.int32, device=dev)
    ws = ops.decode_workspace_int4(1, hq, hkv, dev)
    lens = torch.tensor([T], dtype=torch.int32, device=dev)
    ti = ops.prefill_tile_info([T], dev, ctx=[0])
    got = []
    for at in (0, far):
        st = ops.new_status(dev)
        q = ops.rope_cache_int4(qkv, pos, cs, hq, hkv, torch.arange(T, device=dev) + at * BS, big[0], big[1], status=st)
        table = torch.arange(at, at + n, dtype=torch.int32, device=dev)[None]
        got.append((big[:, at:at + n].clone(), ops.kv_values_int4(big[1])[at:at + n].clone(),
                    ops.decode_attention_int4(q[-1:], big[0], big[1], table, lens, hq, ws, status=st),
                    ops.prefill_attention_paged_int4(q, big[0], big[1], table, ti, hq, hkv, status=st)))
        ops.check_status(st)
    assert all(torch.equal(a, b) for a, b in zip(*got))
    del big, got
    M, N, K = 70000, 32000, 128
    assert M * N * 2 > 2 ** 32
    x = torch.randn(M, K, generator=_g(dev, 142), device=dev).to(torch.bfloat16)
    a, s = ops.quantize_fp8(x)
    w = _weight(N, K, dev, 143)
    out = ops.gemm_fp8(a, s, w.q, w.scale)
    for r0 in (0, 35000, M - 300):
        part = ops.gemm_fp8(a[r0:r0 + 300], s[r0:r0 + 300], w.q, w.scale)
        assert torch.equal(out[r0:r0 + 300], part)


def _runtime(dev, kv, fp8, layers=2, seed=0):
    from connex_b200.models.llama import LlamaConfig
    from connex_b200.runtime.pp import StageRuntime, stage_weights
    cfg = LlamaConfig.tiny(layers=2)
    w = stage_weights(cfg, 0, layers, dev, seed)
    if fp8:
        w = w.to_fp8()
    return cfg, StageRuntime(cfg, 0, layers, dev, num_blocks=128, max_tokens=512, max_batch=8, max_ctx=512, weights=w,
                             kv_dtype=kv)


def _compute(rt, kind, rids, ctx, n_new, ids, n_dec=None):
    from connex.pp.handover import CX_CTX, REQUEST_IDS
    td = {"kind": kind, REQUEST_IDS: rids, CX_CTX: ctx, "n_new": n_new,
          "ids": torch.tensor(ids, dtype=torch.int32, device=rt.device)}
    if n_dec is not None:
        td["n_dec"] = n_dec
    out = rt.compute(td, [])
    return out["x"].float() if "x" in out else out["next"]


def test_stage_runtime(dev):
    """A stage with e4m3 projections over a 4-bit cache: residual rows near those of the plain stage, whole or chunked
    prompt, decode rows in the same steps."""
    g = torch.Generator().manual_seed(3)
    prompt = torch.randint(3, 1000, (200,), generator=g).tolist()
    got = {}
    for name, kv, fp8 in (("plain", torch.bfloat16, False), ("kv", torch.uint8, False), ("both", torch.uint8, True)):
        _, rt = _runtime(dev, kv, fp8, layers=1)
        whole = _compute(rt, "prefill", ["w"], [0], [200], prompt)
        parts, done = [], 0
        for n in (16, 1, 50, 133):
            parts.append(_compute(rt, "mixed", ["c"], [done], [n], prompt[done:done + n], n_dec=1 if n == 1 else 0))
            done += n
        dec = _compute(rt, "decode", ["w", "c"], [200, 200], [1, 1], [5, 5])
        mix = _compute(rt, "mixed", ["w", "d"], [201, 0], [1, 40], [7] + prompt[:40], n_dec=1)
        torch.cuda.synchronize()
        assert int(rt.model.status) == 0
        got[name] = (whole, torch.cat(parts), dec, mix)
    # the attention's share of the residual changes by the cache's steps, a thirtieth of a half's range each; the random
    # weights' attention output is a small part of the rows
    for x, y in zip(got["plain"], got["kv"]):
        assert (x - y).norm() <= 2.0 ** -3 * x.norm()
    # on the way to the residual a row is rounded to e4m3 as the MLP's input and in its middle, and its weights twice:
    # four times 2^-4 of a vector at most
    for x, y in zip(got["plain"], got["both"]):
        assert (x - y).norm() <= 4 * U_E4M3 * x.norm()
    # each token's row is quantised by itself: chunks and whole prompts differ by bf16 roundings only (those of the
    # products' sums, and of what they tip over to another code)
    w, c, dec, _ = got["both"]
    assert (w - c).norm() <= 2.0 ** -5 * w.norm()
    assert (dec[0] - dec[1]).norm() <= 2.0 ** -5 * dec[0].norm()


def test_decode_graphs_and_fork(dev):
    """Decode graphs (padding rows on one trash slot) give the eager rows; forked requests continue like their parent,
    before and after a compaction."""
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(3, 1000, (n,), generator=g).tolist() for n in (37, 16, 90)]
    outs = []
    for graphs in (False, True):
        cfg, rt = _runtime(dev, torch.uint8, True)
        if graphs:
            rt.enable_decode_graphs((4, 8))
        _compute(rt, "prefill", ["a", "b", "c"], [0] * 3, [len(p) for p in prompts], sum(prompts, []))
        lens, steps = [len(p) for p in prompts], []
        for t in range(20):
            steps.append(_compute(rt, "decode", ["a", "b", "c"], lens, [1] * 3, [7 + t, 9 + t, 11 + t]).tolist())
            lens = [n + 1 for n in lens]
        rt.fork("a", ["x", "y"])
        rt.release(["b"])
        assert rt.compact() > 0 or graphs
        for t in range(18):
            s = _compute(rt, "decode", ["a", "x", "y", "c"], [lens[0]] * 3 + [lens[2]], [1] * 4, [30 + t] * 3 + [t + 3]).tolist()
            assert s[0] == s[1] == s[2]
            steps.append(s)
            lens = [n + 1 for n in lens]
        rt.release(["a", "x", "y", "c"])
        assert rt.cache.free_blocks == 128 - (1 if graphs else 0) and not rt.cache._shared
        assert int(rt.model.status) == 0
        outs.append(steps)
    assert outs[0] == outs[1]


@pytest.mark.parametrize("tie", [False, True])
def test_model_against_the_oracle(dev, tie):
    """Prefill and decode of the model; its logits' argmax lies near the top of the fp32 oracle's of the same weights."""
    from connex_b200 import ops
    from connex_b200.models.llama import LlamaConfig, LlamaModel, LlamaWeights, PagedKVCache, reference_forward, slot_mapping
    cfg = LlamaConfig.tiny(layers=2)
    w = LlamaWeights.random(cfg, dev, seed=1).to_fp8()
    if tie:
        w.lm_head = w.embed
    cache = PagedKVCache(cfg, 64, dev, torch.uint8)
    model = LlamaModel(w, cache, max_tokens=512, max_batch=4)
    seq = list(range(3, 140))
    blocks = cache.allocate(cache.blocks_needed(len(seq) + 1))
    t = lambda x, dt: torch.tensor(x, dtype=dt, device=dev)  # noqa: E731
    bt = t([blocks], torch.int32)
    nxt = model.prefill(t(seq, torch.int32), t(list(range(len(seq))), torch.int32),
                        t(slot_mapping(blocks, 0, len(seq), cfg.block_size), torch.int64), [len(seq)],
                        t([len(seq) - 1], torch.int32), ops.prefill_tile_info([len(seq)], dev, ctx=[0]), block_tables=bt)
    tok = int(nxt[0])
    ws = model.decode_workspace(1, len(seq) + 1)
    model.decode(nxt[:1].clone(), t([len(seq)], torch.int32), t(slot_mapping(blocks, len(seq), 1, cfg.block_size), torch.int64),
                 bt, t([len(seq) + 1], torch.int32), len(seq) + 1, ws, t([0], torch.int32))
    torch.cuda.synchronize()
    ops.check_status(model.status)
    # two layers of four roundings of 2^-4 at most, as a share of the logits' norm
    ref = reference_forward(w, [seq + [tok]])[0]
    got = model.logits[0].float()
    assert (got - ref).norm() <= 8 * U_E4M3 * ref.norm()
    k, v = cache.values(1, blocks)
    assert k.shape == (len(blocks), cfg.kv_heads, BS, D) and torch.isfinite(v.float().view(-1, BS, D)[:2]).all()


def test_model_stepper(dev):
    """The serving engine's stepper with e4m3 projections over a 4-bit cache: prefill, chunked prefill and decode agree."""
    from connex_b200.models.llama import LlamaConfig
    from connex_b200.serve.engine import ModelStepper
    st = ModelStepper(LlamaConfig.tiny(), dev, 96, max_batch=4, max_ctx=256, max_step_tokens=256, kv_dtype="int4",
                      weight_dtype="fp8")
    seq = list(range(3, 80))
    a = st.prefill(["p"], [seq])
    b = st.mixed(["q"], [seq], [0], [64])
    b = st.mixed(["q"], [seq], [64], [13])
    assert a == b
    d1 = st.decode(["p", "q"], [seq + a, seq + a])
    assert d1[0] == d1[1]
    st.release(["p", "q"])


def test_checkpoint_to_fp8(dev, tmp_path):
    """load_llama(fp8=True) holds the checkpoint's values to half an e4m3 step."""
    from connex_b200.models import hf
    from connex_b200.models.llama import Fp8Weight, LlamaConfig, LlamaWeights
    cfg = LlamaConfig.tiny(layers=1)
    w = LlamaWeights.random(cfg, "cpu", seed=3)
    hf.save_llama(w, str(tmp_path))
    got = hf.load_llama(str(tmp_path), dev, fp8=True).layers[0]
    for n in ("wqkv", "wo", "w13", "w2"):
        q, x = getattr(got, n), getattr(w.layers[0], n).to(dev).float()
        assert isinstance(q, Fp8Weight)
        step = 2.0 ** -10 * q.scale.repeat_interleave(128, 0).repeat_interleave(128, 1)
        assert ((q.float() - x).abs() <= (U_E4M3 * x.abs()).maximum(step) * (1 + 2.0 ** -10)).all()
    assert got.attn_norm.dtype == torch.bfloat16


def test_qwen3_moe_rank(dev):
    """Decode steps with q/k norms over a 4-bit cache: layer 0 holds the bf16 cache's rows to half a step (its input does
    not depend on the cache), and the last layer's attention is that of the cache it left."""
    from connex_b200 import ops
    from connex_b200.models.qwen3_moe import Qwen3MoeConfig, Qwen3MoeRank
    from connex_b200.ops import reference as R

    class NoExperts:
        def forward(self, h, idx, w, l2p, cnt, out):
            return out.zero_()
    cfg, B, steps, width = Qwen3MoeConfig.tiny(), 3, 37, 4
    lens0 = [0, 5, 16]
    table = torch.randperm(B * width, generator=_g(dev, 171), device=dev).to(torch.int32).view(B, width)
    ids = torch.randint(3, 1000, (steps, B), generator=_g(dev, 172), device=dev).to(torch.int32)
    none = [(None, None)] * cfg.layers
    models = {}
    for dtype in (torch.bfloat16, torch.uint8):
        m = models[dtype] = Qwen3MoeRank(cfg, 0, 1, [[-1]] * cfg.layers, dev, B * width, B, kv_dtype=dtype)
        m.moe = NoExperts()
        for a in m.attn:
            a.q_norm.uniform_(0.5, 1.5, generator=_g(dev, 173))
            a.k_norm.uniform_(0.5, 1.5, generator=_g(dev, 174))
        m.cache.kv.zero_()                                   # rows before the first step: zeros in both
        ws = (ops.decode_workspace(B, cfg.heads, width * BS, dev) if dtype == torch.bfloat16
              else ops.decode_workspace_int4(B, cfg.heads, cfg.kv_heads, dev))
        for t in range(steps):
            pos = torch.tensor([n + t for n in lens0], dtype=torch.int32, device=dev)
            slots = table.gather(1, (pos.long() // BS)[:, None])[:, 0].long() * BS + pos.long() % BS
            m.decode(ids[t], pos, slots, table, pos + 1, width * BS, ws, none, none, none)
        ops.check_status(m.status)
    c, l = m.cache, cfg.layers - 1
    q = m.qkv[:, :cfg.heads * D].reshape(B, cfg.heads, D)
    ref, mag = R.paged_attention_int4(q, c.k(l), c.v(l), table, [n + steps - 1 for n in lens0], [1] * B)
    # weights in f16, the result in bf16; logits of at most some tens to 2^-15
    assert ((m.att.view(B, cfg.heads, D).double() - ref).abs() <= U_BF16 * ref.abs() + 2.0 ** -8 * (mag + ref.abs().max())).all()
    a, b = models[torch.bfloat16].cache, models[torch.uint8].cache
    for x, y, turned in ((a.k(0), b.k(0), True), (a.v(0), b.v(0), False)):
        x = x.double()
        h = x.unflatten(-1, (2, 64))
        step = ((h.amax(-1) - h.amin(-1)) / 15)[..., None]
        # K: both writes round the normed pair to bf16, each to 2^-8 of it, and the rotated elements again; the
        # largest magnitude of the row bounds the pair's
        d = 4 * U_BF16 * x.abs().amax(-1)[..., None, None] if turned else torch.zeros_like(step)
        err = (R.int4_values(y).unflatten(-1, (2, 64)) - h).abs()
        assert (err <= (0.5 + 15 * U_BF16) * step + 4 * d).all()
