"""Block-scaled fp8 projections and the 4-bit KV cache on the CPU: the oracles
themselves, the calls' checks of their arguments, what the models, the loader
and the command line make of them, and which way the product goes."""
import argparse

import pytest
import torch

from connex_b200 import ops
from connex_b200.models.llama import Fp8Weight, LlamaConfig, LlamaModel, LlamaWeights, PagedKVCache
from connex_b200.ops import reference as R

BS, D, ROW = 16, 128, 72


# ------------------------------------------------------------------ oracles
def test_int4_oracle_keeps_half_a_step():
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(50, 3, D, generator=g) * 3 + 1).to(torch.bfloat16)
    rows = R.int4_rows(x)
    assert rows.shape == (50, 3, ROW) and rows.dtype == torch.uint8
    h = x.double().unflatten(-1, (2, 64))
    step = (h.amax(-1) - h.amin(-1)) / 15
    err = (R.int4_values(rows).unflatten(-1, (2, 64)) - h).abs().amax(-1)
    assert (err <= (0.5 + 15 * 2.0 ** -9) * step).all()        # half of the rounded step, 2^-8 larger at most
    # the layout: byte i holds dims 2i and 2i + 1, then scale and minimum of each half
    y = torch.arange(16).repeat(8).to(torch.bfloat16)
    r = R.int4_rows(y)
    assert [int(b) for b in r[:4]] == [0x10, 0x32, 0x54, 0x76]
    assert torch.equal(r[64:].view(torch.bfloat16), torch.tensor([1.0, 0.0, 1.0, 0.0], dtype=torch.bfloat16))


def test_int4_oracle_special_values():
    x = torch.zeros(4, D, dtype=torch.bfloat16)
    x[0, 3] = float("inf")
    x[1, 64:] = 7.0
    x[2, 100] = float("nan")
    x[3, 0], x[3, 1] = torch.finfo(torch.bfloat16).max, -torch.finfo(torch.bfloat16).max
    v = R.int4_values(R.int4_rows(x))
    assert torch.isnan(v[0, :64]).all() and (v[0, 64:] == 0).all()
    assert (v[1, :64] == 0).all() and (v[1, 64:] == 7).all()
    assert torch.isnan(v[2, 64:]).all()


def test_fp8_scale_oracle():
    x = torch.zeros(130, 200)
    x[129, 199], x[0, 0] = -896.0, float("inf")
    s = R.fp8_block_scale(x, 128)
    assert s.shape == (2, 2) and float(s[1, 1]) == 2.0 and float(s[0, 0]) == 2.0 ** -100 / 448
    assert R.fp8_block_scale(x).shape == (130, 2)


# ----------------------------------------------------------------- refusals
def _f8(*shape):
    return torch.zeros(*shape, dtype=torch.uint8).view(torch.float8_e4m3fn)


def _gemm(**kw):
    a = dict(a=_f8(4, 256), a_scale=torch.ones(4, 2), b=_f8(384, 256), b_scale=torch.ones(3, 2))
    a.update(kw)
    return ops.gemm_fp8(a.pop("a"), a.pop("a_scale"), a.pop("b"), a.pop("b_scale"), **a)


BF = torch.bfloat16


@pytest.mark.parametrize("kw,match", [
    (dict(a=torch.zeros(4, 256, dtype=BF)), "a must be float8_e4m3fn"),
    (dict(a=_f8(4, 264), b=_f8(384, 264), a_scale=torch.ones(4, 3), b_scale=torch.ones(3, 3)), "multiple of 16"),
    (dict(a=_f8(4, 512)[:, ::2]), "contiguous rows"),
    (dict(a=_f8(4, 272)[:, 8:264]), "16-byte boundaries"),
    (dict(a=_f8(1, 256).expand(4, 256)), "without overlap"),
    (dict(b=_f8(384, 128)), "same columns"),
    (dict(a=_f8(4, 0), b=_f8(384, 0), a_scale=torch.ones(4, 0), b_scale=torch.ones(3, 0)), "multiple of 16|not none"),
    (dict(b=_f8(388, 256), b_scale=torch.ones(4, 2)), "multiple of 8"),
    (dict(a_scale=torch.ones(4, 3)), "a's scales"),
    (dict(a_scale=torch.ones(2, 4)), "a's scales"),
    (dict(a_scale=torch.ones(4, 2, dtype=torch.float64)), "a's scales"),
    (dict(b_scale=torch.ones(384, 2)), "b's scales"),
    (dict(out=torch.zeros(4, 392, dtype=BF)), r"out must be \[4, 384\]"),
    (dict(out=torch.zeros(4, 384)), "out must be bf16"),
    (dict(out=torch.zeros(4, 388, dtype=BF)[:, :384]), "16-byte boundaries"),
    (dict(out=_f8(4, 384)), "only the SiLU-mul"),
    (dict(residual=torch.zeros(4, 384)), "residual must be bf16"),
    (dict(residual=torch.zeros(3, 384, dtype=BF)), "out's shape"),
    (dict(silu_mul=True), "multiple of 256"),
    (dict(), "must be a CUDA tensor"),
])
def test_gemm_refusals(kw, match):
    with pytest.raises(RuntimeError, match=match):
        _gemm(**kw)


def test_gemm_refuses_a_shifted_residual():
    buf = torch.zeros(6, 384, dtype=BF)
    with pytest.raises(RuntimeError, match="overlaps the residual"):
        _gemm(out=buf[:4], residual=buf[1:5])
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):      # in place: fine but for the device
        _gemm(out=buf[:4], residual=buf[:4])
    with pytest.raises(ValueError, match="scales go with"):
        _gemm(out=buf[:4], out_scale=torch.ones(4, 3))
    with pytest.raises(ValueError, match="no residual"):
        _gemm(silu_mul=True, residual=buf[:4])
    with pytest.raises(RuntimeError, match="out's scales must not overlap"):
        _gemm(b=_f8(512, 256), b_scale=torch.ones(4, 2), silu_mul=True, out_scale=torch.ones(1, 2).expand(4, 2))


@pytest.mark.parametrize("x,kw,match", [
    (torch.zeros(3, 256), {}, "x must be bf16"),
    (torch.zeros(3, 24, dtype=BF), {}, "multiple of 16"),
    (torch.zeros(3, 512, dtype=BF)[:, ::2], {}, "contiguous rows"),
    (torch.zeros(3, 256, dtype=BF), dict(norm=torch.ones(128, dtype=BF)), "norm must be"),
    (torch.zeros(3, 256, dtype=BF), dict(norm=torch.ones(256)), "norm must be"),
    (torch.zeros(1, 16400, dtype=BF), dict(norm=torch.ones(16400, dtype=BF)), "16384 columns"),
    (torch.zeros(3, 256, dtype=BF), dict(out=_f8(3, 272)), "x's shape"),
    (torch.zeros(3, 256, dtype=BF), dict(scale=torch.ones(3, 1)), "scale must be"),
    (torch.zeros(3, 256, dtype=BF), dict(scale=torch.ones(1, 1).expand(3, 2)), "overlap"),
    (torch.zeros(3, 256, dtype=BF), {}, "must be a CUDA tensor"),
])
def test_quantize_refusals(x, kw, match):
    with pytest.raises(RuntimeError, match=match):
        ops.quantize_fp8(x, **kw)


def test_quantize_weight_refusals():
    with pytest.raises(RuntimeError, match="w must be bf16"):
        ops.quantize_weight_fp8(torch.zeros(128, 128))
    with pytest.raises(RuntimeError, match="scale must be"):
        ops.quantize_weight_fp8(torch.zeros(128, 256, dtype=BF), scale=torch.ones(2, 1))
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        ops.quantize_weight_fp8(torch.zeros(128, 256, dtype=BF))


def _args(hq=4, hkv=2, T=3, nb=5):
    c = lambda: torch.zeros(nb, hkv, BS, ROW, dtype=torch.uint8)  # noqa: E731
    return dict(qkv=torch.zeros(T, (hq + 2 * hkv) * D, dtype=BF), pos=torch.zeros(T, dtype=torch.int32),
                cs=torch.zeros(8, D), slots=torch.zeros(T, dtype=torch.int64), k=c(), v=c(),
                q=torch.zeros(T, hq * D, dtype=BF), bt=torch.zeros(T, 4, dtype=torch.int32),
                lens=torch.ones(T, dtype=torch.int32), ws=torch.zeros(4, hq // hkv * 136),
                ti=torch.zeros(1, 5, dtype=torch.int32))


def _write(a, hq=4, hkv=2, **kw):
    return ops.rope_cache_int4(a["qkv"], a["pos"], a["cs"], hq, hkv, a["slots"], a["k"], a["v"], **kw)


def _decode(a, hq=4, **kw):
    return ops.decode_attention_int4(a["q"], a["k"], a["v"], a["bt"], a["lens"], hq, a["ws"], **kw)


def _prefill(a, hq=4, hkv=2, **kw):
    return ops.prefill_attention_paged_int4(a["q"], a["k"], a["v"], a["bt"], a["ti"], hq, hkv, **kw)


@pytest.mark.parametrize("call", [_write, _decode, _prefill])
@pytest.mark.parametrize("bad,match", [
    (dict(k=torch.zeros(5, 2, BS, D, dtype=BF)), "caches must be contiguous uint8"),
    (dict(k=torch.zeros(5, 2, BS, 64, dtype=torch.uint8)), "caches must be"),
    (dict(v=torch.zeros(6, 2, BS, ROW, dtype=torch.uint8)), "caches must be"),
    (dict(k=torch.zeros(5, 2, BS, ROW, dtype=torch.int8)), "caches must be"),
    (dict(k=torch.zeros(5, 2, 32, ROW, dtype=torch.uint8)[:, :, ::2]), "caches must be"),
    (dict(k=torch.zeros(5 * 2 * BS * ROW + 8, dtype=torch.uint8)[8:].view(5, 2, BS, ROW)), "16-byte boundary"),
])
def test_int4_cache_refusals(call, bad, match):
    with pytest.raises(RuntimeError, match=match):
        call({**_args(), **bad})


@pytest.mark.parametrize("call,bad,match", [
    (_write, dict(qkv=torch.zeros(3, 7 * D, dtype=BF)), "exactly"),
    (_write, dict(qkv=torch.zeros(3, 8 * D)), "must be bf16"),
    (_write, dict(pos=torch.zeros(3, dtype=torch.int64)), "positions"),
    (_write, dict(slots=torch.zeros(4, dtype=torch.int64)), "slot_mapping"),
    (_write, dict(cs=torch.zeros(8, 64)), "cos_sin"),
    (_decode, dict(q=torch.zeros(3, 3 * D, dtype=BF)), "Hq heads"),
    (_decode, dict(lens=torch.ones(2, dtype=torch.int32)), "ctx_lens"),
    (_decode, dict(bt=torch.zeros(2, 4, dtype=torch.int32)), "block_tables"),
    (_prefill, dict(ti=torch.zeros(1, 3, dtype=torch.int32)), "tile_info"),
    (_prefill, dict(bt=torch.zeros(3, 4, dtype=torch.int64)), "block_tables"),
    (_write, {}, "must be a CUDA tensor"), (_decode, {}, "must be a CUDA tensor"), (_prefill, {}, "must be a CUDA tensor"),
])
def test_int4_call_refusals(call, bad, match):
    with pytest.raises(RuntimeError, match=match):
        call({**_args(), **bad})


def test_int4_more_refusals():
    a = _args()
    with pytest.raises(RuntimeError, match="q/k norm"):
        _write(a, q_norm=torch.ones(64, dtype=BF))
    with pytest.raises(RuntimeError, match="overlaps"):
        _write(a, out=a["qkv"][:, D:5 * D])
    with pytest.raises(RuntimeError, match="scale must be positive"):
        _prefill(a, scale=-1.0)
    with pytest.raises(RuntimeError, match="16 of them"):
        _decode({**a, "q": torch.zeros(3, 34 * D, dtype=BF)}, hq=34)
    with pytest.raises(ValueError, match="16 query heads"):
        ops.decode_workspace_int4(4, 34, 2, "cuda:0")
    with pytest.raises(ValueError, match="multiple of the KV heads"):
        ops.decode_workspace_int4(4, 10, 4, "cuda:0")
    many = 4097
    with pytest.raises(RuntimeError, match="at most 4096 sequences"):
        _decode({**a, "q": torch.zeros(many, 4 * D, dtype=BF), "bt": torch.zeros(many, 1, dtype=torch.int32),
                 "lens": torch.ones(many, dtype=torch.int32)})
    with pytest.raises(RuntimeError, match=r"uint8 \[..., 72\]"):
        ops.kv_values_int4(torch.zeros(3, 64, dtype=torch.uint8))
    with pytest.raises(RuntimeError, match="out must be"):
        ops.kv_values_int4(torch.zeros(3, ROW, dtype=torch.uint8), out=torch.zeros(3, 64, dtype=BF))
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        ops.kv_values_int4(torch.zeros(3, ROW, dtype=torch.uint8))


# --------------------------------------------------------------------- plan
def test_gemm_plan():
    plan = lambda m, n, k, epi=0: ops._C.gemm_fp8_plan(m, n, k, epi, 148)  # noqa: E731
    for m in (1, 2, 17, 64, 200, 613, 2048, 8192, 1 << 20, (1 << 30) - 1):
        for n in (8, 136, 2048, 28672, 128256):
            for k in (16, 128, 768, 4096, 14336):
                for epi in (0, 1, 2):
                    nt, splits = plan(m, n, k, epi)
                    assert nt in ((0, 16, 32, 64, 128) if epi == 2 else (0, 16, 32, 64, 128, 256))
                    assert splits in (1, 2, 4, 8) and splits <= -(-k // 128)
                    if nt:
                        assert -(-m // nt) <= 65535
    assert plan(8192, 28672, 4096, 2)[0] == 0 and plan(2048, 4096, 14336)[0] == 0
    assert plan(1, 6144, 4096) == (16, 4) and plan(64, 4096, 14336) == (64, 4)


# ---------------------------------------------------------- models and cache
def _cache(layers=2, blocks=12):
    return PagedKVCache(LlamaConfig.tiny(layers=layers), blocks, "cpu", torch.uint8)


def test_int4_pool_forks_copies_and_moves_rows_with_their_scales():
    c = _cache()
    assert c.kind == "int4" and c.scales is None and c.kv.shape == (2, 2, 12, 2, BS, ROW)
    assert c.head_slice_bytes == BS * ROW
    c.kv.random_(0, 255)
    t = c.allocate(3)
    was = c.kv[:, :, t].clone()
    f, = c.fork(t, 40)
    assert f[:2] == t[:2] and f[2] != t[2]
    assert torch.equal(c.kv[:, :, f], was)
    c.free(t)
    tables = [f]
    c.compact(tables)
    assert torch.equal(c.kv[:, :, tables[0]], was) and sorted(tables[0])[-1] < 3


def test_cache_values():
    cfg = LlamaConfig.tiny(layers=1)
    for dtype in (torch.bfloat16, torch.float8_e4m3fn):
        c = PagedKVCache(cfg, 5, "cpu", dtype)
        if dtype == torch.bfloat16:
            c.kv.normal_()
            want = c.kv[0, 1, [3, 0]]
        else:
            c.kv.view(torch.uint8).random_(0, 100)
            c.scales.fill_(0.5)
            want = (c.kv[0, 1].float()[[3, 0]] * 0.5).to(BF)
        k, v = c.values(0, [3, 0])
        assert k.dtype == BF and torch.equal(v, want)


def test_fp8_weight_values_and_names():
    cfg = LlamaConfig.tiny(layers=1)
    w = LlamaWeights.random(cfg, "cpu")
    lw = w.layers[0]
    q = torch.randint(0, 100, lw.w2.shape, dtype=torch.uint8).view(torch.float8_e4m3fn)
    s = torch.rand(cfg.hidden // 128, cfg.ffn // 128)
    lw.w2 = Fp8Weight(q, s)
    assert lw.w2.shape == (cfg.hidden, cfg.ffn) and torch.equal(lw.w2.float().double(), R.fp8_block_values(q, s).float().double())
    names = dict(w.named_tensors())
    assert names["model.layers.0.mlp.down_proj.weight"] is q
    assert names["model.layers.0.mlp.down_proj.weight_scale_inv"] is s
    from connex_b200.models.hf import hf_tensors
    from connex_b200.parallel.tp import shard_layer
    with pytest.raises(ValueError, match="not from quantised"):
        list(hf_tensors(w))
    with pytest.raises(ValueError, match="quantise the shards"):
        shard_layer(lw, cfg, 0, 2)


class _Calls:
    """Stands for the kernels: what they are called with, and the oracles' results where they are small."""

    def __init__(self, monkeypatch):
        self.names = []
        for name in ("rope_cache_int4", "decode_attention_int4", "prefill_attention_paged_int4", "quantize_fp8",
                     "gemm_fp8", "gemm", "rmsnorm", "embedding", "gather_rows", "argmax", "rope_cache",
                     "prefill_attention", "decode_attention"):
            monkeypatch.setattr(ops, name, self._of(name))

    def _of(self, name):
        def call(*a, **kw):
            self.names.append(name)
            if name == "gemm_fp8":
                assert a[0].dtype == torch.float8_e4m3fn and a[1].shape == (a[0].shape[0], -(-a[0].shape[1] // 128))
                assert a[0].shape[1] == a[2].shape[1]
            if name == "quantize_fp8":
                assert kw["out"].shape == a[0].shape and kw["scale"].shape == (a[0].shape[0], a[0].shape[1] // 128)
            return kw.get("out", a[0])
        return call


@pytest.mark.parametrize("parts", [("wqkv", "wo", "w13", "w2"), ("w13",), ("w2",), ("wqkv", "w2")])
@pytest.mark.parametrize("step", ["prefill", "decode"])
def test_model_walks_its_projections(monkeypatch, parts, step):
    """Each projection gets its inputs in its own type, whichever of a layer's are quantised."""
    cfg = LlamaConfig.tiny(layers=2)
    w = LlamaWeights.random(cfg, "cpu")
    for lw in w.layers:
        for n in parts:
            t = getattr(lw, n)
            setattr(lw, n, Fp8Weight(_f8(*t.shape), torch.ones(t.shape[0] // 128, t.shape[1] // 128)))
    model = LlamaModel(w, PagedKVCache(cfg, 8, "cpu", torch.uint8), max_tokens=16, max_batch=4)
    calls = _Calls(monkeypatch)
    i32 = torch.zeros(3, dtype=torch.int32)
    bt = torch.zeros(3, 2, dtype=torch.int32)
    if step == "prefill":
        model.prefill(i32, i32, i32.long(), [1, 1, 1], i32, torch.zeros(3, 5, dtype=torch.int32), block_tables=bt)
    else:
        model.decode(i32, i32, i32.long(), bt, i32, 16, torch.zeros(1), i32)
    per = {n: calls.names.count(n) for n in set(calls.names)}
    assert per["gemm_fp8"] == 2 * len(parts) and per["gemm"] == 2 * (4 - len(parts)) + 1
    # a norm for each of wqkv and w13 that is bf16, and the last one; the others quantise
    assert per["rmsnorm"] == 2 * (2 - len({"wqkv", "w13"} & set(parts))) + 1
    fused = "w13" in parts and "w2" in parts
    assert per.get("quantize_fp8", 0) == 2 * (len(parts) - (1 if fused else 0))
    assert per["rope_cache_int4"] == 2
    assert per["prefill_attention_paged_int4" if step == "prefill" else "decode_attention_int4"] == 2


def test_prefill_over_a_4_bit_cache_needs_tables():
    cfg = LlamaConfig.tiny(layers=1)
    model = LlamaModel(LlamaWeights.random(cfg, "cpu"), PagedKVCache(cfg, 4, "cpu", torch.uint8), max_tokens=8)
    i32 = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="block_tables"):
        model.prefill(i32, i32, i32.long(), [3], i32, torch.zeros(1, 3, dtype=torch.int32))
    from connex_b200.runtime.pd import KVDestination
    with pytest.raises(ValueError, match="not 4-bit"):
        KVDestination.of_cache(model.cache, torch.zeros(1, dtype=torch.int32))


def test_command_line(monkeypatch):
    from connex_b200.serve.__main__ import kv_blocks, model_args
    from connex_b200.serve.engine import torch_kv_dtype
    ap = argparse.ArgumentParser()
    model_args(ap)
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda *a: (60 << 30, 0))
    cfg = LlamaConfig.llama3_8b()
    blocks = lambda *a: kv_blocks(ap.parse_args(list(a)), cfg, 0, 32)  # noqa: E731
    n16, n4 = blocks(), blocks("--kv-dtype", "int4", "--kv-fraction", "0.5", "--max-batch", "1")
    assert 3.5 < n4 / blocks("--kv-fraction", "0.5") < 3.6 and torch_kv_dtype("int4") == torch.uint8
    # e4m3 projections leave a byte of each weight to the pool
    more = blocks("--weight-dtype", "fp8") - n16
    freed = 32 * (6144 * 4096 + 4096 * 4096 + 3 * 14336 * 4096)
    assert abs(more - int(freed * 0.8) // (2 * 32 * 8 * BS * D * 2)) <= 1
    for bad in (["--kv-dtype", "int8"], ["--weight-dtype", "int4"]):
        with pytest.raises(SystemExit):
            ap.parse_args(bad)


def test_loader_takes_an_fp8_checkpoint(tmp_path):
    """Weights in e4m3 with a scale per 128 x 128 block, fused with their scales; other layouts are refused."""
    from safetensors.torch import load_file, save_file

    from connex_b200.models import hf
    cfg = LlamaConfig.tiny(layers=1)
    w = LlamaWeights.random(cfg, "cpu", seed=3)
    hf.save_llama(w, str(tmp_path / "bf16"))
    config = (tmp_path / "bf16" / "config.json").read_text()
    t = load_file(str(next((tmp_path / "bf16").glob("*.safetensors"))))

    def write(name, tensors):                  # a directory of its own: loaded tensors are maps of their files
        d = tmp_path / name
        d.mkdir()
        (d / "config.json").write_text(config)
        save_file(tensors, str(d / "model.safetensors"), metadata={"format": "pt"})
        return str(d)
    plain = {}
    g = torch.Generator().manual_seed(4)
    for n in [n for n in t if "proj" in n]:
        s = R.fp8_block_scale(t[n], 128).float() * (1 + torch.rand(1, generator=g))
        full = s.repeat_interleave(128, 0).repeat_interleave(128, 1)
        t[n] = (t[n].float() / full).to(torch.float8_e4m3fn)
        t[n + "_scale_inv"] = s
        plain[n] = t[n].float() * full
    fp8 = write("fp8", t)
    got = hf.load_llama(fp8, "cpu").layers[0]
    p = "model.layers.0."
    assert isinstance(got.wqkv, Fp8Weight) and got.attn_norm.dtype == BF
    assert torch.equal(got.wqkv.float(), torch.cat([plain[p + f"self_attn.{n}_proj.weight"] for n in "qkv"]))
    assert torch.equal(got.wo.float(), plain[p + "self_attn.o_proj.weight"])
    assert torch.equal(got.w2.float(), plain[p + "mlp.down_proj.weight"])
    gate, up = ops.deinterleave_gate_up(got.w13.float())
    assert torch.equal(gate, plain[p + "mlp.gate_proj.weight"]) and torch.equal(up, plain[p + "mlp.up_proj.weight"])
    # a tensor-parallel shard: cut from the bf16 values
    half = hf.load_llama(fp8, "cpu", tp=(1, 2)).layers[0]
    assert torch.equal(half.w2, plain[p + "mlp.down_proj.weight"][:, cfg.ffn // 2:].to(BF))
    bad = dict(t)
    bad[p + "mlp.down_proj.weight_scale_inv"] = torch.ones(1, 1)
    with pytest.raises(ValueError, match="128 x 128"):
        hf.load_llama(write("scales", bad), "cpu")
    del bad[p + "mlp.down_proj.weight_scale_inv"]
    with pytest.raises(ValueError, match="without"):
        hf.load_llama(write("none", bad), "cpu")
