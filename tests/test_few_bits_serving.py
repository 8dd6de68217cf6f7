"""What serving makes of the operators in few bits, on the CPU: errors that their kernels record, shards of e4m3
projections, the room that they leave to the cache."""
import argparse

import pytest
import torch

from connex_b200 import ops
from connex_b200.models import hf
from connex_b200.models.llama import Fp8Weight, LayerWeights, LlamaConfig, LlamaWeights
from connex_b200.ops import reference as R


def _stage(monkeypatch, layers=(0, 2)):
    """A stage on the CPU whose steps run no kernels."""
    from connex_b200.runtime.pp import StageRuntime
    monkeypatch.setattr(ops, "decode_workspace_int4", lambda *a: torch.zeros(1))      # sized by the GPU's SMs
    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda t: t)
    rt = StageRuntime(LlamaConfig.tiny(layers=2), *layers, "cpu", num_blocks=16, max_tokens=64, max_batch=4, max_ctx=64,
                      kv_dtype=torch.uint8)
    rt.ran = 0

    def run(inp, *a, **kw):
        rt.ran += 1
        return torch.arange(kw["B"]) if rt.model.is_last else torch.zeros(inp.shape[0], rt.cfg.hidden)
    monkeypatch.setattr(rt.model, "run", run)
    monkeypatch.setattr(ops, "prefill_tile_info", lambda *a, **kw: None)
    return rt


def test_steps_fail_with_what_their_kernels_record(monkeypatch):
    """A stepper raises in the step that went wrong, and serves the next one."""
    from connex_b200.serve.engine import ModelStepper
    rt = _stage(monkeypatch)
    st = object.__new__(ModelStepper)
    st.rt = rt
    assert st.prefill(["a"], [[5, 6, 7]]) == [0]
    run = rt.model.run

    def late(*a, **kw):
        rt.model.status.fill_(1)
        return run(*a, **kw)
    monkeypatch.setattr(rt.model, "run", late)
    for step in (lambda: st.decode(["a"], [[5, 6, 7, 8]]), lambda: st.mixed(["b"], [[5, 6, 7]], [0], [3])):
        with pytest.raises(RuntimeError, match="timeout"):
            step()
    monkeypatch.setattr(rt.model, "run", run)
    assert st.decode(["a"], [[5, 6, 7, 8]]) == [0] and int(rt.model.status) == 0


def test_a_stage_stops_after_a_step_that_went_wrong(monkeypatch):
    """A stage whose rows only go on to the next one raises before its next step, and not for a warm-up."""
    from connex.pp.handover import CX_CTX, REQUEST_IDS
    rt = _stage(monkeypatch, (0, 1))
    td = {"kind": "decode", REQUEST_IDS: ["a"], CX_CTX: [0], "n_new": [1], "ids": torch.tensor([4], dtype=torch.int32)}
    rt.compute(td, [])
    rt.model.status.fill_(2)
    rt.compute({**td, CX_CTX: [1]}, [])
    assert rt.compute({"kind": "warmup", "w": torch.ones(1)}, [])["w"] == 1
    with pytest.raises(RuntimeError, match="bounds"):
        rt.compute({**td, CX_CTX: [2]}, [])
    assert rt.ran == 2 and rt.kv_held("a") == 2
    rt.compute({**td, CX_CTX: [2]}, [])
    assert rt.ran == 3


def _fp8_checkpoint(tmp_path, cfg, keep=lambda name: False):
    """A checkpoint whose projections are e4m3 but for those to ``keep``; (directory, fp32 values by name)."""
    from safetensors.torch import load_file, save_file
    hf.save_llama(LlamaWeights.random(cfg, "cpu", seed=3), str(tmp_path / "bf16"))
    t = load_file(str(next((tmp_path / "bf16").glob("*.safetensors"))))
    plain, g = {}, torch.Generator().manual_seed(4)
    for n in [n for n in t if "proj" in n]:
        plain[n] = t[n].float()
        if not keep(n):
            s = R.fp8_block_scale(t[n], 128).float() * (1 + torch.rand(1, generator=g))
            full = s.repeat_interleave(128, 0).repeat_interleave(128, 1)
            t[n], t[n + "_scale_inv"] = (t[n].float() / full).to(torch.float8_e4m3fn), s
            plain[n] = t[n].float() * full
    (tmp_path / "fp8").mkdir()
    (tmp_path / "fp8" / "config.json").write_text((tmp_path / "bf16" / "config.json").read_text())
    save_file(t, str(tmp_path / "fp8" / "model.safetensors"), metadata={"format": "pt"})
    return str(tmp_path / "fp8"), plain


def _shard_of(plain, cfg, i, rank, world):
    """fp32 values of a rank's projections of layer i, from the checkpoint's."""
    p, n = f"model.layers.{i}.", {}
    rows = lambda x: x.chunk(world, 0)[rank]  # noqa: E731
    n["wqkv"] = torch.cat([rows(plain[p + f"self_attn.{m}_proj.weight"]) for m in "qkv"])
    n["wo"] = plain[p + "self_attn.o_proj.weight"].chunk(world, 1)[rank]
    n["w13"] = ops.interleave_gate_up(rows(plain[p + "mlp.gate_proj.weight"]), rows(plain[p + "mlp.up_proj.weight"]))
    n["w2"] = plain[p + "mlp.down_proj.weight"].chunk(world, 1)[rank]
    return n


@pytest.mark.parametrize("rank", [0, 1])
def test_ranks_keep_an_fp8_checkpoints_codes(tmp_path, monkeypatch, rank):
    """Under tensor parallelism with e4m3 projections, by the loader and by the engine's way to a runtime."""
    from connex_b200.parallel.tp import TPGroup
    from connex_b200.serve.engine import _make_runtime
    monkeypatch.setattr(ops, "decode_workspace_int4", lambda *a: torch.zeros(1))
    cfg = LlamaConfig.tiny(layers=2)
    path, plain = _fp8_checkpoint(tmp_path, cfg)
    got = hf.load_llama(path, "cpu", tp=(rank, 2), fp8=True)
    rt = _make_runtime(cfg, 0, 2, "cpu", 8, 2, 64, 64, path, 0, TPGroup(rank, 2), "int4", "fp8")
    assert got.cfg.ffn == rt.cfg.ffn == cfg.ffn // 2
    for i in range(2):
        for name, want in _shard_of(plain, cfg, i, rank, 2).items():
            for lw in (got.layers[i], rt.weights.layers[i]):
                assert isinstance(getattr(lw, name), Fp8Weight) and torch.equal(getattr(lw, name).float(), want)
    # without the flag: the values in bf16
    half = hf.load_llama(path, "cpu", tp=(rank, 2)).layers[1]
    for name, want in _shard_of(plain, cfg, 1, rank, 2).items():
        assert torch.equal(getattr(half, name), want.to(torch.bfloat16))


def test_shards_of_a_quantised_layer():
    """Four ranks' codes put together are the layer's; uneven heads, one block of the FFN each."""
    from connex_b200.parallel.tp import shard_layer
    cfg = LlamaConfig(vocab_size=64, hidden=384, layers=1, heads=8, kv_heads=4, head_dim=128, ffn=512)
    g = torch.Generator().manual_seed(5)

    def e4m3(n, k):
        return Fp8Weight(torch.randint(0, 100, (n, k), generator=g, dtype=torch.uint8).view(torch.float8_e4m3fn),
                         torch.rand(n // 128, k // 128, generator=g))
    norm = torch.ones(cfg.hidden, dtype=torch.bfloat16)
    lw = LayerWeights(norm, e4m3(16 * 128, 384), e4m3(384, 8 * 128), norm, e4m3(1024, 384), e4m3(384, 512))
    plain = LayerWeights(norm, lw.wqkv.float(), lw.wo.float(), norm, lw.w13.float(), lw.w2.float())
    for rank in range(4):
        a, b = shard_layer(lw, cfg, rank, 4, codes=True), shard_layer(plain, cfg, rank, 4)
        for name in ("wqkv", "wo", "w13", "w2"):
            assert torch.equal(getattr(a, name).float(), getattr(b, name))


def test_room_beside_an_fp8_checkpoint(tmp_path, monkeypatch):
    """The pool is sized by the bytes that the weights will take, whichever of them the checkpoint holds in e4m3."""
    from connex_b200.serve.__main__ import kv_blocks, model_args
    cfg = LlamaConfig.tiny(layers=2)
    path, plain = _fp8_checkpoint(tmp_path, cfg, keep=lambda n: "layers.1.mlp.down" in n or "layers.0.self_attn.v" in n)
    ap = argparse.ArgumentParser()
    model_args(ap)
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda *a: ((2 << 30) + (64 << 20), 0))

    def blocks(*a):
        return kv_blocks(ap.parse_args(["--kv-fraction", "1.0", "--max-ctx", "64", *a]), cfg, 0, 2)
    weights = hf.load_llama(path, "cpu")
    freed = sum(t.q.numel() for lw in weights.layers for t in lw.__dict__.values() if isinstance(t, Fp8Weight))
    assert 0 < freed == hf.fp8_elements(path, (0, 2)) < sum(x.numel() for x in plain.values())
    assert hf.fp8_elements(str(tmp_path / "bf16"), (0, 2)) == 0
    block = 2 * 2 * cfg.kv_heads * cfg.block_size * cfg.head_dim * 2
    none = blocks("--checkpoint", str(tmp_path / "bf16"))
    assert none == blocks() and abs(blocks("--checkpoint", path) - none - freed / block) <= 1
    # the flag makes e4m3 of all of them; a tensor-parallel rank without it holds bf16
    assert blocks("--checkpoint", path, "--weight-dtype", "fp8") > blocks("--checkpoint", path)
    assert blocks("--checkpoint", path, "--tp", "2") == none


def test_unknown_types_are_refused():
    """A type that is none is an error, and not bf16."""
    from connex_b200.serve.engine import _make_runtime
    args = (LlamaConfig.tiny(), 0, 1, "cpu", 8, 2, 64, 64, None, 0, None)
    for kv, weight, match in (("int4", "e4m3", "weight type 'e4m3'"), ("bf16", "fp4", "weight type 'fp4'"),
                              ("int8", "bf16", "KV cache type")):
        with pytest.raises(ValueError, match=match):
            _make_runtime(*args, kv, weight)
