"""The 8-bit KV cache and the block operations on the CPU: the quantising
append's plain statement against its definition, shared blocks (fork, free,
compaction) of both cache types, and the refusals of the operators' entry
points -- argument checks come before the device check, so they run here."""
import argparse
import math
import random

import pytest
import torch

from connex_b200 import ops
from connex_b200.models.llama import LlamaConfig, PagedKVCache
from connex_b200.ops import reference as R

BS, D = 16, 128


def _cache(dtype, blocks=24, layers=2):
    cfg = LlamaConfig.tiny(layers=layers)
    c = PagedKVCache(cfg, blocks, "cpu", dtype)
    g = torch.Generator().manual_seed(1)
    raw = torch.randint(0, 120, c.kv.shape, generator=g, dtype=torch.uint8)
    if dtype == torch.float8_e4m3fn:
        c.kv.copy_(raw.view(torch.float8_e4m3fn))
        c.scales.copy_(torch.rand(c.scales.shape, generator=g))
    else:
        c.kv.copy_(raw.float())
    return c


def _rows(c, table, n):
    """What a sequence reads: values (and scales) of its first n tokens, layer by layer."""
    bs = c.cfg.block_size
    out = []
    for i in range(n):
        b, o = table[i // bs], i % bs
        v = c.kv[:, :, b, :, o].float()
        out.append(v if c.scales is None else v * c.scales[:, :, b][..., None])
    return torch.stack(out) if out else torch.zeros(0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("n", [0, 1, 15, 16, 17, 48, 50])
def test_fork_shares_full_blocks_and_copies_the_tail(dtype, n):
    c = _cache(dtype)
    t = c.allocate(4)
    before = _rows(c, t, n)
    free = c.free_blocks
    a, b = c.fork(t, n, 2)
    full = n // BS
    assert a[:full] == b[:full] == t[:full]
    assert len(a) == len(b) == c.blocks_needed(n)
    assert free - c.free_blocks == (2 if n % BS else 0)
    if n % BS:
        assert len({t[full], a[-1], b[-1]}) == 3
    assert torch.equal(_rows(c, a, n), before) and torch.equal(_rows(c, b, n), before)
    # the child writes on in its own block only
    if n % BS:
        c.kv.view(torch.uint8 if dtype == torch.float8_e4m3fn else torch.bfloat16)[:, :, a[-1], :, n % BS:] = 0
        assert torch.equal(_rows(c, t, n), before) and torch.equal(_rows(c, b, n), before)
    for x in (a, t, b):
        c.free(x)
    assert c.free_blocks == 24 and sorted(c._free) == list(range(24)) and not c._shared


def test_free_without_sharing_keeps_its_order():
    c = _cache(torch.bfloat16)
    a, b = c.allocate(3), c.allocate(2)
    c.free(a)
    assert c.allocate(3) == a
    c.free(b)
    assert c.allocate(1) == b[:1]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_compact_keeps_what_sequences_read(dtype):
    rng = random.Random(3)
    for _ in range(20):
        c = _cache(dtype)
        tables, lens = [], []
        pin = c.allocate(1)                          # in no table: stays where it is
        for _ in range(6):
            n = rng.randint(1, 45)
            if c.blocks_needed(n) > c.free_blocks:
                break
            tables.append(c.allocate(c.blocks_needed(n)))
            lens.append(n)
        k = rng.randrange(len(tables))
        need = 1 if lens[k] % BS else 0
        if c.free_blocks >= need:
            tables += c.fork(tables[k], lens[k])
            lens.append(lens[k])
        for _ in range(rng.randint(0, 2)):
            i = rng.randrange(len(tables))
            c.free(tables.pop(i))
            lens.pop(i)
        before = [_rows(c, t, n) for t, n in zip(tables, lens)]
        pinned = c.kv[:, :, pin[0]].clone()
        free = c.free_blocks
        moved = c.compact(tables)
        assert c.free_blocks == free
        used = {b for t in tables for b in t} | set(pin)
        assert used == set(range(len(used))) and sorted(c._free) == list(range(len(used), 24))
        for t, n, x in zip(tables, lens, before):
            assert torch.equal(_rows(c, t, n), x)
        assert torch.equal(c.kv[:, :, pin[0]].view(torch.uint8), pinned.view(torch.uint8))
        assert c.compact(tables) == 0 or moved == 0
        for t in tables:
            c.free(t)
        c.free(pin)
        assert sorted(c._free) == list(range(24)) and not c._shared


def test_cache_refusals():
    c = _cache(torch.bfloat16)
    t = c.allocate(2)
    for n in (-1, 33):
        with pytest.raises(ValueError, match="fork"):
            c.fork(t, n)
    with pytest.raises(ValueError, match="fork"):
        c.fork(t, 5, -1)
    c.allocate(21)
    free = c.free_blocks
    with pytest.raises(ValueError, match="block ids"):
        c.fork([t[0], 24], 20, 1)
    with pytest.raises(ValueError, match="block ids"):
        c.fork([-1, t[0]], 20, 1)
    assert c.free_blocks == free
    shared = dict(c._shared)
    with pytest.raises(MemoryError):
        c.fork(t, 20, 2)
    assert c._shared == shared and c.free_blocks == 1       # a failed fork leaves nothing behind
    for pairs in ([(0, 1), (1, 2)], [(0, 3), (1, 3)], [(2, 2)], [(0, 24)], [(-1, 2)]):
        with pytest.raises(ValueError, match="copy_blocks"):
            c.copy_blocks(pairs)
    c.copy_blocks([])


def test_append_statement_follows_the_definition():
    """Scale: smallest power of two with amax <= 448 s; rows within half a step; old rows keep their values."""
    g = torch.Generator().manual_seed(5)
    for trial in range(40):
        cache = (torch.randn(3, 2, BS, D, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
        scale = torch.exp2(torch.randint(-6, 0, (3, 2), generator=g).float())
        was, old = R.fp8_values(cache, scale), scale.clone()
        n = int(torch.randint(1, 20, (1,), generator=g))
        slots = torch.randint(-1, 3 * BS, (n,), generator=g)
        rows = (torch.randn(n, 2, D, generator=g) * 10.0 ** float(torch.randint(-3, 4, (1,), generator=g))).to(torch.bfloat16)
        R.fp8_append(cache, scale, rows, slots)
        now = R.fp8_values(cache, scale)
        last = {int(s): t for t, s in enumerate(slots.tolist()) if s >= 0}
        for b in range(3):
            mine = {s % BS: t for s, t in last.items() if s // BS == b}
            top = torch.stack([rows[t].double().abs().amax(-1) for t in mine.values()]).amax(0) if mine else None
            for h in range(2):
                s = float(scale[b, h])
                if not mine:
                    assert s == float(old[b, h]) and torch.equal(now[b, h], was[b, h])
                    continue
                floor = 0.0 if 0 in mine else float(old[b, h])
                assert float(top[h]) <= 448 * s and s >= floor
                assert s == floor or float(top[h]) > 224 * s
                for r in range(BS):
                    if r in mine:
                        x = rows[mine[r], h].double()
                        assert ((now[b, h, r] - x).abs() <= (x.abs() * 2.0 ** -4).clamp(min=2.0 ** -10 * s)).all()
                    elif 0 not in mine:
                        assert ((now[b, h, r] - was[b, h, r]).abs() <= 2.0 ** -10 * s).all()


def _args(hq=4, hkv=2, T=3, nb=5, B=2):
    f8 = torch.float8_e4m3fn
    return dict(qkv=torch.zeros(T, (hq + 2 * hkv) * D, dtype=torch.bfloat16), pos=torch.zeros(T, dtype=torch.int32),
                cs=torch.zeros(64, D), slots=torch.zeros(T, dtype=torch.int64),
                k=torch.zeros(nb, hkv, BS, D).to(f8), v=torch.zeros(nb, hkv, BS, D).to(f8), ks=torch.ones(nb, hkv),
                vs=torch.ones(nb, hkv), q=torch.zeros(B, hq * D, dtype=torch.bfloat16),
                bt=torch.zeros(B, 4, dtype=torch.int32), lens=torch.ones(B, dtype=torch.int32),
                ws=torch.zeros(10, 2 * 132), ti=torch.zeros(1, 5, dtype=torch.int32))


def _write(a, hq=4, hkv=2, **kw):
    return ops.rope_cache_fp8(a["qkv"], a["pos"], a["cs"], hq, hkv, a["slots"], a["k"], a["v"], a["ks"], a["vs"], **kw)


def _decode(a, hq=4, **kw):
    return ops.decode_attention_fp8(a["q"], a["k"], a["v"], a["ks"], a["vs"], a["bt"], a["lens"], hq, a["ws"], **kw)


def _prefill(a, hq=4, hkv=2, **kw):
    return ops.prefill_attention_paged_fp8(a["q"], a["k"], a["v"], a["ks"], a["vs"], a["bt"], a["ti"], hq, hkv, **kw)


@pytest.mark.parametrize("call,change,match", [
    (_write, {"qkv": lambda t: t.float()}, "bf16"),
    (_write, {"qkv": lambda t: t[:, 8:]}, "heads of 128"),
    (_write, {"qkv": lambda t: torch.zeros(3, 8 * D + 4, dtype=torch.bfloat16)[:, 4:]}, "16-byte"),
    (_write, {"qkv": lambda t: t[:, :1].expand(3, 8 * D)}, "contiguous rows|16-byte"),
    (_write, {"pos": lambda t: t.long()}, "positions"),
    (_write, {"pos": lambda t: t[:2]}, "positions"),
    (_write, {"slots": lambda t: t.int()}, "slot_mapping"),
    (_write, {"slots": lambda t: torch.zeros(4, dtype=torch.int64)}, "slot_mapping"),
    (_write, {"cs": lambda t: t.double()}, "cos_sin"),
    (_write, {"cs": lambda t: t[:, :64]}, "cos_sin"),
    (_write, {"k": lambda t: t.view(torch.uint8)}, "float8_e4m3fn"),
    (_write, {"v": lambda t: t[:4]}, "float8_e4m3fn"),
    (_write, {"k": lambda t: t[:, :1], "v": lambda t: t[:, :1]}, "float8_e4m3fn"),
    (_write, {"ks": lambda t: t.double()}, "scales"),
    (_write, {"vs": lambda t: t[:4]}, "scales"),
    (_write, {}, "must be a CUDA tensor"),
    (_decode, {"q": lambda t: t.half()}, "bf16"),
    (_decode, {"q": lambda t: t[:, :256]}, "Hq heads"),
    (_decode, {"bt": lambda t: t.long()}, "block_tables"),
    (_decode, {"bt": lambda t: t[:1]}, "block_tables"),
    (_decode, {"bt": lambda t: torch.zeros(2, 8, dtype=torch.int32)[:, ::2]}, "block_tables"),
    (_decode, {"lens": lambda t: t.long()}, "ctx_lens"),
    (_decode, {"lens": lambda t: t[:1]}, "ctx_lens"),
    (_decode, {"vs": lambda t: t.t().contiguous()}, "scales"),
    (_decode, {}, "must be a CUDA tensor"),
    (_prefill, {"q": lambda t: t.float()}, "bf16"),
    (_prefill, {"q": lambda t: t[:, :256]}, "Hq heads"),
    (_prefill, {"ti": lambda t: t[:, :3]}, "tile_info"),
    (_prefill, {"ti": lambda t: t.long()}, "tile_info"),
    (_prefill, {"bt": lambda t: t.long()}, "block_tables"),
    (_prefill, {"k": lambda t: t.view(torch.uint8)}, "float8_e4m3fn"),
    (_prefill, {"ks": lambda t: t.double()}, "scales"),
    (_prefill, {}, "must be a CUDA tensor"),
])
def test_refusals(call, change, match):
    a = _args()
    a.update({n: f(a[n]) for n, f in change.items()})
    with pytest.raises(RuntimeError, match=match):
        call(a)


def test_more_refusals():
    a = _args()
    with pytest.raises(RuntimeError, match="q/k norm"):
        _write(a, q_norm=torch.ones(64, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="overlaps"):
        _write(a, out=a["qkv"][:, D:5 * D])
    with pytest.raises(RuntimeError, match="out must be"):
        _write(a, out=a["qkv"][:, :3 * D])
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        _write(a, out=a["qkv"][:, :4 * D])                          # in place is allowed
    with pytest.raises(RuntimeError, match="multiple of the KV heads"):
        _decode(a, hq=3)
    with pytest.raises(RuntimeError, match="16 of them"):
        _decode({**_args(hq=34), "q": torch.zeros(2, 34 * D, dtype=torch.bfloat16)}, hq=34)
    with pytest.raises(ValueError, match="multiple of the KV heads"):
        ops.decode_workspace_fp8(4, 10, 4, "cuda:0")
    with pytest.raises(ValueError, match="16 query heads"):
        ops.decode_workspace_fp8(4, 34, 2, "cuda:0")
    kv = torch.zeros(2, 2, 5, 2, BS, D, dtype=torch.bfloat16)
    pairs = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.kv_copy_blocks(kv[:, :, ::2], pairs)
    with pytest.raises(RuntimeError, match="pairs"):
        ops.kv_copy_blocks(kv, pairs.long())
    with pytest.raises(RuntimeError, match="with its scales"):
        ops.kv_copy_blocks(kv.to(torch.float8_e4m3fn), pairs)
    with pytest.raises(RuntimeError, match="scales"):
        ops.kv_copy_blocks(kv.to(torch.float8_e4m3fn), pairs, torch.ones(2, 2, 5, 3))
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        ops.kv_copy_blocks(kv, pairs)
    # a status word of another device would be a bad address for the kernel
    elsewhere = torch.zeros(1, dtype=torch.int32, device="meta")
    for call in (_write, _decode, _prefill):
        with pytest.raises(RuntimeError, match="every tensor must be on"):
            call(a, status=elsewhere)
    with pytest.raises(RuntimeError, match="every tensor must be on"):
        ops.kv_copy_blocks(kv, pairs, status=elsewhere)


def test_layerwise_transfer_refuses_an_8_bit_cache():
    from connex_b200.runtime.pd import KVDestination
    c = _cache(torch.float8_e4m3fn)
    with pytest.raises(ValueError, match="scales do not travel"):
        KVDestination.of_cache(c, torch.zeros(1, dtype=torch.int32))
    KVDestination.of_cache(_cache(torch.bfloat16), torch.zeros(1, dtype=torch.int32))


def test_cli_kv_dtype(monkeypatch):
    from connex_b200.serve.__main__ import kv_blocks, model_args
    from connex_b200.serve.engine import torch_kv_dtype
    ap = argparse.ArgumentParser()
    model_args(ap)
    cfg = LlamaConfig.tiny()
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda *a: (60 << 30, 0))
    n16, n8 = (kv_blocks(ap.parse_args(["--kv-dtype", d]), cfg, 0, 2) for d in ("bf16", "fp8"))
    assert 1.99 < n8 / n16 <= 2.0
    assert torch_kv_dtype("fp8") == torch.float8_e4m3fn and torch_kv_dtype("bf16") == torch.bfloat16
    with pytest.raises(ValueError, match="bf16 or fp8"):
        torch_kv_dtype("int8")
    with pytest.raises(SystemExit):
        ap.parse_args(["--kv-dtype", "int8"])


@pytest.mark.parametrize("given", [None, "fp8"])
def test_stepper_from_the_command_line(monkeypatch, given):
    """``--kv-dtype`` reaches the runtime; callers with options of their own that do not name it get bf16."""
    from connex_b200.serve import __main__ as m, engine
    ap = argparse.ArgumentParser()
    m.model_args(ap)
    a = ap.parse_args([] if given is None else ["--kv-dtype", given])
    if given is None:
        del a.kv_dtype
    for k, v in dict(num_stages=1, num_blocks=64, device="cpu", no_graphs=True).items():
        setattr(a, k, v)
    seen = {}
    monkeypatch.setattr(torch.cuda, "set_device", lambda d: None)
    monkeypatch.setattr(engine, "ModelStepper", lambda *x, **kw: seen.update(kw))
    m.build_stepper(a)
    assert seen["kv_dtype"] == (given or "bf16")


@pytest.mark.parametrize("scale", [0.0, -0.1, math.inf, math.nan])
def test_prefill_scale(scale):
    with pytest.raises(RuntimeError, match="scale must be positive"):
        _prefill(_args(), scale=scale)


def test_refusals_that_name_a_number():
    """Messages with numbers in them are exceptions like the others."""
    a = _args(B=5000)
    with pytest.raises(RuntimeError, match="at most 4096 sequences"):
        _decode(a)
    a = _args(B=9000)
    with pytest.raises(RuntimeError, match="B up to 8192"):
        _prefill(a)
    jobs = torch.zeros(1, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="jobs_dev must be contiguous"):
        ops._C.wsync(jobs, jobs, 0, [], [], 0, 0, 0, 0)


@pytest.mark.parametrize("shape", [(1, 2, 4, 0, BS, D), (1, 2, 4, 2, 0, D), (1, 2, 4, 2, BS, 0)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_copy_of_blocks_without_bytes_is_refused(shape, dtype):
    """A block without bytes has no vectors for the kernel to walk."""
    kv = torch.empty(shape, dtype=dtype)
    scales = torch.ones(shape[:4]) if dtype == torch.float8_e4m3fn else None
    with pytest.raises(RuntimeError, match="multiples of 16 bytes"):
        ops.kv_copy_blocks(kv, torch.tensor([[0, 1]], dtype=torch.int32), scales)


def test_copy_of_more_pairs_than_an_index_counts_is_refused():
    """The kernel finds pair i at words 2 i and 2 i + 1, counted in 32 bits."""
    kv = torch.empty(1, 2, 4, 2, BS, D, dtype=torch.bfloat16, device="meta")
    pairs = torch.empty(2 ** 30, 2, dtype=torch.int32, device="meta")
    with pytest.raises(RuntimeError, match="too many"):
        ops.kv_copy_blocks(kv, pairs)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        ops.kv_copy_blocks(kv, pairs[:2 ** 30 - 1])


@pytest.mark.parametrize("k,v", [
    (torch.float8_e4m3fn, torch.float8_e4m3fn), (torch.bfloat16, torch.float8_e4m3fn),
    (torch.float8_e4m3fn, torch.bfloat16), (torch.uint8, torch.uint8)])
def test_bf16_write_refuses_a_cache_of_another_type(k, v):
    """It stores two bytes per element: past the end of an 8-bit cache."""
    a = _args()
    with pytest.raises(RuntimeError, match="rope_cache: caches must be"):
        ops.rope_cache(a["qkv"], a["pos"], a["cs"], 4, 2, a["slots"], torch.zeros(5, 2, BS, D).to(k),
                       torch.zeros(5, 2, BS, D).to(v))


@pytest.mark.parametrize("k,v", [
    ((5, 1, BS, D), (5, 1, BS, D)), ((5, 2, BS, D), (4, 2, BS, D)), ((5, 2, BS, 64), (5, 2, BS, 64)),
    ((10, BS, D), (10, BS, D)), ((5, 2, 0, D), (5, 2, 0, D))])
def test_bf16_write_refuses_a_cache_of_another_shape(k, v):
    a = _args()
    k, v = torch.zeros(k, dtype=torch.bfloat16), torch.zeros(v, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="rope_cache: caches must be"):
        ops.rope_cache(a["qkv"], a["pos"], a["cs"], 4, 2, a["slots"], k, v)
    whole = torch.zeros(5, 4, BS, D, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="rope_cache: caches must be"):
        ops.rope_cache(a["qkv"], a["pos"], a["cs"], 4, 2, a["slots"], whole[:, ::2], whole[:, ::2])
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        ops.rope_cache(a["qkv"], a["pos"], a["cs"], 4, 4, a["slots"], whole, whole.clone())


def test_bf16_decode_refuses_values_in_8_bits():
    """Both caches are read at two bytes per element."""
    a = _args()
    k, ws = torch.zeros(5, 2, BS, D, dtype=torch.bfloat16), torch.zeros(1 << 16)
    with pytest.raises(RuntimeError, match="vc must be bf16"):
        ops.decode_attention(a["q"], k, a["v"], a["bt"], a["lens"], 4, 64, ws)


def _runtime(monkeypatch, dtype, layers=(0, 2), blocks=32):
    """A stage of the model on the CPU: its bookkeeping runs here, its kernels do not."""
    from connex_b200.runtime.pp import StageRuntime
    monkeypatch.setattr(ops, "decode_workspace_fp8", lambda *a: torch.zeros(1))       # sized by the GPU's SMs
    return StageRuntime(LlamaConfig.tiny(layers=2), *layers, "cpu", num_blocks=blocks, max_tokens=64, max_batch=8,
                        max_ctx=128, kv_dtype=dtype)


def test_stage_refuses_a_prefill_that_does_not_read_the_8_bit_cache(monkeypatch):
    """The 8-bit write leaves the fused rows' keys unrotated, so attention over those rows would be wrong."""
    model = _runtime(monkeypatch, torch.float8_e4m3fn).model
    ids = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="8-bit cache"):
        model.run(ids, ids, ids.long(), prefill=True, tile_info=torch.tensor([[0, 3, 0]], dtype=torch.int32), B=1)


def _hold(rt, rid, n, value):
    """What a step leaves behind: blocks, held tokens and, with the log on, the step's rows."""
    rt._blocks_for(rid, n)
    if rt.act is not None:
        rt._log([rid], [0], [n], torch.full((n, rt.cfg.hidden), float(value), dtype=torch.bfloat16))
    rt.held[rid] = n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_fork_gives_every_request_a_log_of_its_own(monkeypatch, dtype):
    """A request that was released and comes back by a fork, then a new one: each replays its own rows."""
    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda t: t)
    rt = _runtime(monkeypatch, dtype, (0, 1))
    rt.enable_activation_log(6)
    _hold(rt, "a", 20, 1)
    _hold(rt, "b", 5, 2)
    rt.release(["b"])
    rt.fork("a", ["b", "c"])
    _hold(rt, "d", 7, 4)
    rt.fork("d", ["e"])
    assert len(set(rt.act_slot.values())) == len(rt.act_slot)
    for rid, n, value in (("a", 20, 1), ("b", 20, 1), ("c", 20, 1), ("d", 7, 4), ("e", 7, 4)):
        x, lens = rt.replay([rid])
        assert lens == [n] and (x == value).all(), rid


def test_fork_with_a_log_refuses_before_it_changes_anything(monkeypatch):
    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda t: t)
    rt = _runtime(monkeypatch, torch.bfloat16, (0, 1))
    _hold(rt, "early", 20, 0)                        # before the log was kept
    rt.enable_activation_log(3)
    _hold(rt, "a", 20, 1)
    _hold(rt, "gone", 4, 2)
    rt.release(["gone"])

    def state():
        return (dict(rt.held), {r: list(t) for r, t in rt.tables.items()}, dict(rt.act_slot), dict(rt.cache._shared),
                list(rt.cache._free))
    before = state()
    with pytest.raises(ValueError, match="activation log"):
        rt.fork("early", ["x"])
    with pytest.raises(MemoryError, match="activation log full"):
        rt.fork("a", ["x", "y"])
    assert state() == before
    rt.fork("a", ["x", "gone"])                      # "gone" has its slot already
    assert (rt.replay(["gone"])[0] == 1).all() and (rt.replay(["x"])[0] == 1).all()
    with pytest.raises(MemoryError, match="activation log full"):
        _hold(rt, "z", 3, 3)
    assert "z" not in rt.act_slot


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_compact_leaves_blocks_of_owners_it_was_not_given(dtype):
    """A shared block moves only when every table that names it is changed with it."""
    c = _cache(dtype)
    low = c.allocate(3)
    parent = c.allocate(3)
    child, = c.fork(parent, 2 * BS + 5)
    c.free(low)
    want = [_rows(c, t, 2 * BS + 5) for t in (parent, child)]
    assert c.compact([child]) == 1                    # its own last block; the shared ones have another owner
    assert child[:2] == parent[:2] == [3, 4] and child[2] < 3
    for t, x in zip((parent, child), want):
        assert torch.equal(_rows(c, t, 2 * BS + 5), x)
    assert c.compact([child, child]) == 0             # one owner named twice is still one
    assert c.compact([child, parent]) == 2
    assert set(child) | set(parent) == set(range(4))
    for t, x in zip((parent, child), want):
        assert torch.equal(_rows(c, t, 2 * BS + 5), x)
    c.free(parent)
    c.free(child)
    assert sorted(c._free) == list(range(24)) and not c._shared


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("start,stop", [(0, 1), (5, 6), (16, 17), (20, 40), (47, 50), (0, 64), (48, 49)])
def test_a_step_behind_a_fork_writes_blocks_of_its_own(monkeypatch, dtype, start, stop):
    """A request that goes on from before the end of its shared blocks leaves the other owners' rows alone."""
    rt = _runtime(monkeypatch, dtype)
    c = rt.cache
    raw = torch.randint(0, 120, c.kv.shape, generator=torch.Generator().manual_seed(7), dtype=torch.uint8)
    c.kv.copy_(raw.view(torch.float8_e4m3fn) if c.scales is not None else raw.float())
    _hold(rt, "a", 50, 0)
    before = _rows(c, rt.tables["a"], 50)
    rt.fork("a", ["x", "y"])
    t = rt._blocks_for("x", stop, start)
    assert torch.equal(_rows(c, t, start).flatten(), before[:start].flatten())
    for p in range(start, stop):                      # the step's writes
        c.kv.view(torch.uint8 if c.scales is not None else torch.bfloat16)[:, :, t[p // BS], :, p % BS] = 1
        if c.scales is not None:
            c.scales[:, :, t[p // BS]] *= 4
    for r in ("a", "y"):
        assert torch.equal(_rows(c, rt.tables[r], 50), before)
    rt.release(["a", "x", "y"])
    assert sorted(c._free) == list(range(32)) and not c._shared


def test_blocks_of_ones_own_need_room():
    c = _cache(torch.bfloat16)
    t = c.allocate(4)
    x, = c.fork(t, 64)
    c.allocate(19)
    held = list(x), dict(c._shared)
    with pytest.raises(MemoryError):
        c.own(x, 20, 40)
    assert (x, c._shared) == held and c.free_blocks == 1
    c.own(x, 64, 70)                                  # behind the shared blocks: nothing to do
    assert (x, c._shared) == held


@pytest.mark.parametrize("fraction", [0.8, 0.95, 1.0])
@pytest.mark.parametrize("layers", [1, 2, 8, 32])
@pytest.mark.parametrize("batch,ctx,step", [(64, 4096, 8192), (8, 130000, 8192), (256, 8192, 16), (1, 128, 128)])
def test_pool_leaves_room_for_a_prefill_steps_blocks(monkeypatch, fraction, layers, batch, ctx, step):
    """A prompt step holds the blocks that it reads as bf16, a layer at a time, beside the pool."""
    from connex_b200.serve.__main__ import kv_blocks, model_args
    ap = argparse.ArgumentParser()
    model_args(ap)
    cfg, free = LlamaConfig(max_pos=131072), 60 << 30
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda *a: (free, 0))

    def blocks(dtype):
        return kv_blocks(ap.parse_args(["--kv-dtype", dtype, "--kv-fraction", str(fraction), "--max-batch", str(batch),
                                        "--max-ctx", str(ctx), "--max-step-tokens", str(step)]), cfg, 0, layers)
    weights = 2 * (layers * (6144 * 4096 + 4096 * 4096 + 3 * 14336 * 4096) + 2 * 128256 * 4096)
    room = free - weights - (2 << 30)
    n, block = blocks("fp8"), 2 * layers * 8 * (BS * D + 4)
    read = min(n, min(batch, step) * -(-ctx // BS))                  # of a step, at most
    copy = 2 * 8 * BS * D * 2
    assert n * block + read * copy <= room
    more = n + 1                                                     # one block more would not fit, or pass the share
    assert more * block > room * fraction or more * block + min(more, min(batch, step) * -(-ctx // BS)) * copy > room
    assert blocks("bf16") == int(room * fraction) // (2 * layers * 8 * BS * D * 2)


@pytest.mark.parametrize("n_blocks", [None, 7])
def test_model_prefill_hands_on_the_blocks_it_reads(monkeypatch, n_blocks):
    """Without the number the workspace is the tables' whole rectangle."""
    from connex_b200.models.llama import LlamaModel, LlamaWeights
    cfg = LlamaConfig.tiny(layers=1)
    model = LlamaModel(LlamaWeights.random(cfg, "cpu"), PagedKVCache(cfg, 24, "cpu", torch.float8_e4m3fn), 64, 4)
    for name in ("embedding", "rmsnorm", "gemm"):
        monkeypatch.setattr(ops, name, lambda *a, **kw: None)
    for name in ("_layer_tail", "_head"):
        monkeypatch.setattr(model, name, lambda *a: None)
    monkeypatch.setattr(model, "_rotate_and_cache", lambda i, qkv, *a: qkv)
    seen = []
    monkeypatch.setattr(ops, "prefill_attention_paged_fp8", lambda *a, **kw: seen.append(kw["n_blocks"]))
    ids = torch.zeros(40, dtype=torch.int32)
    kw = {} if n_blocks is None else {"n_blocks": n_blocks}
    model.prefill(ids, ids, ids.long(), [8, 32], ids[:2], torch.zeros(2, 5, dtype=torch.int32),
                  block_tables=torch.zeros(2, 20, dtype=torch.int32), **kw)
    assert seen == [n_blocks]


@pytest.mark.parametrize("heads,fit", [(1, 4), (4, 4), (8, 4), (9, 3), (10, 3), (16, 3)])
def test_decode_plans_for_the_ctas_that_an_sm_holds(heads, fit):
    """Query heads per KV head past 8 take three CTAs' registers, and the lengths of some 1400 sequences
    the fourth one's shared memory (228 KB of an SM, one of them the system's for each CTA)."""
    per_sm = [ops._C.decode_fp8_resident(B, heads) for B in (1, 64, 1300, 1500, 4096)]
    assert per_sm == [fit, fit, fit, 3, 3]


def test_every_stage_takes_the_cache_type_from_the_command_line(monkeypatch):
    """``--kv-dtype`` of a later pipeline stage reaches its runtime and its pool's size."""
    from connex_b200.models import hf  # noqa: F401
    from connex_b200.runtime import pp
    from connex_b200.serve import __main__ as m, stage
    ap = argparse.ArgumentParser()
    m.model_args(ap)
    seen = {}

    class Stop(Exception):
        pass

    def runtime(cfg, l0, l1, dev, **kw):
        seen.update(kw, layers=(l0, l1))
        raise Stop
    monkeypatch.setattr(torch.cuda, "set_device", lambda d: None)
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda *a: (60 << 30, 0))
    monkeypatch.setattr(pp, "StageRuntime", runtime)
    blocks = {}
    for given, dtype in (("bf16", torch.bfloat16), ("fp8", torch.float8_e4m3fn)):
        a = ap.parse_args(["--num-stages", "2", "--kv-dtype", given])
        a.stage, a.rule = 1, False
        with pytest.raises(Stop):
            stage.run_stage(a, None)
        assert seen["kv_dtype"] == dtype and seen["layers"] == (16, 32)
        blocks[given] = seen["num_blocks"]
    assert 1.99 < blocks["fp8"] / blocks["bf16"] <= 2.0
