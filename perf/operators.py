"""Cases and plain forms of the 8-bit paged KV cache operators.

The cache holds e4m3 values in 16-token blocks ``[blocks, Hkv, 16, 128]`` with
one power-of-two fp32 scale per (block, KV head) for K and one for V.  Four
operators work on it, as a serving step uses them layer by layer:

* ``write``    rotate q and k, quantise k and v into their cache slots, raising
               a block's scale (and requantising its rows) when a token needs it
* ``decode``   attention of one new token per sequence over its cached tokens
* ``prefill``  causal attention of prompt chunks that continue cached sequences
* ``copy``     move whole blocks of every layer (fork, compaction), for the
               8-bit cache with its scales and for the bf16 cache

``own`` false: elementary torch operations in fp32.  ``own`` true: the calls of
``connex_b200.ops``.
"""
import math
import random

import torch

own = False

BS, D = 16, 128          # tokens of a cache block, head size
MIN_EXP = -100           # exponent of the smallest block scale
THETA = 500000.0


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one serving step of 64 generating requests: a launch-bound call per layer
        dict(name="write-decode", op="write", hq=32, hkv=8, seqs=64, new=1, ctx=4096, norm=False, mix=11),
        # a full prefill step: four 2048-token prompts
        dict(name="write-prefill", op="write", hq=32, hkv=8, seqs=4, new=2048, ctx=0, norm=False, mix=12),
        # a mixed step of ragged chunks that begin inside a block, with per-head q/k norms
        dict(name="write-chunks", op="write", hq=32, hkv=4, seqs=5, new=613, ctx=1777, norm=True, mix=13),
        # one request alone: latency
        dict(name="decode-single", op="decode", hq=32, hkv=8, batch=1, ctx=500, even=True, mix=21),
        # a full decode batch at the flagship's context
        dict(name="decode-batch", op="decode", hq=32, hkv=8, batch=64, ctx=4096, even=True, mix=22),
        # requests of very different ages, eight query heads per KV head
        dict(name="decode-ragged", op="decode", hq=32, hkv=4, batch=96, ctx=8191, even=False, mix=23),
        # long documents at the 128k positions of the long-context configuration
        dict(name="decode-long", op="decode", hq=32, hkv=8, batch=2, ctx=131072, even=True, mix=24),
        # the tails of several prompts: short ragged chunks over medium contexts
        dict(name="prefill-short", op="prefill", hq=32, hkv=8, seqs=5, new=131, ctx=2000, even=False, mix=31),
        # one chunk of a long prompt in the middle of its reading
        dict(name="prefill-chunk", op="prefill", hq=32, hkv=8, seqs=1, new=2048, ctx=6144, even=True, mix=32),
        # the last chunk of a 32k prompt
        dict(name="prefill-long", op="prefill", hq=32, hkv=4, seqs=1, new=2048, ctx=30720, even=True, mix=33),
        # sixteen sequences forked: their partly filled last blocks copied in all layers of a bf16 cache
        dict(name="copy-fork", op="copy", hkv=8, layers=32, blocks=256, pairs=16, fp8=False, mix=41),
        # compaction of a fragmented 8-bit pool
        dict(name="copy-compact", op="copy", hkv=8, layers=32, blocks=1024, pairs=400, fp8=True, mix=42),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["write", "decode", "prefill", "copy"])
    mix = rng.randrange(1, 1 << 30)
    hq, hkv = rng.choice([(32, 8), (32, 4), (8, 2), (28, 4), (16, 1), (6, 2), (4, 4), (5, 1)])
    if op == "write":
        if rng.random() < 0.5:
            return dict(op=op, hq=hq, hkv=hkv, seqs=_log(rng, 1, 256), new=1, ctx=_log(rng, 1, 8192),
                        norm=rng.random() < 0.3, mix=mix)
        new = _log(rng, 2, 2048)
        return dict(op=op, hq=hq, hkv=hkv, seqs=rng.randint(1, max(1, min(8, 8192 // new))), new=new,
                    ctx=rng.choice([0, _log(rng, 1, 4096)]), norm=rng.random() < 0.3, mix=mix)
    if op == "decode":
        ctx = _log(rng, 1, 131072)
        return dict(op=op, hq=hq, hkv=hkv, batch=_log(rng, 1, max(1, min(128, 262144 // ctx))), ctx=ctx,
                    even=rng.random() < 0.3, mix=mix)
    if op == "prefill":
        new, ctx = _log(rng, 1, 2048), rng.choice([0, _log(rng, 1, 16384)])
        most = max(1, min(8, 67_000_000 // (new * (new + ctx))))
        return dict(op=op, hq=hq, hkv=hkv, seqs=rng.randint(1, most), new=new, ctx=ctx, even=rng.random() < 0.3,
                    mix=mix)
    blocks = _log(rng, 32, 512)
    return dict(op=op, hkv=hkv, layers=rng.randint(1, 32), blocks=blocks, pairs=_log(rng, 1, blocks // 2),
                fp8=rng.random() < 0.6, mix=mix)


def _spread(case, n, top, low):
    """``n`` whole numbers of [low, top], the largest first; spread over their logarithm."""
    r = random.Random(case["mix"] * 7 + n)
    return [top] + [low if top <= low else _log(r, max(low, 1), top) for _ in range(n - 1)]


def _rows(case):
    """(tokens in the cache before, new tokens) of each sequence of the case."""
    if case["op"] == "decode":
        n = [case["ctx"]] * case["batch"] if case["even"] else _spread(case, case["batch"], case["ctx"], 1)
        return [(c, 1) for c in n]
    seqs, new, ctx = case["seqs"], case["new"], case["ctx"]
    if case["op"] == "write":
        news = [new] * seqs if new == 1 or ctx == 0 else _spread(case, seqs, new, 1)
        return list(zip(_spread(case, seqs, ctx, 1) if ctx else [0] * seqs, news))
    if case["even"]:
        return [(ctx, new)] * seqs
    return list(zip(_spread(case, seqs, ctx, 1) if ctx else [0] * seqs, _spread(case, seqs, new, 1)))


# ----------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _two(e):
    """2^e in fp32 for whole e of [-126, 127]."""
    return ((e + 127).to(torch.int32) << 23).view(torch.float32)


def _pick(cache, at):
    """e4m3 rows, picked as bytes."""
    return cache.view(torch.uint8)[at].view(cache.dtype)


def _cache(blocks, hkv, g):
    """e4m3 rows with scales around 2^-6, so that the values are of order one."""
    x = torch.randn(blocks, hkv, BS, D, generator=g, device="cuda").mul_(60.0).clamp_(-448, 448)
    e = torch.randint(-8, -5, (blocks, hkv), generator=g, device="cuda")
    return x.to(torch.float8_e4m3fn), _two(e)


def _tables(lens, g, spare=3):
    """Block table [B, width] (unused entries 0) of a shuffled pool, and the pool's blocks."""
    need = [-(-n // BS) for n in lens]
    total = sum(need) + spare
    perm = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    width = max(need)
    at = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
    col = torch.arange(width, device="cuda")
    table = perm[(at[:, None] + col).clamp_(max=total - 1)]
    keep = col < torch.tensor(need, device="cuda")[:, None]
    return torch.where(keep, table, torch.zeros_like(table)).contiguous(), total


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = _gen(seed)
    op, hkv = case["op"], case["hkv"]
    bf = dict(dtype=torch.bfloat16, device="cuda")
    if op == "copy":
        n, nb, layers = case["pairs"], case["blocks"], case["layers"]
        perm = torch.randperm(nb, generator=g, device="cuda").to(torch.int32)
        pairs = torch.stack([perm[:n], perm[n:2 * n]], dim=1).contiguous()
        shape = (layers, 2, nb, hkv, BS, D)
        s = dict(case=case, pairs=pairs, scales=None)
        if case["fp8"]:
            raw = torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8)
            s["kv"] = raw.masked_fill_((raw & 127) == 127, 0).view(torch.float8_e4m3fn)
            s["scales"] = _two(torch.randint(-9, -4, shape[:4], generator=g, device="cuda"))
        else:
            s["kv"] = torch.empty(shape, **bf).normal_(generator=g)
        return s
    hq, rows = case["hq"], _rows(case)
    lens = [c + (0 if op == "decode" else n) for c, n in rows]      # a decode context holds its new token
    table, nb = _tables(lens, g)
    k, ks = _cache(nb, hkv, g)
    v, vs = _cache(nb, hkv, g)
    s = dict(case=case, k=k, v=v, ks=ks, vs=vs, table=table, rows=rows)
    if op == "decode":
        s["q"] = torch.randn(len(rows), hq * D, generator=g, device="cuda").mul_(1.5).to(torch.bfloat16)
        s["lens"] = _i32(lens)
        return s
    T = sum(n for _, n in rows)
    if op == "prefill":
        s["q"] = torch.randn(T, hq * D, generator=g, device="cuda").mul_(1.5).to(torch.bfloat16)
        return s
    seq = torch.repeat_interleave(torch.arange(len(rows)), torch.tensor([n for _, n in rows])).cuda()
    pos = torch.cat([torch.arange(c, c + n) for c, n in rows]).cuda()
    s["pos"] = pos.to(torch.int32)
    s["slots"] = table[seq, pos // BS].long() * BS + pos % BS
    # per-head magnitudes differ, so some blocks need a larger scale than their cached rows had
    mag = torch.exp2(torch.rand(hq + 2 * hkv, 1, generator=g, device="cuda") * 3 - 1.5)
    s["qkv"] = (torch.randn(T, hq + 2 * hkv, D, generator=g, device="cuda") * mag).to(torch.bfloat16).view(T, -1)
    if case["norm"]:
        s["qn"], s["kn"] = (torch.rand(D, generator=g, device="cuda").add_(0.5).to(torch.bfloat16) for _ in range(2))
    inv = 1.0 / (THETA ** (torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D))
    ang = torch.arange(max(lens), dtype=torch.float64, device="cuda")[:, None] * inv
    s["cos_sin"] = torch.cat([ang.cos(), ang.sin()], dim=1).float()
    return s


# ------------------------------------------------------------ plain forms
def _norm(x, w):
    """Per-head RMS norm, stored in bf16 as a layer of its own would."""
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()
    return y.to(torch.bfloat16).float()


def _rotate(x, cs):
    c, s = cs[:, None, :D // 2], cs[:, None, D // 2:]
    a, b = x[..., :D // 2], x[..., D // 2:]
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1).to(torch.bfloat16)


def _exponent(a):
    """The smallest e with a <= 448 * 2^e."""
    m, p = torch.frexp(a)
    e = p - 9 + (m > 0.875).to(p.dtype)
    return torch.where(a > 0, e, torch.full_like(e, MIN_EXP)).clamp(min=MIN_EXP)


def _append(cache, scale, x, slots):
    """Rows ``x`` [T, Hkv, D] (bf16) into their slots.  A block whose first row is
    written starts anew; any other keeps at least its old scale."""
    blk, off = slots // BS, slots % BS
    nb, hkv = scale.shape
    amax = torch.zeros(nb, hkv, device=x.device).index_reduce_(0, blk, x.float().abs().amax(-1), "amax")
    fresh = torch.zeros(nb, dtype=torch.bool, device=x.device).index_fill_(0, torch.where(off == 0, blk, blk[0]), True)
    fresh[blk[0]] = ((off == 0) & (blk == blk[0])).any()
    need = _exponent(amax)
    old = torch.frexp(scale)[1] - 1
    new = torch.where(fresh[:, None], need, torch.maximum(need, old))[blk]          # [T, Hkv]
    shift = torch.where(fresh[blk][:, None], torch.zeros_like(new), old[blk] - new)
    kept = _pick(cache, blk).float() * _two(shift.clamp(min=-126))[..., None, None]
    cache.view(torch.uint8)[blk] = kept.to(torch.float8_e4m3fn).view(torch.uint8)
    rows = (x.float() * _two(-new)[..., None]).to(torch.float8_e4m3fn)
    cache.view(torch.uint8)[blk, :, off] = rows.view(torch.uint8)
    scale[blk] = _two(new)


def _write(s):
    c = s["case"]
    hq, hkv = c["hq"], c["hkv"]
    x = s["qkv"].float().view(-1, hq + 2 * hkv, D)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], s["qkv"].view(-1, hq + 2 * hkv, D)[:, hq + hkv:]
    if c["norm"]:
        q, k = _norm(q, s["qn"]), _norm(k, s["kn"])
    cs = s["cos_sin"][s["pos"].long()]
    _append(s["k"], s["ks"], _rotate(k, cs), s["slots"])
    _append(s["v"], s["vs"], v, s["slots"])
    return {"q": _rotate(q, cs).reshape(-1, hq * D), "k": s["k"], "v": s["v"], "k_scale": s["ks"], "v_scale": s["vs"]}


def _gathered(cache, scale, table):
    """[B, Hkv, tokens, D] fp32 of every sequence's blocks."""
    t = table.long()
    x = _pick(cache, t).float() * scale[t][..., None, None]                                # [B, W, Hkv, BS, D]
    return x.permute(0, 2, 1, 3, 4).reshape(t.shape[0], x.shape[2], -1, D)


def _decode(s):
    c = s["case"]
    hq, hkv, B = c["hq"], c["hkv"], s["table"].shape[0]
    k, v = _gathered(s["k"], s["ks"], s["table"]), _gathered(s["v"], s["vs"], s["table"])
    off = (torch.arange(k.shape[2], device="cuda") >= s["lens"][:, None])[:, None, None]       # [B, 1, 1, tokens]
    q = s["q"].float().view(B, hkv, hq // hkv, D)
    a = (q @ k.transpose(2, 3)).mul_(1.0 / math.sqrt(D)).masked_fill_(off, -math.inf)
    p = (a - a.amax(-1, keepdim=True)).exp_()
    o = (p @ v) / p.sum(-1, keepdim=True)
    return o.reshape(B, hq * D).to(torch.bfloat16)


def _prefill(s):
    c = s["case"]
    hq, hkv, rows = c["hq"], c["hkv"], s["rows"]
    S, nmax, G = len(rows), max(n for _, n in rows), hq // hkv
    ctx, new = (torch.tensor([r[i] for r in rows], device="cuda") for i in (0, 1))
    at = torch.cumsum(new, 0) - new
    col = torch.arange(nmax, device="cuda")
    idx = (at[:, None] + col).clamp(max=s["q"].shape[0] - 1)                                   # [S, nmax]
    q = s["q"].float()[idx].view(S, nmax, hkv, G, D).permute(0, 2, 3, 1, 4).reshape(S, hkv, G * nmax, D)
    k, v = _gathered(s["k"], s["ks"], s["table"]), _gathered(s["v"], s["vs"], s["table"])
    a = (q @ k.transpose(2, 3)).mul_(1.0 / math.sqrt(D)).view(S, hkv, G, nmax, -1)
    key = torch.arange(a.shape[-1], device="cuda")
    a.masked_fill_((key > (ctx[:, None] + col)[..., None])[:, None, None], -math.inf)
    a.sub_(a.amax(-1, keepdim=True)).exp_()
    o = (a.view(S, hkv, G * nmax, -1) @ v) / a.sum(-1).view(S, hkv, G * nmax, 1)
    o = o.view(S, hkv, G, nmax, D).permute(0, 3, 1, 2, 4).reshape(S, nmax, hq * D)
    return o[col < new[:, None]].to(torch.bfloat16)


def _copy(s):
    src, dst = s["pairs"][:, 0].long(), s["pairs"][:, 1].long()
    kv = s["kv"].view(torch.uint8) if s["case"]["fp8"] else s["kv"]
    kv[:, :, dst] = kv[:, :, src]
    if s["scales"] is not None:
        s["scales"][:, :, dst] = s["scales"][:, :, src]
    return {"kv": s["kv"], "scales": s["scales"]}


# -------------------------------------------------- the framework's calls
def _own(s):
    from connex_b200 import ops
    c = s["case"]
    if c["op"] == "write":
        q = ops.rope_cache_fp8(s["qkv"], s["pos"], s["cos_sin"], c["hq"], c["hkv"], s["slots"], s["k"], s["v"],
                               s["ks"], s["vs"], q_norm=s.get("qn"), k_norm=s.get("kn"))
        return {"q": q, "k": s["k"], "v": s["v"], "k_scale": s["ks"], "v_scale": s["vs"]}
    if c["op"] == "decode":
        if "ws" not in s:                # a serving program makes the workspace once
            s["ws"] = ops.decode_workspace_fp8(c["batch"], c["hq"], c["hkv"], "cuda")
        return ops.decode_attention_fp8(s["q"], s["k"], s["v"], s["ks"], s["vs"], s["table"], s["lens"], c["hq"],
                                        s["ws"])
    if c["op"] == "prefill":
        if "tiles" not in s:             # made once per step, used by every layer
            s["tiles"] = ops.prefill_tile_info([n for _, n in s["rows"]], "cuda", ctx=[x for x, _ in s["rows"]])
        return ops.prefill_attention_paged_fp8(s["q"], s["k"], s["v"], s["ks"], s["vs"], s["table"], s["tiles"],
                                               c["hq"], c["hkv"])
    ops.kv_copy_blocks(s["kv"], s["pairs"], s["scales"])
    return {"kv": s["kv"], "scales": s["scales"]}


def run(state):
    if own:
        return _own(state)
    return {"write": _write, "decode": _decode, "prefill": _prefill, "copy": _copy}[state["case"]["op"]](state)


# ------------------------------------------------------------------- work
def work(case):
    op, hkv = case["op"], case["hkv"]
    if op == "copy":
        per = hkv * BS * D * (1 if case["fp8"] else 2) + (4 * hkv if case["fp8"] else 0)
        return {"bytes": 2.0 * case["pairs"] * 2 * case["layers"] * per, "flops": 0.0}
    hq, rows = case["hq"], _rows(case)
    if op == "write":
        T = sum(n for _, n in rows)
        blocks = sum((c + n - 1) // BS - c // BS + 1 for c, n in rows)
        # q, k, v in; q and the e4m3 rows out; a table row, a position and a slot per token; scales read and written
        return {"bytes": float(T * ((2 * hq + 2 * hkv) * D * 2 + 2 * hkv * D + D * 4 + 12) + blocks * 2 * hkv * 8),
                "flops": float(T * ((hq + hkv) * D * 3 + 2 * hkv * D))}
    lens = [c + (0 if op == "decode" else n) for c, n in rows]
    T = sum(n for _, n in rows)
    blocks = sum(-(-n // BS) for n in lens)
    pairs = sum(lens) if op == "decode" else sum(n * c + n * (n + 1) // 2 for c, n in rows)
    return {"bytes": float(2 * hkv * D * sum(lens) + blocks * (8 * hkv + 4) + 2 * T * hq * D * 2),
            "flops": 4.0 * pairs * hq * D}


# ------------------------------------------------------- 64-bit definition
def exact(case, seed):
    if case["op"] == "copy":
        return None
    s = prepare(case, seed)
    return _exact_write(s) if case["op"] == "write" else _exact_attention(s)


def _exact_attention(s):
    """softmax(q k^T / sqrt(D)) v per sequence and KV head, the keys up to the query's own position."""
    c = s["case"]
    hq, hkv = c["hq"], c["hkv"]
    G, out, at = hq // hkv, [], 0
    for b, (ctx, n) in enumerate(s["rows"]):
        if c["op"] == "decode":
            ctx -= 1
        ids = s["table"][b, :-(-(ctx + n) // BS)].long()
        o = torch.empty(n, hq, D, dtype=torch.float64, device="cuda")
        for h in range(hkv):
            k, v = ((_pick(t[:, h], ids).double() * z[ids, h].double()[:, None, None]).reshape(-1, D)[:ctx + n]
                    for t, z in ((s["k"], s["ks"]), (s["v"], s["vs"])))
            dead = torch.arange(ctx + n, device="cuda") > ctx + torch.arange(n, device="cuda")[:, None]
            for j in range(h * G, (h + 1) * G):
                a = s["q"][at:at + n, j * D:(j + 1) * D].double() @ k.t() / math.sqrt(D)
                o[:, j] = torch.softmax(a.masked_fill(dead, -math.inf), -1) @ v
        out.append(o.reshape(n, hq * D))
        at += n
    return torch.cat(out)


def _exact_write(s):
    """Block by block: which rows arrive, the scale that holds them, every row on the e4m3 grid."""
    c = s["case"]
    hq, hkv = c["hq"], c["hkv"]
    x = s["qkv"].double().view(-1, hq + 2 * hkv, D)
    cs = s["cos_sin"].double()[s["pos"].long()]
    rot = torch.complex(cs[:, :D // 2], cs[:, D // 2:])[:, None]

    def turn(t, w):
        if c["norm"]:
            t = t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6) * w.double()
            t = t.to(torch.bfloat16).double()
        z = torch.complex(t[..., :D // 2], t[..., D // 2:]) * rot
        return torch.cat([z.real, z.imag], -1)

    def grid(y):
        """To the nearest e4m3 value, ties to even: 3 fraction bits, exponents from -6 up."""
        e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -30))).clamp(min=-6)
        step = torch.exp2(e - 3)
        return torch.round(y / step) * step

    slots = s["slots"].tolist()
    by = {}
    for t, slot in enumerate(slots):
        by.setdefault(slot // BS, []).append(t)

    def fill(cache, scale, new):
        data, sc = cache.double(), scale.double()
        ids = torch.tensor(list(by), device="cuda")
        first = torch.tensor([min(slots[t] % BS for t in ts) for ts in by.values()], device="cuda")
        rows = torch.full((len(by), BS), -1, dtype=torch.long)
        for i, ts in enumerate(by.values()):
            for t in ts:
                rows[i, slots[t] % BS] = t
        rows = rows.cuda()
        put = rows >= 0
        val = new[rows.clamp(min=0)].transpose(1, 2) * put[:, None, :, None]                   # [blocks, Hkv, BS, D]
        top = val.abs().amax((2, 3))
        need = torch.ceil(torch.log2((top / 448).clamp(min=2.0 ** MIN_EXP))).clamp(min=MIN_EXP)
        # log2 is exact enough except next to a power of two: settle those by comparison
        need = torch.where(top > 448 * torch.exp2(need), need + 1, need)
        need = torch.where((need > MIN_EXP) & (top <= 448 * torch.exp2(need - 1)), need - 1, need)
        old = sc[ids]
        size = torch.where((first == 0)[:, None], torch.exp2(need), torch.maximum(old, torch.exp2(need)))
        keep = torch.where((first == 0)[:, None], torch.ones_like(size), old / size)
        data[ids] = torch.where(put[:, None, :, None], grid(val / size[..., None, None]),
                                grid(data[ids] * keep[..., None, None]))
        sc[ids] = size
        return data, sc

    k = turn(x[:, hq:hq + hkv], s.get("kn")).to(torch.bfloat16).double()     # quantised from its bf16 value
    kd, ks = fill(s["k"], s["ks"], k)
    vd, vs = fill(s["v"], s["vs"], x[:, hq + hkv:])
    return {"q": turn(x[:, :hq], s.get("qn")).reshape(-1, hq * D), "k": kd, "v": vd, "k_scale": ks, "v_scale": vs}
