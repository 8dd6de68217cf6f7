"""Cases and plain forms of the operators for serving in few bits.

Weights and activations in e4m3 with a scale for each block of 128, and a paged
KV cache in 4 bits, as a serving step uses them layer by layer:

* ``quant``    rows of activations to e4m3, one fp32 scale per row and 128
               columns, optionally after an RMS norm
* ``gemm``     the product of such rows with a weight in e4m3 that has one fp32
               scale per 128 x 128 block; the residual added, or SiLU(gate) * up
               quantised for the next product
* ``write``    rotate q and k, k and v into the 4-bit cache
* ``decode``   attention of one new token per sequence over its 4-bit cache
* ``prefill``  causal attention of prompt chunks that continue cached sequences

The 4-bit cache holds [blocks, Hkv, 16 tokens, 72 bytes]: 64 bytes of 4-bit codes
(dims 2i and 2i + 1 in the low and high half of byte i), then scale and minimum,
bf16 each, of dims 0..63 and of dims 64..127.  A value is minimum + code * scale.

``own`` false: elementary torch operations in fp32.  ``own`` true: the calls of
``connex_b200.ops``.
"""
import math
import random

import torch

own = False

BS, D, HALF = 16, 128, 64          # tokens of a cache block, head size, dims that share a scale
ROW = 72                           # bytes of a cached token's head
Q = 128                            # columns (and weight rows) that share an fp8 scale
THETA = 500000.0
EPS = 1e-5
TINY = 2.0 ** -100                 # largest magnitude of a block, at least


# ------------------------------------------------------------------ cases
def listed():
    return [
        # the normed input of a projection in a step of 64 generating requests: a launch-bound call per layer
        dict(name="quant-decode", op="quant", rows=64, k=4096, norm=True),
        # the attention's output of a full prefill step, before the output projection
        dict(name="quant-prefill", op="quant", rows=8192, k=4096, norm=False),
        # one request alone: the fused QKV projection, latency
        dict(name="gemm-single", op="gemm", m=1, n=6144, k=4096, epi="store"),
        # the down projection of 64 generating requests: the weight's bytes count
        dict(name="gemm-decode", op="gemm", m=64, n=4096, k=14336, epi="add"),
        # ragged prompt chunks through the output projection of a 2048-wide model
        dict(name="gemm-chunks", op="gemm", m=613, n=2048, k=4096, epi="add"),
        # a full prefill step through gate and up
        dict(name="gemm-prefill", op="gemm", m=8192, n=28672, k=4096, epi="silu"),
        # one decode step's new rows, written somewhere inside a block
        dict(name="write-decode", op="write", hq=32, hkv=8, seqs=64, new=1, ctx=20, norm=False, mix=11),
        # ragged chunks of five prompts that begin inside a block, with per-head q/k norms
        dict(name="write-chunks", op="write", hq=32, hkv=4, seqs=5, new=1613, ctx=77, norm=True, mix=13),
        # a full decode batch at the flagship's context
        dict(name="decode-batch", op="decode", hq=32, hkv=8, batch=64, ctx=4096, even=True, mix=22),
        # requests of very different ages, eight query heads per KV head
        dict(name="decode-ragged", op="decode", hq=32, hkv=4, batch=96, ctx=8191, even=False, mix=23),
        # the tails of several prompts: short ragged chunks over medium contexts
        dict(name="prefill-short", op="prefill", hq=32, hkv=8, seqs=5, new=131, ctx=2000, even=False, mix=31),
        # one chunk of a long prompt in the middle of its reading
        dict(name="prefill-chunk", op="prefill", hq=32, hkv=8, seqs=1, new=2048, ctx=6144, even=True, mix=32),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quant", "gemm", "gemm", "write", "decode", "prefill"])
    if op == "quant":
        return dict(op=op, rows=_log(rng, 1, 8192), k=16 * _log(rng, 1, 896), norm=rng.random() < 0.5)
    if op == "gemm":
        epi = rng.choice(["store", "add", "silu"])
        m = _log(rng, 1, 8192)
        n = 256 * _log(rng, 1, 112) if epi == "silu" else 8 * _log(rng, 8, 3584)
        k = 16 * _log(rng, 8, 896)
        return dict(op=op, m=min(m, 8192 * 28672 * 4096 // (n * k)), n=n, k=k, epi=epi)
    mix = rng.randrange(1, 1 << 30)
    hq, hkv = rng.choice([(32, 8), (32, 4), (8, 2), (28, 4), (16, 1), (6, 2), (4, 4), (5, 1)])
    if op == "write":
        if rng.random() < 0.5:
            return dict(op=op, hq=hq, hkv=hkv, seqs=_log(rng, 1, 256), new=1, ctx=rng.randint(0, 40),
                        norm=rng.random() < 0.3, mix=mix)
        new = _log(rng, 2, 2048)
        return dict(op=op, hq=hq, hkv=hkv, seqs=rng.randint(1, max(1, min(8, 8192 // new))), new=new,
                    ctx=rng.choice([0, rng.randint(1, 100)]), norm=rng.random() < 0.3, mix=mix)
    if op == "decode":
        ctx = _log(rng, 1, 131072)
        return dict(op=op, hq=hq, hkv=hkv, batch=_log(rng, 1, max(1, min(128, 262144 // ctx))), ctx=ctx,
                    even=rng.random() < 0.3, mix=mix)
    new, ctx = _log(rng, 1, 2048), rng.choice([0, _log(rng, 1, 16384)])
    most = max(1, min(8, 67_000_000 // (new * (new + ctx))))
    return dict(op=op, hq=hq, hkv=hkv, seqs=rng.randint(1, most), new=new, ctx=ctx, even=rng.random() < 0.3, mix=mix)


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


def _quant4(x):
    """bf16 [..., 128] -> bytes [..., 72]."""
    f = x.float().unflatten(-1, (2, HALF))
    lo, hi = f.amin(-1), f.amax(-1)
    scale, low = ((hi - lo) / 15).to(torch.bfloat16), lo.to(torch.bfloat16)
    inv = torch.where(scale > 0, 1.0 / scale.float(), torch.zeros_like(hi))
    code = ((f - lo[..., None]) * inv[..., None]).round_().clamp_(0, 15).to(torch.uint8).flatten(-2)
    packed = code[..., 0::2] | (code[..., 1::2] << 4)
    return torch.cat([packed, torch.stack([scale, low], -1).flatten(-2).view(torch.uint8)], -1)


def _values4(raw, dtype=torch.float32):
    """bytes [..., 72] -> the values that they stand for [..., 128]."""
    code = torch.stack([raw[..., :HALF] & 15, raw[..., :HALF] >> 4], -1).flatten(-2)
    par = raw[..., HALF:].contiguous().view(torch.bfloat16).to(dtype)
    return (code.to(dtype).unflatten(-1, (2, HALF)) * par[..., 0::2, None] + par[..., 1::2, None]).flatten(-2)


def _cache(blocks, hkv, g, skew):
    """Cached rows of order one; with ``skew`` around a mean of their own in each channel, as keys are."""
    x = torch.randn(blocks, hkv, BS, D, generator=g, device="cuda")
    if skew:
        x.add_(torch.randn(hkv, 1, D, generator=g, device="cuda"))
    return _quant4(x.to(torch.bfloat16))


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


def _prepare_rows(case, g):
    """Activations: columns of different sizes, a few of them far larger than the others."""
    x = torch.randn(case["rows"], case["k"], generator=g, device="cuda")
    size = torch.exp2(torch.rand(case["k"], generator=g, device="cuda") * 2 - 1)
    size[::97] *= 20
    s = dict(case=case, x=(x * size).to(torch.bfloat16))
    if case["norm"]:
        s["w"] = torch.rand(case["k"], generator=g, device="cuda").add_(0.5).to(torch.bfloat16)
    return s


def _prepare_gemm(case, g):
    m, n, k = case["m"], case["n"], case["k"]
    kb, nb = -(-k // Q), -(-n // Q)
    s = dict(case=case)
    s["a"] = torch.randn(m, k, generator=g, device="cuda").mul_(120).clamp_(-448, 448).to(torch.float8_e4m3fn)
    s["b"] = torch.randn(n, k, generator=g, device="cuda").mul_(120).clamp_(-448, 448).to(torch.float8_e4m3fn)
    # scales that bring activations to the order of one and weights to a hundredth; a row's scales lie side by
    # side with the other rows', as the quantising call leaves them
    s["sa"] = torch.rand(kb, m, generator=g, device="cuda").add_(0.5).div_(120).t()
    s["sb"] = torch.rand(nb, kb, generator=g, device="cuda").add_(0.5).div_(120 * 64)
    if case["epi"] == "add":
        s["x"] = torch.randn(m, n, generator=g, device="cuda").to(torch.bfloat16)
    return s


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "quant":
        return _prepare_rows(case, g)
    if op == "gemm":
        return _prepare_gemm(case, g)
    hq, hkv, rows = case["hq"], case["hkv"], _rows(case)
    lens = [c + (0 if op == "decode" else n) for c, n in rows]      # a decode context holds its new token
    table, nb = _tables(lens, g)
    s = dict(case=case, k=_cache(nb, hkv, g, True), v=_cache(nb, hkv, g, False), table=table, rows=rows)
    if op == "decode":
        s["q"] = torch.randn(len(rows), hq * D, generator=g, device="cuda").to(torch.bfloat16)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        return s
    T = sum(n for _, n in rows)
    if op == "prefill":
        s["q"] = torch.randn(T, hq * D, generator=g, device="cuda").to(torch.bfloat16)
        return s
    seq = torch.repeat_interleave(torch.arange(len(rows)), torch.tensor([n for _, n in rows])).cuda()
    pos = torch.cat([torch.arange(c, c + n) for c, n in rows]).cuda()
    s["pos"] = pos.to(torch.int32)
    s["slots"] = table[seq, pos // BS].long() * BS + pos % BS
    s["qkv"] = torch.randn(T, (hq + 2 * hkv) * D, generator=g, device="cuda").to(torch.bfloat16)
    if case["norm"]:
        s["qn"], s["kn"] = (torch.rand(D, generator=g, device="cuda").add_(0.5).to(torch.bfloat16) for _ in range(2))
    inv = 1.0 / (THETA ** (torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D))
    ang = torch.arange(max(lens), dtype=torch.float64, device="cuda")[:, None] * inv
    s["cos_sin"] = torch.cat([ang.cos(), ang.sin()], dim=1).float()
    return s


# ------------------------------------------------------------ plain forms
def _blocked(x):
    """fp32 [T, K] -> e4m3 [T, K] and its scales [T, K / 128]."""
    T, K = x.shape
    kb = -(-K // Q)
    f = torch.zeros(T, kb * Q, device=x.device)
    f[:, :K] = x
    f = f.view(T, kb, Q)
    top = f.abs().amax(-1).clamp_(min=TINY)
    q = (f * (448.0 / top)[..., None]).clamp_(-448, 448).view(T, -1)[:, :K].to(torch.float8_e4m3fn)
    return q, top / 448.0


def _quant(s):
    x = s["x"].float()
    if s["case"]["norm"]:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * s["w"].float()
    q, scale = _blocked(x)
    return {"q": q, "scale": scale}


def _spread_scale(q, scale):
    """e4m3 [R, K] times scales [R or R / 128, K / 128] -> fp32."""
    R, K = q.shape
    if scale.shape[0] != R:
        scale = scale.repeat_interleave(Q, 0)[:R]
    return q.float() * scale.repeat_interleave(Q, 1)[:, :K]


def _gemm(s):
    y = _spread_scale(s["a"], s["sa"]) @ _spread_scale(s["b"], s["sb"]).t()
    epi = s["case"]["epi"]
    if epi == "silu":                       # gate and up alternate, 128 rows of the weight each
        y = y.unflatten(1, (-1, 2, Q))
        gate, up = y[:, :, 0].flatten(1), y[:, :, 1].flatten(1)
        q, scale = _blocked(gate / (1 + torch.exp(-gate)) * up)
        return {"q": q, "scale": scale}
    return (y + s["x"].float() if epi == "add" else y).to(torch.bfloat16)


def _norm(x, w):
    """Per-head RMS norm, stored in bf16 as a layer of its own would."""
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()
    return y.to(torch.bfloat16).float()


def _rotate(x, cs):
    c, s = cs[:, None, :D // 2], cs[:, None, D // 2:]
    a, b = x[..., :D // 2], x[..., D // 2:]
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1).to(torch.bfloat16)


def _write(s):
    c = s["case"]
    hq, hkv = c["hq"], c["hkv"]
    rows = s["qkv"].view(-1, hq + 2 * hkv, D)
    x = rows.float()
    q, k = x[:, :hq], x[:, hq:hq + hkv]
    if c["norm"]:
        q, k = _norm(q, s["qn"]), _norm(k, s["kn"])
    cs = s["cos_sin"][s["pos"].long()]
    blk, off = s["slots"] // BS, s["slots"] % BS
    s["k"][blk, :, off] = _quant4(_rotate(k, cs))
    s["v"][blk, :, off] = _quant4(rows[:, hq + hkv:])
    return {"q": _rotate(q, cs).reshape(-1, hq * D), "k": _values4(s["k"]).to(torch.bfloat16),
            "v": _values4(s["v"]).to(torch.bfloat16)}


def _gathered(cache, table):
    """[B, Hkv, tokens, D] fp32 of every sequence's blocks."""
    t = table.long()
    return _values4(cache[t]).permute(0, 2, 1, 3, 4).reshape(t.shape[0], cache.shape[1], -1, D)


def _decode(s):
    c = s["case"]
    hq, hkv, B = c["hq"], c["hkv"], s["table"].shape[0]
    k, v = _gathered(s["k"], s["table"]), _gathered(s["v"], s["table"])
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
    k, v = _gathered(s["k"], s["table"]), _gathered(s["v"], s["table"])
    a = (q @ k.transpose(2, 3)).mul_(1.0 / math.sqrt(D)).view(S, hkv, G, nmax, -1)
    key = torch.arange(a.shape[-1], device="cuda")
    a.masked_fill_((key > (ctx[:, None] + col)[..., None])[:, None, None], -math.inf)
    a.sub_(a.amax(-1, keepdim=True)).exp_()
    o = (a.view(S, hkv, G * nmax, -1) @ v) / a.sum(-1).view(S, hkv, G * nmax, 1)
    o = o.view(S, hkv, G, nmax, D).permute(0, 3, 1, 2, 4).reshape(S, nmax, hq * D)
    return o[col < new[:, None]].to(torch.bfloat16)


# -------------------------------------------------- the framework's calls
def _own(s):
    from connex_b200 import ops
    c = s["case"]
    if c["op"] == "quant":
        q, scale = ops.quantize_fp8(s["x"], norm=s.get("w"), eps=EPS)
        return {"q": q, "scale": scale}
    if c["op"] == "gemm":
        out = ops.gemm_fp8(s["a"], s["sa"], s["b"], s["sb"], residual=s.get("x"), silu_mul=c["epi"] == "silu")
        return {"q": out[0], "scale": out[1]} if c["epi"] == "silu" else out
    if c["op"] == "write":
        q = ops.rope_cache_int4(s["qkv"], s["pos"], s["cos_sin"], c["hq"], c["hkv"], s["slots"], s["k"], s["v"],
                                q_norm=s.get("qn"), k_norm=s.get("kn"))
        return {"q": q, "k": ops.kv_values_int4(s["k"]), "v": ops.kv_values_int4(s["v"])}
    if c["op"] == "decode":
        if "ws" not in s:                # a serving program makes the workspace once
            s["ws"] = ops.decode_workspace_int4(c["batch"], c["hq"], c["hkv"], "cuda")
        return ops.decode_attention_int4(s["q"], s["k"], s["v"], s["table"], s["lens"], c["hq"], s["ws"])
    if "tiles" not in s:                 # made once per step, used by every layer
        s["tiles"] = ops.prefill_tile_info([n for _, n in s["rows"]], "cuda", ctx=[x for x, _ in s["rows"]])
    return ops.prefill_attention_paged_int4(s["q"], s["k"], s["v"], s["table"], s["tiles"], c["hq"], c["hkv"])


def run(state):
    if own:
        return _own(state)
    return {"quant": _quant, "gemm": _gemm, "write": _write, "decode": _decode,
            "prefill": _prefill}[state["case"]["op"]](state)


# ------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "quant":
        T, K = case["rows"], case["k"]
        return {"bytes": float(T * (3 * K + 4 * -(-K // Q)) + (2 * K if case["norm"] else 0)), "flops": 4.0 * T * K}
    if op == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        kb, nb = -(-k // Q), -(-n // Q)
        out = {"store": 2 * m * n, "add": 4 * m * n, "silu": m * n // 2 + 4 * m * (n // 2 // Q)}[case["epi"]]
        return {"bytes": float(m * k + n * k + 4 * kb * (m + nb) + out), "flops": 2.0 * m * n * k}
    hq, hkv, rows = case["hq"], case["hkv"], _rows(case)
    if op == "write":
        T = sum(n for _, n in rows)
        blocks = 3 + sum(-(-(c + n) // BS) for c, n in rows)
        # q, k, v in; q and the cached rows out; a table row, a position and a slot per token; the caches' values
        return {"bytes": float(T * ((2 * hq + 2 * hkv) * D * 2 + 2 * hkv * ROW + D * 4 + 12)
                               + 2 * blocks * hkv * BS * (ROW + 2 * D)),
                "flops": float(T * ((hq + hkv) * D * 3 + 2 * hkv * D * 4) + 4 * blocks * hkv * BS * D)}
    lens = [c + (0 if op == "decode" else n) for c, n in rows]
    T = sum(n for _, n in rows)
    pairs = sum(lens) if op == "decode" else sum(n * c + n * (n + 1) // 2 for c, n in rows)
    return {"bytes": float(2 * hkv * ROW * sum(lens) + 4 * sum(-(-n // BS) for n in lens) + 2 * T * hq * D * 2),
            "flops": 4.0 * pairs * hq * D}


# ------------------------------------------------------- 64-bit definition
def exact(case, seed):
    s = prepare(case, seed)
    return {"quant": _exact_quant, "gemm": _exact_gemm, "write": _exact_write, "decode": _exact_attention,
            "prefill": _exact_attention}[case["op"]](s)


def _grid8(y):
    """To the nearest e4m3 value, ties to even: 3 fraction bits, exponents from -6 up."""
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -30))).clamp(min=-6)
    step = torch.exp2(e - 3)
    return torch.round(y / step) * step


def _exact_blocks(x):
    parts = [x[:, i:i + Q] for i in range(0, x.shape[1], Q)]
    size = torch.stack([p.abs().amax(1).clamp(min=TINY) / 448 for p in parts], 1)
    return {"q": torch.cat([_grid8(p / size[:, i, None]) for i, p in enumerate(parts)], 1), "scale": size}


def _exact_quant(s):
    x = s["x"].double()
    if s["case"]["norm"]:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * s["w"].double()
    return _exact_blocks(x)


def _exact_gemm(s):
    """Block by block: sums over 128 columns, then their two scales."""
    c = s["case"]
    y = torch.zeros(c["m"], c["n"], dtype=torch.float64, device="cuda")
    for n0 in range(0, c["n"], 4096):                       # weight rows at a time: the products stay small
        n1 = min(c["n"], n0 + 4096)
        rows = torch.arange(n0, n1, device="cuda") // Q
        for i, k0 in enumerate(range(0, c["k"], Q)):
            part = s["a"][:, k0:k0 + Q].double() @ s["b"][n0:n1, k0:k0 + Q].double().t()
            y[:, n0:n1] += part * s["sa"][:, i, None].double() * s["sb"][rows, i].double()
    if c["epi"] == "silu":
        j = torch.arange(c["n"] // 2, device="cuda")
        at = j // Q * (2 * Q) + j % Q
        gate = y[:, at]
        return _exact_blocks(gate * torch.sigmoid(gate) * y[:, at + Q])
    return y + s["x"].double() if c["epi"] == "add" else y


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
            k, v = (_unpacked(t[ids, h]).reshape(-1, D)[:ctx + n] for t in (s["k"], s["v"]))
            dead = torch.arange(ctx + n, device="cuda") > ctx + torch.arange(n, device="cuda")[:, None]
            for j in range(h * G, (h + 1) * G):
                a = s["q"][at:at + n, j * D:(j + 1) * D].double() @ k.t() / math.sqrt(D)
                o[:, j] = torch.softmax(a.masked_fill(dead, -math.inf), -1) @ v
        out.append(o.reshape(n, hq * D))
        at += n
    return torch.cat(out)


def _unpacked(raw):
    """bytes [..., 72] -> fp64 [..., 128], dim by dim of a byte."""
    x = torch.empty(*raw.shape[:-1], D, dtype=torch.float64, device=raw.device)
    code = raw[..., :HALF].to(torch.int64)
    x[..., 0::2], x[..., 1::2] = (code % 16).double(), (code // 16).double()
    bits = raw[..., HALF:].to(torch.int32)
    par = ((bits[..., 1::2] << 24) | (bits[..., 0::2] << 16)).view(torch.float32).double()      # bf16: the upper half
    x[..., :HALF] = x[..., :HALF] * par[..., 0:1] + par[..., 1:2]
    x[..., HALF:] = x[..., HALF:] * par[..., 2:3] + par[..., 3:4]
    return x


def _exact_write(s):
    """Row by row: 16 levels from the minimum of a half up, the step in bf16."""
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

    def levels(t):
        out = []
        for h in (t[..., :HALF], t[..., HALF:]):
            low = h.amin(-1, keepdim=True)
            step = ((h.amax(-1, keepdim=True) - low) / 15).to(torch.bfloat16).double()
            code = torch.round((h - low) / step.clamp(min=1e-300)).clamp(0, 15)
            out.append(low + code * step)
        return torch.cat(out, -1)

    blk, off = s["slots"] // BS, s["slots"] % BS
    k, v = _unpacked(s["k"]), _unpacked(s["v"])
    k[blk, :, off] = levels(turn(x[:, hq:hq + hkv], s.get("kn")).to(torch.bfloat16).double())   # as its bf16 value
    v[blk, :, off] = levels(x[:, hq + hkv:])
    return {"q": turn(x[:, :hq], s.get("qn")).reshape(-1, hq * D), "k": k, "v": v}
