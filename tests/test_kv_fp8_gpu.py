"""The 8-bit paged KV cache on the GPU: the quantising write, decode and
chunked prefill attention over it and block copies, each against a plain
64-bit statement.

Tolerances.  One rounding to a type t is off by at most eps(t) / 2 of the
value: bf16 2^-8, f16 2^-11, fp32 2^-24, e4m3 2^-4 (and half of its smallest
step, 2^-10 of the scale, below the normal range)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

D, BS = 128, 16
U_BF16, U_F16, U_F32, U_E4M3 = 2.0 ** -8, 2.0 ** -11, 2.0 ** -24, 2.0 ** -4


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def _g(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _cache(nb, hkv, dev, seed, lo=-8, hi=-4):
    g = _g(dev, seed)
    x = (torch.randn(nb, hkv, BS, D, generator=g, device=dev) * 60).clamp(-448, 448).to(torch.float8_e4m3fn)
    e = torch.randint(lo, hi, (nb, hkv), generator=g, device=dev)
    return x, torch.ldexp(torch.ones(nb, hkv, device=dev), e).float()


def _nan_rows(cache, table, lens):
    """Cache rows behind each sequence's last token hold NaN bytes."""
    raw = cache.view(torch.uint8)
    for b, n in enumerate(lens):
        if n % BS:
            raw[int(table[b, n // BS]), :, n % BS:] = 0x7F
        elif n == 0:
            raw[int(table[b, 0])] = 0xFF


def _table(lens, dev, seed, width=None):
    need = [max(1, -(-n // BS)) for n in lens]
    perm = torch.randperm(sum(need) + 3, generator=_g(dev, seed), device=dev).to(torch.int32)
    w = width or max(need)
    t = torch.full((len(lens), w), -1, dtype=torch.int32, device=dev)   # ids behind the end are never read
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = perm[at:at + n]
        at += n
    return t, sum(need) + 3


def _attention_tolerance(ref, mag, q, k_cache, k_scale, table, ctx, n_new, u_weight, vmax):
    """|out - ref| <= bf16 of the result + the weights' rounding (u_weight, and
    f16's smallest half step for each) + the logits' fp32 sums (128 products:
    128 * 2^-24 of sum |q_i k_i| each, twice: the weight and the sum)."""
    from connex_b200.ops import reference as R
    big, s = [], 0
    hkv = k_cache.shape[1]
    for b, (c, n) in enumerate(zip(ctx, n_new)):
        if c + n == 0 or n == 0:
            s += n
            continue
        ids = table[b, :-(-(c + n) // BS)].long()
        k = R.fp8_values(k_cache.view(torch.uint8)[ids].view(k_cache.dtype), k_scale[ids]).nan_to_num(0.0)
        k = k.transpose(0, 1).reshape(hkv, -1, D)[:, :c + n].abs().repeat_interleave(q.shape[1] // hkv, 0)
        qs = q[s:s + n].double().abs().transpose(0, 1)
        big.append((qs @ k.transpose(1, 2)).max().item() / math.sqrt(D))
        s += n
    logit = (max(big) if big else 0.0) * D * U_F32
    n = max([c + m for c, m in zip(ctx, n_new)] + [1])
    return U_BF16 * ref.abs() + mag * (2 * u_weight + 4 * logit + n * U_F32 + 2.0 ** -20) + n * 2.0 ** -25 * vmax


DECODE_LENS = [[1], [0, 5, 0], [16], [17, 1, 15, 16, 31, 33], [500], [4096, 3, 0, 1000], [129] * 70, [20000, 1],
               [128] * 64, [1500] * 40 + [0, 1480]]


@pytest.mark.parametrize("heads", [(32, 8), (8, 8), (6, 2), (7, 1), (16, 1), (20, 2), (32, 4)])
@pytest.mark.parametrize("lens", DECODE_LENS, ids=lambda v: f"{len(v)}x{max(v)}")
def test_decode_attention(dev, heads, lens):
    from connex_b200 import ops
    from connex_b200.ops import reference as R
    hq, hkv = heads
    table, nb = _table(lens, dev, 1)
    k, ks = _cache(nb, hkv, dev, 2)
    v, vs = _cache(nb, hkv, dev, 3, -12, 3)
    _nan_rows(k, table, lens)
    _nan_rows(v, table, lens)
    B = len(lens)
    # q as a slice of wider rows, as the fused projection leaves it
    wide = (torch.randn(B, (hq + 2) * D, generator=_g(dev, 4), device=dev) * 1.5).to(torch.bfloat16)
    q = wide[:, :hq * D]
    st = ops.new_status(dev)
    ws = ops.decode_workspace_fp8(B, hq, hkv, dev)
    lt = torch.tensor(lens, dtype=torch.int32, device=dev)
    out = ops.decode_attention_fp8(wide, k, v, ks, vs, table, lt, hq, ws, status=st)
    torch.cuda.synchronize()
    ops.check_status(st, "decode_attention_fp8")
    ctx = [max(0, n - 1) for n in lens]
    live = torch.tensor([n > 0 for n in lens], device=dev)
    got = out.view(B, hq, D).double()
    assert torch.equal(got[~live], torch.zeros_like(got[~live]))
    rows = q.reshape(B, hq, D)[live]
    tl = table[live]
    ref, mag = R.paged_attention_fp8(rows, k, v, ks, vs, tl, [c for c, n in zip(ctx, lens) if n], [1] * int(live.sum()))
    tol = _attention_tolerance(ref, mag, rows, k, ks, tl, [c for c, n in zip(ctx, lens) if n], [1] * int(live.sum()),
                               U_F16, float(vs.max()) * 448)
    assert ((got[live] - ref).abs() <= tol).all(), float(((got[live] - ref).abs() / tol).max())
    # the workspace is left ready: the same call again, the same bits
    again = ops.decode_attention_fp8(wide, k, v, ks, vs, table, lt, hq, ws)
    assert torch.equal(again.view(torch.int16), out.view(torch.int16))


@pytest.mark.parametrize("heads", [(4, 1), (20, 2)])
def test_decode_of_many_sequences(dev, heads):
    """Up to the most sequences of a call, next to calls of a few with the same workspace: the grid depends on
    their number, the workspace's layout does not."""
    from connex_b200 import ops
    from connex_b200.ops import reference as R
    hq, hkv = heads
    ws = ops.decode_workspace_fp8(4096, hq, hkv, dev)
    for seed, lens in enumerate(([i % 70 for i in range(4096)], [3000, 1, 900], [200 + i % 90 for i in range(1450)], [5000])):
        table, nb = _table(lens, dev, 131 + seed)
        k, ks = _cache(nb, hkv, dev, 141 + seed)
        v, vs = _cache(nb, hkv, dev, 151 + seed)
        q = (torch.randn(len(lens), hq * D, generator=_g(dev, 161 + seed), device=dev) * 1.5).to(torch.bfloat16)
        lt = torch.tensor(lens, dtype=torch.int32, device=dev)
        st = ops.new_status(dev)
        out = ops.decode_attention_fp8(q, k, v, ks, vs, table, lt, hq, ws, status=st)
        ops.check_status(st)
        live = [b for b, n in enumerate(lens) if n]
        assert not out[[b for b, n in enumerate(lens) if not n]].any()
        ctx, ones = [lens[b] - 1 for b in live], [1] * len(live)
        rows, tl = q[live].view(-1, hq, D), table[live]
        ref, mag = R.paged_attention_fp8(rows, k, v, ks, vs, tl, ctx, ones)
        tol = _attention_tolerance(ref, mag, rows, k, ks, tl, ctx, ones, U_F16, float(vs.max()) * 448)
        assert ((out[live].view(-1, hq, D).double() - ref).abs() <= tol).all()
        again = ops.decode_attention_fp8(q, k, v, ks, vs, table, lt, hq, ws)
        assert torch.equal(again.view(torch.int16), out.view(torch.int16))


PREFILL_ROWS = [[(0, 100)], [(64, 128)], [(1000, 300), (17, 5)], [(2000, 1), (130, 513)], [(5, 64), (0, 200), (3999, 129)],
                [(2048, 600)], [(7, 9), (0, 1), (15, 1), (16, 1)], [(300, 0), (41, 30)], [(12000, 33), (500, 257)]]


@pytest.mark.parametrize("heads", [(8, 2), (3, 3), (7, 1), (16, 1), (6, 2)])
@pytest.mark.parametrize("rows", PREFILL_ROWS, ids=lambda v: "_".join(f"{c}+{n}" for c, n in v))
def test_prefill_attention(dev, heads, rows):
    from connex_b200 import ops
    from connex_b200.ops import reference as R
    hq, hkv = heads
    ctx, new = [c for c, _ in rows], [n for _, n in rows]
    lens = [c + n for c, n in rows]
    table, nb = _table(lens, dev, 5)
    k, ks = _cache(nb, hkv, dev, 6)
    v, vs = _cache(nb, hkv, dev, 7, -10, -2)
    _nan_rows(k, table, lens)
    _nan_rows(v, table, lens)
    T = sum(new)
    q = (torch.randn(T, hq * D, generator=_g(dev, 8), device=dev) * 1.5).to(torch.bfloat16)
    st = ops.new_status(dev)
    ti = ops.prefill_tile_info(new, dev, ctx=ctx)
    out = ops.prefill_attention_paged_fp8(q, k, v, ks, vs, table, ti, hq, hkv, status=st)
    torch.cuda.synchronize()
    ops.check_status(st, "prefill_attention_paged_fp8")
    ref, mag = R.paged_attention_fp8(q.view(T, hq, D), k, v, ks, vs, table, ctx, new)
    tol = _attention_tolerance(ref, mag, q.view(T, hq, D), k, ks, table, ctx, new, U_BF16, float(vs.max()) * 448)
    err = (out.view(T, hq, D).double() - ref).abs()
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("mode", [1, 2, 4])
@pytest.mark.parametrize("rows", [[(12000, 33), (500, 257)], [(2048, 600)]])
def test_prefill_with_other_exponentials(dev, mode, rows):
    """attention_exp_split holds for this attention, too: other bits, within the mode's own error."""
    from connex_b200 import ops
    from connex_b200.ops import reference as R
    hq, hkv = 8, 2
    ctx, new = [c for c, _ in rows], [n for _, n in rows]
    table, nb = _table([c + n for c, n in rows], dev, 181)
    k, ks = _cache(nb, hkv, dev, 182)
    v, vs = _cache(nb, hkv, dev, 183, -10, -2)
    q = (torch.randn(sum(new), hq * D, generator=_g(dev, 184), device=dev) * 0.25).to(torch.bfloat16)
    ti = ops.prefill_tile_info(new, dev, ctx=ctx)
    st = ops.new_status(dev)
    plain = ops.prefill_attention_paged_fp8(q, k, v, ks, vs, table, ti, hq, hkv, status=st)
    try:
        ops._C.attention_exp_split(mode)
        out = ops.prefill_attention_paged_fp8(q, k, v, ks, vs, table, ti, hq, hkv, status=st)
        torch.cuda.synchronize()
    finally:
        ops._C.attention_exp_split(0)
    ops.check_status(st)
    assert not torch.equal(out.view(torch.int16), plain.view(torch.int16))
    q3 = q.view(-1, hq, D)
    ref, mag = R.paged_attention_fp8(q3, k, v, ks, vs, table, ctx, new)
    # a weight's relative error: its rounding to bf16 and the cubic's 7.5e-5 (1e-4 with its own fp32 roundings); or
    # 2^-7 of the packed instruction and an exponent rounded to bf16, 2^-8 of its size, which is at most twice the
    # largest logit in base 2 and 8 for the late rescale
    if mode == 1:
        norms = (R.fp8_values(k.view(torch.uint8).view(k.dtype), ks).square().sum(-1).sqrt().max().item()
                 * q3.double().square().sum(-1).sqrt().max().item())
        u = 2.0 ** -7 + U_BF16 * math.log(2) * (2 * norms / math.sqrt(D) / math.log(2) + 8)
    else:
        u = U_BF16 + 1e-4
    tol = _attention_tolerance(ref, mag, q3, k, ks, table, ctx, new, u, float(vs.max()) * 448)
    assert ((out.view(-1, hq, D).double() - ref).abs() <= tol).all()


def test_prefill_profile(dev):
    """attention_profile's counters are filled by this attention, too, and its result is the same."""
    from connex_b200 import ops
    hq, hkv = 8, 2
    table, nb = _table([2148], dev, 191)
    k, ks = _cache(nb, hkv, dev, 192)
    v, vs = _cache(nb, hkv, dev, 193)
    q = torch.randn(300, hq * D, generator=_g(dev, 194), device=dev).to(torch.bfloat16)
    ti = ops.prefill_tile_info([300], dev, ctx=[1848])
    plain = ops.prefill_attention_paged_fp8(q, k, v, ks, vs, table, ti, hq, hkv)
    sms = torch.cuda.get_device_properties(dev).multi_processor_count
    buf = torch.zeros(sms, 16, dtype=torch.int64, device=dev)
    ops._C.attention_profile(buf.data_ptr())
    try:
        out = ops.prefill_attention_paged_fp8(q, k, v, ks, vs, table, ti, hq, hkv)
        torch.cuda.synchronize()
    finally:
        ops._C.attention_profile(0)
    assert torch.equal(out.view(torch.int16), plain.view(torch.int16))
    # CTAs with work: the MMA thread's total, both softmax warpgroups' waits, work and epilogues
    busy = buf[buf[:, 5] > 0]
    assert busy.shape[0] > 0 and (busy[:, 6:14].sum(0) > 0).all()


@pytest.mark.parametrize("heads", [(128, 1), (12, 1), (40, 8)])
def test_prefill_other_groups(dev, heads):
    """Groups of which all, some or none of the heads share a tile's rows."""
    test_prefill_attention(dev, heads, [(200, 9), (40, 130)])


def test_prefill_replayed(dev):
    """A captured call divides the work from what the tiles hold at its replay, and gives an eager call's bits."""
    from connex_b200 import ops
    hq, hkv = 8, 2
    table, nb = _table([5000, 700], dev, 9)
    table = table.clamp(min=0)
    k, ks = _cache(nb, hkv, dev, 10)
    v, vs = _cache(nb, hkv, dev, 11)
    q = torch.randn(300, hq * D, generator=_g(dev, 12), device=dev).to(torch.bfloat16)
    tiles = [ops.prefill_tile_info([200, 100], dev, ctx=c) for c in ([4800, 600], [3, 0], [100, 333])]
    ti = tiles[0].clone()
    call = lambda: ops.prefill_attention_paged_fp8(q, k, v, ks, vs, table, ti, hq, hkv)  # noqa: E731
    call()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for t in tiles + tiles[:1]:
        assert t.shape == ti.shape
        ti.copy_(t)
        g.replay()
        got = out.clone()
        g.replay()
        assert torch.equal(out, got) and torch.equal(call(), got)


def _write_case(dev, rows, hq, hkv, seed, norm=False, spread=3.0):
    """A cache that holds each sequence's first ctx tokens, and n new rows."""
    from connex_b200 import ops
    lens = [c + n for c, n in rows]
    table, nb = _table(lens, dev, seed)
    k, ks = _cache(nb, hkv, dev, seed + 1, -9, -4)
    v, vs = _cache(nb, hkv, dev, seed + 2, -9, -4)
    pos = [p for c, n in rows for p in range(c, c + n)]
    slots = [int(table[b, p // BS]) * BS + p % BS for b, (c, n) in enumerate(rows) for p in range(c, c + n)]
    g = _g(dev, seed + 3)
    mag = torch.exp2(torch.rand(hq + 2 * hkv, 1, generator=g, device=dev) * 2 * spread - spread)
    qkv = (torch.randn(len(pos), hq + 2 * hkv, D, generator=g, device=dev) * mag).to(torch.bfloat16).view(len(pos), -1)
    cs = ops.rope_cos_sin(max(lens), D, 5e5, dev)
    w = [(torch.rand(D, generator=g, device=dev) + 0.5).to(torch.bfloat16) for _ in range(2)] if norm else [None, None]
    return dict(k=k, ks=ks, v=v, vs=vs, pos=torch.tensor(pos, dtype=torch.int32, device=dev),
                slots=torch.tensor(slots, dtype=torch.int64, device=dev), qkv=qkv, cs=cs, qn=w[0], kn=w[1], nb=nb)


def _turned(x, pos, cs, w):
    """Rotated rows in 64 bits, and a bound on what a flip of the norm's bf16 rounding moves them."""
    x = x.double()
    slack = torch.zeros_like(x)
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.double()
        x = x.to(torch.bfloat16).double()
        pair = x.abs() + x.abs().roll(D // 2, -1)
        slack = 2 * U_BF16 * pair
    t = cs.double()[pos.long()][:, None]
    c, s = t[..., :D // 2], t[..., D // 2:]
    a, b = x[..., :D // 2], x[..., D // 2:]
    # two products and a sum in fp32
    slack = slack + 4 * U_F32 * (x.abs() + x.abs().roll(D // 2, -1))
    return torch.cat([a * c - b * s, b * c + a * s], -1), slack


WRITE_ROWS = [[(0, 1)], [(0, 16)], [(15, 1)], [(16, 1)], [(37, 1), (100, 1), (0, 1), (15, 1)], [(0, 33), (7, 9), (5, 70)],
              [(1000, 129)], [(3, 2), (20, 40), (0, 300)], [(i, 1) for i in range(70)]]


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("heads", [(8, 2), (3, 3), (7, 1), (32, 8), (20, 5)])
@pytest.mark.parametrize("rows", WRITE_ROWS, ids=lambda v: f"{len(v)}x{v[0][0]}+{v[0][1]}")
def test_write(dev, rows, heads, norm):
    from connex_b200 import ops
    from connex_b200.ops import reference as R
    hq, hkv = heads
    s = _write_case(dev, rows, hq, hkv, 11, norm)
    T = s["qkv"].shape[0]
    x = s["qkv"].view(T, hq + 2 * hkv, D)
    before = {n: s[n].clone() for n in ("k", "ks", "v", "vs", "qkv")}
    st = ops.new_status(dev)
    q = ops.rope_cache_fp8(s["qkv"], s["pos"], s["cs"], hq, hkv, s["slots"], s["k"], s["v"], s["ks"], s["vs"], status=st,
                           q_norm=s["qn"], k_norm=s["kn"])
    torch.cuda.synchronize()
    ops.check_status(st, "rope_cache_fp8")
    assert torch.equal(s["qkv"], before["qkv"])
    ref, slack = _turned(x[:, :hq], s["pos"], s["cs"], s["qn"])
    err = (q.view(T, hq, D).double() - ref).abs()
    assert (err <= U_BF16 * ref.abs() + 2 * slack).all()
    # v is quantised as it stands: the very bytes and scales
    v, vs = before["v"].clone(), before["vs"].clone()
    R.fp8_append(v, vs, x[:, hq + hkv:], s["slots"])
    assert torch.equal(vs, s["vs"])
    touched = torch.zeros(s["nb"], dtype=torch.bool, device=dev)
    touched[s["slots"] // BS] = True
    assert torch.equal(v.float(), s["v"].float())
    assert torch.equal(before["v"][~touched].view(torch.uint8), s["v"][~touched].view(torch.uint8))
    assert torch.equal(before["k"][~touched].view(torch.uint8), s["k"][~touched].view(torch.uint8))
    assert torch.equal(before["ks"][~touched], s["ks"][~touched])
    # k: each row within half an e4m3 step of its rotated value, held by its scale
    kr, ks_ = _turned(x[:, hq:hq + hkv], s["pos"], s["cs"], s["kn"])
    val = R.fp8_values(s["k"], s["ks"])
    blk, off = s["slots"] // BS, s["slots"] % BS
    got, sc = val[blk, :, off], s["ks"].double()[blk][..., None]
    tol = (1 + 2 * U_BF16) * (U_E4M3 * kr.abs()).maximum(2.0 ** -10 * sc) + U_BF16 * kr.abs() + 2 * ks_
    assert ((got - kr).abs() <= tol).all()
    # the scale is the smallest that holds the rows (or the old one, where the block goes on)
    low = torch.zeros(s["nb"], hkv, dtype=torch.float64, device=dev).index_reduce_(0, blk, (kr.abs() * (1 - 2 * U_BF16) - 2 * ks_).amax(-1), "amax")
    top = torch.zeros(s["nb"], hkv, dtype=torch.float64, device=dev).index_reduce_(0, blk, (kr.abs() * (1 + 2 * U_BF16) + 2 * ks_).amax(-1), "amax")
    fresh = torch.zeros(s["nb"], dtype=torch.bool, device=dev)
    fresh[blk[off == 0]] = True
    old = torch.where(fresh[:, None], torch.zeros_like(low), before["ks"].double())
    assert (s["ks"].double() >= torch.maximum(R.fp8_scale(low), old))[touched].all()
    assert (s["ks"].double() <= torch.maximum(R.fp8_scale(top), old))[touched].all()
    # rows that the call did not write keep their values, to half the smallest step of a raised scale
    kept = torch.ones(s["nb"], BS, dtype=torch.bool, device=dev)
    kept[blk, off] = False
    kept &= touched[:, None] & ~fresh[:, None]
    was = R.fp8_values(before["k"], before["ks"])
    d = (val - was).abs().transpose(1, 2)[kept]
    room = (2.0 ** -10 * s["ks"].double() * (s["ks"] != before["ks"]))[:, None, :, None].expand(-1, BS, -1, D)[kept]
    assert (d <= room).all()


def test_write_order_repeats_and_skips(dev):
    """Rows of one block apart from each other, a slot written twice, slots below zero."""
    from connex_b200 import ops
    from connex_b200.ops import reference as R
    hq, hkv, nb = 4, 2, 40
    k, ks = _cache(nb, hkv, dev, 21)
    v, vs = _cache(nb, hkv, dev, 22)
    slots = [5 * BS + 3, 7 * BS, 5 * BS + 4, 7 * BS + 1, -1, 5 * BS + 3, 9 * BS + 15, 7 * BS, -7, 5 * BS + 2]
    T = len(slots)
    qkv = torch.randn(T, (hq + 2 * hkv) * D, generator=_g(dev, 23), device=dev).to(torch.bfloat16) * 4
    pos = torch.arange(T, dtype=torch.int32, device=dev)
    cs = ops.rope_cos_sin(64, D, 1e4, dev)
    st = ops.new_status(dev)
    rv, rvs = v.clone(), vs.clone()
    sl = torch.tensor(slots, dtype=torch.int64, device=dev)
    ops.rope_cache_fp8(qkv, pos, cs, hq, hkv, sl, k, v, ks, vs, status=st)
    ops.check_status(st)
    R.fp8_append(rv, rvs, qkv.view(T, -1, D)[:, hq + hkv:], sl)
    assert torch.equal(vs, rvs) and torch.equal(v.float(), rv.float())


def test_write_out_of_range(dev):
    """Bad slots and positions are recorded, cached nowhere, and change nothing else."""
    from connex_b200 import ops
    hq, hkv, nb = 4, 2, 6
    for slots, pos in (([nb * BS, 0], [0, 1]), ([0, 16], [64, 1]), ([0, 1], [3, -1]), ([1 << 40, 5], [0, 0])):
        k, ks = _cache(nb, hkv, dev, 31)
        v, vs = _cache(nb, hkv, dev, 32)
        good = [0 <= s < nb * BS and 0 <= p < 64 for s, p in zip(slots, pos)]
        qkv = torch.randn(2, (hq + 2 * hkv) * D, generator=_g(dev, 33), device=dev).to(torch.bfloat16)
        st = ops.new_status(dev)
        k0, v0 = k.clone(), v.clone()
        cs = ops.rope_cos_sin(64, D, 1e4, dev)
        q = ops.rope_cache_fp8(qkv, torch.tensor(pos, dtype=torch.int32, device=dev), cs, hq, hkv,
                               torch.tensor(slots, dtype=torch.int64, device=dev), k, v, ks, vs, status=st)
        with pytest.raises(RuntimeError, match="bounds"):
            ops.check_status(st)
        assert torch.isfinite(q.float()).all()
        hit = {s // BS for s, g in zip(slots, good) if g}
        for b in range(nb):
            if b not in hit:
                assert torch.equal(k[b].view(torch.uint8), k0[b].view(torch.uint8))
                assert torch.equal(v[b].view(torch.uint8), v0[b].view(torch.uint8))
        for i, p in enumerate(pos):
            if not 0 <= p < 64:
                assert not q[i].any()


def test_write_special_values(dev):
    """NaN and infinities are stored as NaN and leave the scale alone; zeros take the smallest scale."""
    from connex_b200 import ops
    hq, hkv, nb = 2, 1, 4
    k, ks = _cache(nb, hkv, dev, 41)
    v, vs = _cache(nb, hkv, dev, 42)
    qkv = torch.zeros(3, (hq + 2 * hkv) * D, device=dev, dtype=torch.bfloat16)
    qkv[0, -D:] = 3.0
    qkv[0, -D] = float("inf")
    qkv[0, -D + 1] = float("nan")
    qkv[0, -D + 2] = float("-inf")
    qkv[2, -D:] = torch.finfo(torch.bfloat16).max
    cs = ops.rope_cos_sin(64, D, 1e4, dev)
    i32 = torch.tensor([0, 1, 2], dtype=torch.int32, device=dev)
    ops.rope_cache_fp8(qkv, i32, cs, hq, hkv, torch.tensor([0, 16, 32], dtype=torch.int64, device=dev), k, v, ks, vs)
    row = v[0, 0, 0].float()
    assert torch.isnan(row[:3]).all() and torch.equal(row[3:] * vs[0, 0], torch.full((D - 3,), 3.0, device=dev))
    assert float(vs[1, 0]) == 2.0 ** -100 and not v[1, 0, 0].float().any()
    # the largest bf16 is 1.992 * 2^127: in steps of 2^124 the nearest e4m3 value is 2^128, so the scale is 2^120
    assert float(vs[2, 0]) == 2.0 ** 120 and torch.equal(v[2, 0, 0].float(), torch.full((D,), 256.0, device=dev))


def test_write_long_call(dev):
    """Past 8192 rows a call runs as successive ones; a block at the seam holds both parts."""
    from connex_b200 import ops
    from connex_b200.ops import reference as R
    hq, hkv, T = 1, 1, 8192 + 40
    nb = T // BS + 4
    k, ks = _cache(nb, hkv, dev, 51)
    v, vs = _cache(nb, hkv, dev, 52)
    qkv = torch.randn(T, 3 * D, generator=_g(dev, 53), device=dev).to(torch.bfloat16)
    slots = torch.arange(5, T + 5, device=dev)
    pos = torch.arange(T, dtype=torch.int32, device=dev)
    rv, rvs = v.clone(), vs.clone()
    ops.rope_cache_fp8(qkv, pos, ops.rope_cos_sin(T, D, 1e4, dev), hq, hkv, slots, k, v, ks, vs)
    rows = qkv.view(T, 3, D)[:, 2:]
    R.fp8_append(rv, rvs, rows[:8192], slots[:8192])
    R.fp8_append(rv, rvs, rows[8192:], slots[8192:])
    assert torch.equal(vs, rvs) and torch.equal(v.float(), rv.float())


def test_write_in_place(dev):
    """out as qkv's own q columns gives the same q."""
    from connex_b200 import ops
    s = _write_case(dev, [(0, 40), (9, 3)], 6, 2, 61)
    a = ops.rope_cache_fp8(s["qkv"], s["pos"], s["cs"], 6, 2, s["slots"], s["k"], s["v"], s["ks"], s["vs"])
    ops.rope_cache_fp8(s["qkv"], s["pos"], s["cs"], 6, 2, s["slots"], s["k"], s["v"], s["ks"], s["vs"],
                       out=s["qkv"][:, :6 * D])
    assert torch.equal(s["qkv"][:, :6 * D], a)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("layers,nb,hkv,n", [(1, 4, 1, 1), (3, 50, 2, 17), (32, 40, 8, 20), (2, 9000, 1, 4000)])
def test_copy_blocks(dev, dtype, layers, nb, hkv, n):
    from connex_b200 import ops
    from connex_b200.ops import reference as R
    g = _g(dev, 71)
    kv = torch.randint(0, 256, (layers, 2, nb, hkv, BS, D * dtype.itemsize), generator=g, device=dev,
                       dtype=torch.uint8).view(dtype)
    scales = torch.rand(layers, 2, nb, hkv, generator=g, device=dev) if dtype == torch.float8_e4m3fn else None
    perm = torch.randperm(nb, generator=g, device=dev).to(torch.int32)
    pairs = torch.stack([perm[:n], perm[n:2 * n]], 1).contiguous()
    if n > 3:                                # one source for two destinations; a repeated pair; a block onto itself
        pairs[1, 0] = pairs[0, 0]
        pairs[2] = pairs[0]
        pairs[3, 1] = pairs[3, 0]
    ref, rs = kv.clone(), None if scales is None else scales.clone()
    R.kv_copy_blocks(ref, pairs, rs)
    st = ops.new_status(dev)
    ops.kv_copy_blocks(kv, pairs, scales, status=st)
    ops.check_status(st, "kv_copy_blocks")
    assert torch.equal(kv.view(torch.uint8), ref.view(torch.uint8))
    assert scales is None or torch.equal(scales, rs)


def test_copy_blocks_conflicts(dev):
    """Pairs without a defined result are left out and recorded; the others run."""
    from connex_b200 import ops
    g = _g(dev, 81)
    base = torch.randn(2, 2, 12, 1, BS, D, generator=g, device=dev).to(torch.bfloat16)
    for pairs, done in (([(0, 1), (1, 2)], [(1, 2)]), ([(0, 5), (3, 5)], []), ([(0, 12), (3, 4)], [(3, 4)]),
                        ([(-1, 2), (3, 4)], [(3, 4)]), ([(6, 7), (7, 6)], []), ([(2, 2), (3, 2)], [])):
        kv, ref = base.clone(), base.clone()
        for a, b in done:
            ref[:, :, b] = base[:, :, a]
        st = ops.new_status(dev)
        ops.kv_copy_blocks(kv, torch.tensor(pairs, dtype=torch.int32, device=dev), status=st)
        with pytest.raises(RuntimeError, match="bounds"):
            ops.check_status(st)
        assert torch.equal(kv, ref), pairs


def test_decode_bad_pages_and_lengths(dev):
    """A block id out of range is left out, a length beyond the table cut; both recorded."""
    from connex_b200 import ops
    from connex_b200.ops import reference as R
    hq, hkv = 8, 2
    k, ks = _cache(20, hkv, dev, 91)
    v, vs = _cache(20, hkv, dev, 92)
    q = torch.randn(2, hq * D, generator=_g(dev, 93), device=dev).to(torch.bfloat16)
    ws = ops.decode_workspace_fp8(2, hq, hkv, dev)
    for table, lens, like in (([[3, 20, 5], [1, 2, 4]], [48, 48], ([[3, 5, 5], [1, 2, 4]], [32, 48])),
                              ([[3, -5, 5], [1, 2, 4]], [48, 20], ([[3, 5, 5], [1, 2, 4]], [32, 20])),
                              ([[3, 4, 5], [1, 2, 6]], [49, -3], ([[3, 4, 5], [1, 2, 6]], [48, 0]))):
        st = ops.new_status(dev)
        i = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        out = ops.decode_attention_fp8(q, k, v, ks, vs, i(table), i(lens), hq, ws, status=st)
        with pytest.raises(RuntimeError, match="bounds"):
            ops.check_status(st)
        t, n = like
        ref, mag = R.paged_attention_fp8(q.view(2, hq, D), k, v, ks, vs, i(t), [x - 1 if x else 0 for x in n], [1, 1])
        for b in range(2):
            if n[b] == 0:
                assert not out[b].any()
            else:
                err = (out[b].view(hq, D).double() - ref[b]).abs()
                assert (err <= U_BF16 * ref[b].abs() + mag[b] * 2.0 ** -8 + 1e-6).all()


def test_prefill_bad_pages_and_tiles(dev):
    """A block id out of range reads as zeros; a tile that fits neither the rows nor the tables is left out."""
    from connex_b200 import ops
    from connex_b200.ops import reference as R
    hq, hkv, nb = 4, 2, 12
    k, ks = _cache(nb, hkv, dev, 121)
    v, vs = _cache(nb, hkv, dev, 122)
    q = torch.randn(40, hq * D, generator=_g(dev, 123), device=dev).to(torch.bfloat16)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    table = i32([[3, 4, 1], [5, 6, 2]])
    good = [(0, 20, 0, 28, 0), (20, 20, 0, 10, 1)]
    st = ops.new_status(dev)
    ref = ops.prefill_attention_paged_fp8(q, k, v, ks, vs, table, i32(good), hq, hkv, status=st)
    ops.check_status(st)
    for bad in ((20, 20, 0, 29, 1), (21, 20, 0, 10, 1), (-1, 5, 0, 0, 1), (20, 20, 0, 10, 2), (20, 20, 20, 10, 1),
                (20, 0, 0, 10, 1), (20, 20, 0, -1, 1), (20, 20, -1, 10, 1), (20, 20, 0, 2**31 - 1, 1)):
        st = ops.new_status(dev)
        out = torch.full_like(ref, 7.0)
        ops.prefill_attention_paged_fp8(q, k, v, ks, vs, table, i32([good[0], bad]), hq, hkv, out=out, status=st)
        with pytest.raises(RuntimeError, match="bounds"):
            ops.check_status(st)
        assert torch.equal(out[:20], ref[:20]) and (out[20:] == 7.0).all()
    # room for just the blocks read (3 of the first sequence, 2 of the second), and for one fewer
    st = ops.new_status(dev)
    out = ops.prefill_attention_paged_fp8(q, k, v, ks, vs, table, i32(good), hq, hkv, status=st, n_blocks=5)
    ops.check_status(st)
    assert torch.equal(out, ref)
    out = ops.prefill_attention_paged_fp8(q, k, v, ks, vs, table, i32(good), hq, hkv, status=st, n_blocks=4)
    with pytest.raises(RuntimeError, match="bounds"):
        ops.check_status(st)
    assert torch.equal(out[:20], ref[:20])
    for bad in (nb, -1, 2**31 - 1):
        st = ops.new_status(dev)
        t = table.clone()
        t[1, 1] = bad
        out = ops.prefill_attention_paged_fp8(q, k, v, ks, vs, t, i32(good), hq, hkv, status=st)
        with pytest.raises(RuntimeError, match="bounds"):
            ops.check_status(st)
        assert torch.equal(out[:20], ref[:20])
        k0, v0 = k.clone(), v.clone()
        k0.view(torch.uint8)[6] = 0
        v0.view(torch.uint8)[6] = 0
        want, mag = R.paged_attention_fp8(q.view(40, hq, D)[20:], k0, v0, ks, vs, table[1:], [10], [20])
        err = (out[20:].view(20, hq, D).double() - want).abs()
        assert (err <= U_BF16 * want.abs() + mag * 2.0 ** -6 + 1e-6).all()


def test_two_streams_at_once(dev):
    """Calls on two streams, each with a workspace of its own, give the bits of calls one after another."""
    from connex_b200 import ops
    hq, hkv = 16, 4
    sides = []
    for i, lens in enumerate(([3000, 17, 900], [64, 5000, 1, 333])):
        table, nb = _table(lens, dev, 151 + i)
        k, ks = _cache(nb, hkv, dev, 153 + i)
        v, vs = _cache(nb, hkv, dev, 155 + i)
        new = [min(n, 70) for n in lens]
        q = torch.randn(sum(new), hq * D, generator=_g(dev, 157 + i), device=dev).to(torch.bfloat16)
        cache = (k, v, ks, vs, table)
        sides.append((cache, q, torch.tensor(lens, dtype=torch.int32, device=dev),
                      ops.prefill_tile_info(new, dev, ctx=[n - m for n, m in zip(lens, new)]),
                      ops.decode_workspace_fp8(len(lens), hq, hkv, dev)))

    def both(side):
        cache, q, lens, ti, ws = side
        return (ops.decode_attention_fp8(q[:len(lens)], *cache, lens, hq, ws),
                ops.prefill_attention_paged_fp8(q, *cache, ti, hq, hkv))
    want = [both(side) for side in sides]
    streams = [torch.cuda.Stream(dev) for _ in sides]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (side, stream) in enumerate(zip(sides, streams)):
            with torch.cuda.stream(stream):
                got[i].append(both(side))
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        assert all(torch.equal(x, y) for run in runs for x, y in zip(run, w))


def test_offsets_past_32_bits(dev):
    """Blocks that lie more than 4 GB into the cache give the bits of the same blocks at its start."""
    from connex_b200 import ops
    hq, hkv, far = 16, 8, 270000
    assert far * hkv * BS * D > 2 ** 32
    n, T = 40, 600
    big = torch.empty(1, 2, far + n, hkv, BS, D, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
    sc = torch.ones(1, 2, far + n, hkv, device=dev)
    qkv = torch.randn(T, (hq + 2 * hkv) * D, generator=_g(dev, 141), device=dev).to(torch.bfloat16)
    cs = ops.rope_cos_sin(T, D, 5e5, dev)
    pos = torch.arange(T, dtype=torch.int32, device=dev)
    ws = ops.decode_workspace_fp8(1, hq, hkv, dev)
    lens = torch.tensor([T], dtype=torch.int32, device=dev)
    ti = ops.prefill_tile_info([T], dev, ctx=[0])
    got = []
    for at in (0, far):
        k, v, ks, vs = big[0, 0], big[0, 1], sc[0, 0], sc[0, 1]
        st = ops.new_status(dev)
        q = ops.rope_cache_fp8(qkv, pos, cs, hq, hkv, torch.arange(T, device=dev) + at * BS, k, v, ks, vs, status=st)
        table = torch.arange(at, at + n, dtype=torch.int32, device=dev)[None]
        got.append((k[at:at + n].clone().view(torch.uint8).flatten()[:T * hkv * D], ks[at:at + n].clone(),
                    ops.decode_attention_fp8(q[-1:], k, v, ks, vs, table, lens, hq, ws, status=st),
                    ops.prefill_attention_paged_fp8(q, k, v, ks, vs, table, ti, hq, hkv, status=st)))
        ops.check_status(st)
    full = T // BS * hkv * BS * D
    assert torch.equal(got[0][0][:full], got[1][0][:full])
    assert all(torch.equal(a, b) for a, b in zip(got[0][1:], got[1][1:]))
    pairs = torch.tensor([[far + i, i + 1] for i in range(30)], dtype=torch.int32, device=dev)
    ops.kv_copy_blocks(big, pairs, sc)
    assert torch.equal(big[:, :, 1:31].view(torch.uint8), big[:, :, far:far + 30].view(torch.uint8))
    assert torch.equal(sc[:, :, 1:31], sc[:, :, far:far + 30])


def test_empty_calls(dev):
    """No rows, no sequences, no tiles, no table, no pairs: nothing is written and nothing fails."""
    from connex_b200 import ops
    hq, hkv, nb = 8, 2, 6
    k, ks = _cache(nb, hkv, dev, 131)
    v, vs = _cache(nb, hkv, dev, 132)
    was = [t.view(torch.uint8).clone() for t in (k, v)]
    i32 = lambda *n: torch.zeros(*n, dtype=torch.int32, device=dev)  # noqa: E731
    st = ops.new_status(dev)
    cs = ops.rope_cos_sin(64, D, 5e5, dev)
    qkv = torch.zeros(0, (hq + 2 * hkv) * D, dtype=torch.bfloat16, device=dev)
    out = ops.rope_cache_fp8(qkv, i32(0), cs, hq, hkv, torch.zeros(0, dtype=torch.int64, device=dev), k, v, ks, vs, status=st)
    assert out.shape == (0, hq * D)
    ws = ops.decode_workspace_fp8(3, hq, hkv, dev)
    q = torch.ones(3, hq * D, dtype=torch.bfloat16, device=dev)
    assert ops.decode_attention_fp8(q[:0], k, v, ks, vs, i32(0, 4), i32(0), hq, ws, status=st).shape == (0, hq * D)
    assert (ops.decode_attention_fp8(q, k, v, ks, vs, i32(3, 0), i32(3), hq, ws, status=st) == 0).all()
    tiles = torch.tensor([[0, 3, 0, 0, 0]], dtype=torch.int32, device=dev)
    ops.prefill_attention_paged_fp8(q[:0], k, v, ks, vs, i32(1, 4), tiles, hq, hkv, status=st)
    kept = torch.full((3, hq * D), 7.0, dtype=torch.bfloat16, device=dev)
    ops.prefill_attention_paged_fp8(q, k, v, ks, vs, i32(1, 4), tiles[:0], hq, hkv, out=kept, status=st)
    assert (kept == 7.0).all()
    for table, n in ((i32(0, 4), None), (i32(1, 0), None), (i32(1, 4), 0)):
        with pytest.raises(RuntimeError, match="no block table"):
            ops.prefill_attention_paged_fp8(q, k, v, ks, vs, table, tiles, hq, hkv, status=st, n_blocks=n)
    ops.kv_copy_blocks(torch.stack((k, v))[None], i32(0, 2), torch.stack((ks, vs))[None], status=st)
    ops.check_status(st)
    assert all(torch.equal(t.view(torch.uint8), w) for t, w in zip((k, v), was))
    # a length but no table: cut, and recorded
    assert (ops.decode_attention_fp8(q, k, v, ks, vs, i32(3, 0), i32(3) + 5, hq, ws, status=st) == 0).all()
    with pytest.raises(RuntimeError, match="bounds"):
        ops.check_status(st)


def test_decode_nan_and_extreme_logits(dev):
    """A NaN key poisons its own head only; logits far apart and q's of any size stay exact enough."""
    from connex_b200 import ops
    from connex_b200.ops import reference as R
    hq, hkv = 4, 2
    table, nb = _table([100, 60], dev, 101)
    k, ks = _cache(nb, hkv, dev, 102)
    v, vs = _cache(nb, hkv, dev, 103)
    ws = ops.decode_workspace_fp8(2, hq, hkv, dev)
    lens = torch.tensor([100, 60], dtype=torch.int32, device=dev)
    for size in (1e-30, 1e-3, 300.0, 1e30):
        q = (torch.randn(2, hq * D, generator=_g(dev, 104), device=dev) * size).to(torch.bfloat16)
        out = ops.decode_attention_fp8(q, k, v, ks, vs, table, lens, hq, ws).view(2, hq, D).double()
        ref, mag = R.paged_attention_fp8(q.view(2, hq, D), k, v, ks, vs, table, [99, 59], [1, 1])
        tol = _attention_tolerance(ref, mag, q.view(2, hq, D), k, ks, table, [99, 59], [1, 1], U_F16, float(vs.max()) * 448)
        assert ((out - ref).abs() <= tol).all(), size
    k.view(torch.uint8)[table[0, 2].long(), 1, 5, 7] = 0x7F
    q = torch.randn(2, hq * D, generator=_g(dev, 105), device=dev).to(torch.bfloat16)
    out = ops.decode_attention_fp8(q, k, v, ks, vs, table, lens, hq, ws).view(2, hq, D)
    assert torch.isnan(out[0, 2:].float()).all()
    assert torch.isfinite(out[0, :2].float()).all() and torch.isfinite(out[1].float()).all()


def test_step_in_a_graph(dev):
    """Write and decode captured together and replayed while the lengths grow, next
    to the same steps run eagerly; a second graph with its own workspace on another stream."""
    from connex_b200 import ops
    hq, hkv, B, width = 8, 2, 5, 8
    nb = B * width + 1
    table = torch.arange(1, nb, dtype=torch.int32, device=dev).view(B, width)
    cs = ops.rope_cos_sin(256, D, 1e4, dev)

    def make():
        c = [torch.zeros(nb, hkv, BS, D, device=dev).to(torch.float8_e4m3fn) for _ in range(2)]
        c += [torch.ones(nb, hkv, device=dev) for _ in range(2)]
        io = dict(qkv=torch.zeros(B, (hq + 2 * hkv) * D, dtype=torch.bfloat16, device=dev),
                  pos=torch.zeros(B, dtype=torch.int32, device=dev), slots=torch.full((B,), -1, dtype=torch.int64, device=dev),
                  lens=torch.ones(B, dtype=torch.int32, device=dev), ws=ops.decode_workspace_fp8(B, hq, hkv, dev),
                  st=ops.new_status(dev))
        return c, io

    def step(c, io):
        q = ops.rope_cache_fp8(io["qkv"], io["pos"], cs, hq, hkv, io["slots"], *c, status=io["st"])
        return ops.decode_attention_fp8(q, *c, table, io["lens"], hq, io["ws"], status=io["st"])
    sides = [make() for _ in range(3)]
    graphs = []
    for c, io in sides[:2]:
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            step(c, io)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(c, io)
        graphs.append((g, out, s))
    for t in range(40):
        x = (torch.randn(B, (hq + 2 * hkv) * D, generator=_g(dev, 200 + t), device=dev) * (1 + t % 7)).to(torch.bfloat16)
        pos = torch.tensor([(t + 3 * b) % 100 if t >= 0 else 0 for b in range(B)], dtype=torch.int32, device=dev)
        for c, io in sides:
            io["qkv"].copy_(x)
            io["pos"].copy_(pos)
            io["slots"].copy_(table.gather(1, (pos.long() // BS)[:, None])[:, 0].long() * BS + pos.long() % BS)
            io["lens"].copy_(pos + 1)
        torch.cuda.synchronize()
        for g, _, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
        eager = step(*sides[2])
        torch.cuda.synchronize()
        for (g, out, _), (c, io) in zip(graphs, sides):
            assert torch.equal(out.view(torch.int16), eager.view(torch.int16)), t
            for a, b in zip(c, sides[2][0]):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    for _, io in sides:
        ops.check_status(io["st"])


def _runtime(dev, dtype, seed=0, layers=2, max_batch=8):
    from connex_b200.models.llama import LlamaConfig
    from connex_b200.runtime.pp import StageRuntime
    cfg = LlamaConfig.tiny(layers=2)
    return cfg, StageRuntime(cfg, 0, layers, dev, num_blocks=128, max_tokens=512, max_batch=max_batch, max_ctx=512,
                             seed=seed, kv_dtype=dtype)


def _compute(rt, kind, rids, ctx, n_new, ids, n_dec=None):
    from connex.pp.handover import CX_CTX, REQUEST_IDS
    td = {"kind": kind, REQUEST_IDS: rids, CX_CTX: ctx, "n_new": n_new,
          "ids": torch.tensor(ids, dtype=torch.int32, device=rt.device)}
    if n_dec is not None:
        td["n_dec"] = n_dec
    out = rt.compute(td, [])
    return out["x"].float() if "x" in out else out["next"]


def test_stage_runtime_8_bit(dev):
    """A stage of the model over an 8-bit cache: residual rows near those of the
    bf16 cache, whole or chunked prompt, decode rows in the same steps."""
    g = torch.Generator().manual_seed(3)
    prompt = torch.randint(3, 1000, (200,), generator=g).tolist()
    got = {}
    for dtype in (torch.bfloat16, torch.float8_e4m3fn):
        _, rt = _runtime(dev, dtype, layers=1)
        whole = _compute(rt, "prefill", ["w"], [0], [200], prompt)
        parts, done = [], 0
        for n in (16, 1, 50, 133):
            parts.append(_compute(rt, "mixed", ["c"], [done], [n], prompt[done:done + n], n_dec=1 if n == 1 else 0))
            done += n
        dec = _compute(rt, "decode", ["w", "c"], [200, 200], [1, 1], [5, 5])
        mix = _compute(rt, "mixed", ["w", "d"], [201, 0], [1, 40], [7] + prompt[:40], n_dec=1)
        torch.cuda.synchronize()
        assert int(rt.model.status) == 0
        got[dtype] = (whole, torch.cat(parts), dec, mix)
    a, b = got[torch.bfloat16], got[torch.float8_e4m3fn]
    # the attention's share of the residual changes by at most e4m3's 2^-4 of it (K and V); the random
    # weights' attention output is a small part of the rows
    for x, y in zip(a, b):
        assert (x - y).norm() <= 2.0 ** -4 * x.norm()
    w, c, dec, _ = b
    assert (w - c).norm() <= 2.0 ** -6 * w.norm()          # only rows of shared blocks were scaled twice
    assert (dec[0] - dec[1]).norm() <= 2.0 ** -6 * dec[0].norm()


def test_decode_graphs_and_fork_8_bit(dev):
    """Decode graphs (padding rows on one trash slot) give the eager rows; forked
    requests continue like their parent, before and after a compaction."""
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(3, 1000, (n,), generator=g).tolist() for n in (37, 16, 90)]
    outs = []
    for graphs in (False, True):
        cfg, rt = _runtime(dev, torch.float8_e4m3fn)
        if graphs:
            rt.enable_decode_graphs((4, 8))
        _compute(rt, "prefill", ["a", "b", "c"], [0] * 3, [len(p) for p in prompts], sum(prompts, []))
        lens, steps = [len(p) for p in prompts], []
        for t in range(20):
            steps.append(_compute(rt, "decode", ["a", "b", "c"], lens, [1] * 3, [7 + t, 9 + t, 11 + t]).tolist())
            lens = [n + 1 for n in lens]
        rt.fork("a", ["x", "y"])
        assert rt.held["x"] == lens[0] and rt.tables["x"][0] == rt.tables["a"][0]
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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_fork_that_goes_back_leaves_its_parent_alone(dev, dtype):
    """A forked request continued from before its shared blocks' end, with other tokens: the parent's cached
    rows keep their bytes, and the child's step equals one of a request that shares nothing."""
    g = torch.Generator().manual_seed(6)
    prompt = torch.randint(3, 1000, (50,), generator=g).tolist()
    other = torch.randint(3, 1000, (9,), generator=g).tolist()
    cfg, rt = _runtime(dev, dtype)
    _compute(rt, "prefill", ["a", "z"], [0, 0], [50, 50], prompt * 2)
    rt.fork("a", ["x"])
    raw = torch.uint8 if rt.cache.scales is not None else torch.int16

    def rows(rid):
        ids = torch.tensor(rt.tables[rid][:3], device=dev)
        parts = [rt.cache.kv[:, :, ids].view(raw)]
        return parts + ([rt.cache.scales[:, :, ids]] if rt.cache.scales is not None else [])
    before = rows("a")
    got = _compute(rt, "mixed", ["x", "z"], [20, 20], [9, 9], other * 2, n_dec=0).tolist()
    assert got[0] == got[1]
    assert all(torch.equal(p, q) for p, q in zip(rows("a"), before))
    assert rt.tables["x"][0] == rt.tables["a"][0] and rt.tables["x"][1] != rt.tables["a"][1]
    assert int(rt.model.status) == 0
    rt.release(["a", "x", "z"])
    assert rt.cache.free_blocks == 128 and not rt.cache._shared


def test_model_stepper_8_bit(dev):
    """The serving engine's stepper over an 8-bit cache: prefill, chunked prefill and decode agree."""
    from connex_b200.models.llama import LlamaConfig
    from connex_b200.serve.engine import ModelStepper
    st = ModelStepper(LlamaConfig.tiny(), dev, 96, max_batch=4, max_ctx=256, max_step_tokens=256, kv_dtype="fp8")
    seq = list(range(3, 80))
    a = st.prefill(["p"], [seq])
    b = st.mixed(["q"], [seq], [0], [64])
    b = st.mixed(["q"], [seq], [64], [13])
    assert a == b
    d1 = st.decode(["p", "q"], [seq + a, seq + a])
    assert d1[0] == d1[1]
    st.release(["p", "q"])


def test_qwen3_moe_rank_8_bit(dev):
    """Decode steps with q/k norms: layer 0 holds the bf16 cache's rows to half an e4m3 step (its input does not
    depend on the cache), and each step's attention is that of the cache it left."""
    from connex_b200 import ops
    from connex_b200.models.qwen3_moe import Qwen3MoeConfig, Qwen3MoeRank
    from connex_b200.ops import reference as R

    class NoExperts:
        def forward(self, h, idx, w, l2p, cnt, out):
            return out.zero_()
    cfg, B, steps = Qwen3MoeConfig.tiny(), 3, 37
    lens0 = [0, 5, 16]
    width = 4
    table = torch.randperm(B * width, generator=_g(dev, 171), device=dev).to(torch.int32).view(B, width)
    ids = torch.randint(3, 1000, (steps, B), generator=_g(dev, 172), device=dev).to(torch.int32)
    none = [(None, None)] * cfg.layers
    models = {}
    for dtype in (torch.bfloat16, torch.float8_e4m3fn):
        m = models[dtype] = Qwen3MoeRank(cfg, 0, 1, [[-1]] * cfg.layers, dev, B * width, B, kv_dtype=dtype)
        m.moe = NoExperts()
        for a in m.attn:
            a.q_norm.uniform_(0.5, 1.5, generator=_g(dev, 173))
            a.k_norm.uniform_(0.5, 1.5, generator=_g(dev, 174))
        # rows before the first step: zeros in both
        m.cache.kv.view(torch.int16 if dtype == torch.bfloat16 else torch.uint8).zero_()
        ws = (ops.decode_workspace(B, cfg.heads, width * BS, dev) if dtype == torch.bfloat16
              else ops.decode_workspace_fp8(B, cfg.heads, cfg.kv_heads, dev))
        for t in range(steps):
            pos = torch.tensor([n + t for n in lens0], dtype=torch.int32, device=dev)
            slots = table.gather(1, (pos.long() // BS)[:, None])[:, 0].long() * BS + pos.long() % BS
            m.decode(ids[t], pos, slots, table, pos + 1, width * BS, ws, none, none, none)
            if dtype == torch.float8_e4m3fn and t % 9 == 0:
                c, l = m.cache, cfg.layers - 1
                q = m.qkv[:, :cfg.heads * D].reshape(B, cfg.heads, D)
                ctx = [n + t for n in lens0]
                args = (c.k(l), c.v(l), c.k_scale(l), c.v_scale(l), table, ctx, [1] * B)
                ref, mag = R.paged_attention_fp8(q, *args)
                tol = _attention_tolerance(ref, mag, q, c.k(l), c.k_scale(l), table, ctx, [1] * B, U_F16,
                                           float(c.v_scale(l).max()) * 448)
                assert ((m.att.view(B, cfg.heads, D).double() - ref).abs() <= tol).all()
        ops.check_status(m.status)
    a, b = models[torch.bfloat16].cache, models[torch.float8_e4m3fn].cache
    for x, y, s, turned in ((a.k(0), b.k(0), b.k_scale(0), True), (a.v(0), b.v(0), b.v_scale(0), False)):
        x = x.double()
        # K: both writes round the normed pair to bf16, each to 2^-8 of it, and the rotated elements again; the
        # pair's two magnitudes add up to at most sqrt(2) of its length
        pair = torch.hypot(x[..., :D // 2], x[..., D // 2:]).repeat(1, 1, 1, 2) * math.sqrt(2) * (1 + 2 * U_BF16)
        d = 2 * U_BF16 * (x.abs() + pair) if turned else torch.zeros_like(x)
        # a row is rounded when it arrives and once more for each later growth of its block's scale, each of
        # which at least doubles it: halves of the smallest step, 2^-10 (1 + 1/2 + 1/4 + ..) of the last scale
        bound = d + U_E4M3 * (x.abs() + d) + 2 * 2.0 ** -10 * s.double()[..., None, None]
        assert ((R.fp8_values(y, s) - x).abs() <= bound).all()


def test_push_moves_an_8_bit_cache_in_two_calls(dev):
    """kv_push_layer takes the values by head slices of 2 KB and the scales as one 16-byte unit per block."""
    from connex_b200 import ops
    nb, hkv = 12, 4
    k, ks = _cache(nb, hkv, dev, 111)
    v, vs = _cache(nb, hkv, dev, 112)
    dst = [torch.zeros_like(t) for t in (k, v, ks, vs)]
    pairs = torch.tensor([[3, 7], [5, 1]], dtype=torch.int32, device=dev)
    ops.kv_push_layer(k.data_ptr(), v.data_ptr(), dst[0].data_ptr(), dst[1].data_ptr(), pairs, src_heads=hkv,
                      dst_heads=hkv, chunk_bytes=BS * D, src_blocks=nb, dst_blocks=nb)
    ops.kv_push_layer(ks.data_ptr(), vs.data_ptr(), dst[2].data_ptr(), dst[3].data_ptr(), pairs, src_heads=1,
                      dst_heads=1, chunk_bytes=4 * hkv, src_blocks=nb, dst_blocks=nb)
    for s, d in ((3, 7), (5, 1)):
        for a, b in zip((k, v, ks, vs), dst):
            assert torch.equal(a[s].view(torch.uint8), b[d].view(torch.uint8))
