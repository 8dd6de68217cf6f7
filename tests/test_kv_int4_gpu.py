"""The 4-bit paged KV cache on the GPU: the quantising write, its values, decode
and chunked prefill attention over it, each against a plain 64-bit statement.

Tolerances.  One rounding to a type t is off by at most eps(t) / 2 of the
value: bf16 2^-8, f16 2^-11, fp32 2^-24."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

D, BS, ROW = 128, 16, 72
U_BF16, U_F16, U_F32 = 2.0 ** -8, 2.0 ** -11, 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def _g(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _cache(nb, hkv, dev, seed, spread=0):
    """Random rows; with ``spread``, halves whose sizes differ by up to 2^spread."""
    from connex_b200.ops import reference as R
    g = _g(dev, seed)
    x = torch.randn(nb, hkv, BS, 2, D // 2, generator=g, device=dev) + torch.randn(hkv, 1, 2, D // 2, generator=g, device=dev)
    x = x * torch.exp2(torch.rand(nb, hkv, BS, 2, 1, generator=g, device=dev) * spread - spread / 2)
    return R.int4_rows(x.flatten(-2).to(torch.bfloat16))


def _nan_rows(cache, table, lens):
    """Cache rows behind each sequence's last token hold NaN scales and minima."""
    for b, n in enumerate(lens):
        if n % BS:
            cache[int(table[b, n // BS]), :, n % BS:] = 0xFF
        elif n == 0:
            cache[int(table[b, 0])] = 0x7F


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


def _attention_tolerance(ref, mag, q, k_cache, v_cache, table, ctx, n_new, u_weight, u_kv=0.0):
    """|out - ref| <= bf16 of the result + the weights' rounding (u_weight, and f16's smallest half step of the largest
    scale for each) + the logits' error: fp32 sums of 128 products of q with code * scale and with the minimum,
    16 times the size of a value at most each, and u_kv of each value where it is rounded.  Twice: weight and sum.
    V's product, too, adds up code * scale and the minimum's part by themselves: sums of at most 16 times |v|'s."""
    from connex_b200.ops import reference as R
    big, scales, s = 0.0, 0.0, 0
    hkv = k_cache.shape[1]
    span = torch.zeros_like(ref)
    for b, (c, n) in enumerate(zip(ctx, n_new)):
        if c + n and n:
            ids = table[b, :-(-(c + n) // BS)].long()
            par = [x[ids].transpose(0, 1).reshape(hkv, -1, ROW)[:, :c + n, 64:].contiguous().view(torch.bfloat16).double()
                   for x in (k_cache, v_cache)]
            size = [(15 * p[..., 0::2] + p[..., 1::2].abs()).nan_to_num(0.0).repeat_interleave(64, -1) for p in par]
            k = size[0].repeat_interleave(q.shape[1] // hkv, 0)
            big = max(big, (q[s:s + n].double().abs().transpose(0, 1) @ k.transpose(1, 2)).max().item() / math.sqrt(D))
            scales = max(scales, par[1][..., 0::2].nan_to_num(0.0).max().item())
            span[s:s + n] = size[1].amax(1).repeat_interleave(q.shape[1] // hkv, 0)
        s += n
    logit = big * (D * U_F32 + u_kv)
    n = max([c + m for c, m in zip(ctx, n_new)] + [1])
    return (U_BF16 * ref.abs() + (mag + span) * (2 * u_weight + u_kv + 4 * logit + n * U_F32 + 2.0 ** -20)
            + n * 2.0 ** -25 * 15 * scales)


DECODE_LENS = [[1], [0, 5, 0], [16], [17, 1, 15, 16, 31, 33], [500], [4096, 3, 0, 1000], [129] * 70, [20000, 1],
               [128] * 64, [1500] * 40 + [0, 1480]]


@pytest.mark.parametrize("spread", [0, 12])
@pytest.mark.parametrize("heads", [(32, 8), (8, 8), (6, 2), (7, 1), (16, 1), (20, 2), (32, 4)])
@pytest.mark.parametrize("lens", DECODE_LENS, ids=lambda v: f"{len(v)}x{max(v)}")
def test_decode_attention(dev, heads, lens, spread):
    from connex_b200 import ops
    from connex_b200.ops import reference as R
    hq, hkv = heads
    table, nb = _table(lens, dev, 1)
    k, v = _cache(nb, hkv, dev, 2), _cache(nb, hkv, dev, 3, spread)
    _nan_rows(k, table, lens)
    _nan_rows(v, table, lens)
    B = len(lens)
    # q as a slice of wider rows, as the fused projection leaves it
    wide = torch.randn(B, (hq + 2) * D, generator=_g(dev, 4), device=dev).to(torch.bfloat16)
    q = wide[:, :hq * D]
    st = ops.new_status(dev)
    ws = ops.decode_workspace_int4(B, hq, hkv, dev)
    lt = torch.tensor(lens, dtype=torch.int32, device=dev)
    out = ops.decode_attention_int4(wide, k, v, table, lt, hq, ws, status=st)
    torch.cuda.synchronize()
    ops.check_status(st, "decode_attention_int4")
    ctx = [n - 1 for n in lens if n]
    live = torch.tensor([n > 0 for n in lens], device=dev)
    got = out.view(B, hq, D).double()
    assert torch.equal(got[~live], torch.zeros_like(got[~live]))
    rows, tl = q.reshape(B, hq, D)[live], table[live]
    ref, mag = R.paged_attention_int4(rows, k, v, tl, ctx, [1] * len(ctx))
    tol = _attention_tolerance(ref, mag, rows, k, v, tl, ctx, [1] * len(ctx), U_F16)
    assert ((got[live] - ref).abs() <= tol).all(), float(((got[live] - ref).abs() / tol).max())
    # most of that is room: on the whole the result is as good as its rounding to bf16 and the weights' to f16
    assert (got[live] - ref).norm() <= (U_BF16 + 2 * U_F16) * ref.norm()
    # the workspace is left ready: the same call again, the same bits
    again = ops.decode_attention_int4(wide, k, v, table, lt, hq, ws)
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
    k, v = _cache(nb, hkv, dev, 6), _cache(nb, hkv, dev, 7, 4)
    _nan_rows(k, table, lens)
    _nan_rows(v, table, lens)
    T = sum(new)
    q = torch.randn(T, hq * D, generator=_g(dev, 8), device=dev).to(torch.bfloat16)
    st = ops.new_status(dev)
    ti = ops.prefill_tile_info(new, dev, ctx=ctx)
    out = ops.prefill_attention_paged_int4(q, k, v, table, ti, hq, hkv, status=st)
    torch.cuda.synchronize()
    ops.check_status(st, "prefill_attention_paged_int4")
    ref, mag = R.paged_attention_int4(q.view(T, hq, D), k, v, table, ctx, new)
    tol = _attention_tolerance(ref, mag, q.view(T, hq, D), k, v, table, ctx, new, U_BF16, U_BF16)
    err = (out.view(T, hq, D).double() - ref).abs()
    assert (err <= tol).all(), float((err / tol).max())
    assert (out.view(T, hq, D).double() - ref).norm() <= 4 * U_BF16 * ref.norm()


def _write_case(dev, rows, hq, hkv, seed, norm=False):
    from connex_b200 import ops
    lens = [c + n for c, n in rows]
    table, nb = _table(lens, dev, seed)
    pos, slots = [], []
    for b, (c, n) in enumerate(rows):
        for p in range(c, c + n):
            pos.append(p)
            slots.append(int(table[b, p // BS]) * BS + p % BS)
    g = _g(dev, seed + 3)
    mag = torch.exp2(torch.rand(hq + 2 * hkv, 1, generator=g, device=dev) * 8 - 4)
    qkv = (torch.randn(len(pos), hq + 2 * hkv, D, generator=g, device=dev) * mag).to(torch.bfloat16).view(len(pos), -1)
    w = [(torch.rand(D, generator=g, device=dev) + 0.5).to(torch.bfloat16) for _ in range(2)] if norm else [None, None]
    cs = ops.rope_cos_sin(max(lens) + 1, D, 5e5, dev)
    return dict(k=_cache(nb, hkv, dev, seed + 1), v=_cache(nb, hkv, dev, seed + 2), nb=nb,
                pos=torch.tensor(pos, dtype=torch.int32, device=dev),
                slots=torch.tensor(slots, dtype=torch.int64, device=dev), qkv=qkv, cs=cs, qn=w[0], kn=w[1])


def _turned(x, pos, cs, w):
    """Rotated rows in 64 bits, and a bound on what a flip of the norm's bf16 rounding moves them."""
    x = x.double()
    slack = torch.zeros_like(x)
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.double()
        x = x.to(torch.bfloat16).double()
        slack = 2 * U_BF16 * (x.abs() + x.abs().roll(D // 2, -1))
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
    before = {n: s[n].clone() for n in ("k", "v", "qkv")}
    st = ops.new_status(dev)
    q = ops.rope_cache_int4(s["qkv"], s["pos"], s["cs"], hq, hkv, s["slots"], s["k"], s["v"], status=st, q_norm=s["qn"],
                            k_norm=s["kn"])
    torch.cuda.synchronize()
    ops.check_status(st, "rope_cache_int4")
    assert torch.equal(s["qkv"], before["qkv"])
    ref, slack = _turned(x[:, :hq], s["pos"], s["cs"], s["qn"])
    assert ((q.view(T, hq, D).double() - ref).abs() <= U_BF16 * ref.abs() + 2 * slack).all()
    # rows that the call did not write stay as they are
    blk, off = s["slots"] // BS, s["slots"] % BS
    kept = torch.ones(s["nb"], BS, dtype=torch.bool, device=dev)
    kept[blk, off] = False
    for n in ("k", "v"):
        assert torch.equal(s[n].transpose(1, 2)[kept], before[n].transpose(1, 2)[kept])
    # v is quantised as it stands.  Minimum and scale to the bit; a code may differ where (x - min) / scale lies between
    # two whole numbers, by the roundings of the difference, the reciprocal and the product: 15 * 3 * 2^-24 of a step
    got, want = s["v"][blk, :, off], R.int4_rows(x[:, hq + hkv:])
    assert torch.equal(got[..., 64:], want[..., 64:])
    _codes_hold(got, x[:, hq + hkv:].double(), torch.zeros(T, hkv, D, dtype=torch.float64, device=dev))
    # k: its minimum and range are those of the rotated rows, rounded to bf16
    kr, ks = _turned(x[:, hq:hq + hkv], s["pos"], s["cs"], s["kn"])
    _codes_hold(s["k"][blk, :, off], kr, U_BF16 * kr.abs() + 2 * ks)


def _codes_hold(rows, x, slack):
    """Cached ``rows`` hold ``x`` (known to within ``slack``): the minimum, the scale (of bf16), each value to half a step."""
    from connex_b200.ops import reference as R
    par = rows[..., 64:].contiguous().view(torch.bfloat16).double()
    scale, low = par[..., 0::2], par[..., 1::2]
    h, e = x.unflatten(-1, (2, 64)), slack.unflatten(-1, (2, 64)).amax(-1)
    assert ((low - h.amin(-1)).abs() <= e).all()
    span = h.amax(-1) - h.amin(-1)
    assert ((scale * 15 - span).abs() <= U_BF16 * span * (1 + U_BF16) + 2 * e * (1 + U_BF16)).all()
    # half a step; at the top up to 15 times the scale's rounding more, the code 15 being the last
    step = span / 15
    tol = (0.5 + 15 * U_BF16 + 2.0 ** -18) * step + 4 * e
    assert ((R.int4_values(rows).unflatten(-1, (2, 64)) - h).abs() <= tol[..., None]).all()


def test_values(dev):
    from connex_b200 import ops
    from connex_b200.ops import reference as R
    for shape in ((1,), (3, 2), (40, 4, 16), (5000, 1)):
        x = torch.randn(*shape, D, generator=_g(dev, 21), device=dev).to(torch.bfloat16)
        rows = R.int4_rows(x)
        out = ops.kv_values_int4(rows)
        ref = R.int4_values(rows)
        # code * scale and the sum in fp32 (minimum + code * scale: up to 16 times the value's own size), then bf16
        par = rows[..., 64:].contiguous().view(torch.bfloat16).double()
        size = (par[..., 1::2].abs() + 15 * par[..., 0::2]).repeat_interleave(64, -1)
        assert ((out.double() - ref).abs() <= U_BF16 * ref.abs() + 2 * U_F32 * size).all()
    assert ops.kv_values_int4(torch.empty(0, 3, ROW, dtype=torch.uint8, device=dev)).shape == (0, 3, D)


def test_write_out_of_range(dev):
    """Bad slots and positions are recorded, cached nowhere, and change nothing else; slots below zero are skipped."""
    from connex_b200 import ops
    from connex_b200.ops import reference as R
    hq, hkv, nb = 4, 2, 6
    cs = ops.rope_cos_sin(64, D, 1e4, dev)
    for slots, pos in (([nb * BS, 0], [0, 1]), ([0, 16], [64, 1]), ([0, 1], [3, -1]), ([1 << 40, 5], [0, 0]),
                       ([-1, 17], [1, 2]), ([-7, -1 << 50], [1, 2])):
        k, v = _cache(nb, hkv, dev, 31), _cache(nb, hkv, dev, 32)
        k0, v0 = k.clone(), v.clone()
        good = [0 <= s < nb * BS and 0 <= p < 64 for s, p in zip(slots, pos)]
        qkv = torch.randn(2, (hq + 2 * hkv) * D, generator=_g(dev, 33), device=dev).to(torch.bfloat16)
        st = ops.new_status(dev)
        q = ops.rope_cache_int4(qkv, torch.tensor(pos, dtype=torch.int32, device=dev), cs, hq, hkv,
                                torch.tensor(slots, dtype=torch.int64, device=dev), k, v, status=st)
        if all(g or s < 0 for g, s in zip(good, slots)):
            ops.check_status(st)
        else:
            with pytest.raises(RuntimeError, match="bounds"):
                ops.check_status(st)
        assert torch.isfinite(q.float()).all()
        for i, (s, g) in enumerate(zip(slots, good)):
            if g:
                R.int4_append(v0, qkv.view(2, -1, D)[i:i + 1, hq + hkv:], torch.tensor([s], device=dev))
                k0[s // BS, :, s % BS] = k[s // BS, :, s % BS]
            if not 0 <= pos[i] < 64:
                assert not q[i].any()
        assert torch.equal(k, k0) and torch.equal(v[..., 64:], v0[..., 64:])
        assert ((R.int4_values(v) - R.int4_values(v0)).abs().nan_to_num(0.0) <= 0.5).all()


def test_write_special_values(dev):
    """A half with NaN or infinities reads as NaN, the other one stays; constants, tiny and huge values."""
    from connex_b200 import ops
    hq, hkv, nb = 2, 1, 5
    k, v = _cache(nb, hkv, dev, 41), _cache(nb, hkv, dev, 42)
    top = torch.finfo(torch.bfloat16).max
    qkv = torch.zeros(5, (hq + 2 * hkv) * D, device=dev, dtype=torch.bfloat16)
    rows = qkv[:, -D:]
    rows[0] = 3.0                                  # a constant: the minimum itself
    rows[0, 3] = float("inf")
    rows[1, 64:] = 7.0
    rows[1, 64 + 9] = float("nan")
    rows[2, :64] = torch.arange(64, device=dev).to(torch.bfloat16) * 2.0 ** -130
    rows[2, 64:] = top
    rows[2, 70] = 0.0                              # a range of the largest number
    rows[3, :32] = top
    rows[3, 32:64] = -top                          # a range beyond fp32
    rows[4, 64:] = -5.0
    i32 = torch.arange(5, dtype=torch.int32, device=dev)
    ops.rope_cache_int4(qkv, i32, ops.rope_cos_sin(64, D, 1e4, dev), hq, hkv, torch.arange(5, device=dev) * BS, k, v)
    val = ops.kv_values_int4(v)[:, 0, 0].float()
    assert torch.isnan(val[0, :64]).all() and (val[0, 64:] == 3.0).all()
    assert (val[1, :64] == 0).all() and torch.isnan(val[1, 64:]).all()
    assert ((val[2, :64] - rows[2, :64].float()).abs() <= 2.2 * 2.0 ** -130).all()
    assert (val[2, 64:] >= top * 0.99).sum() == 63 and val[2, 70] == 0
    assert torch.isnan(val[3, :64]).all() and (val[3, 64:] == 0).all()
    assert (val[4, :64] == 0).all() and (val[4, 64:] == -5.0).all()
    assert (ops.kv_values_int4(k)[:, 0, 0] == 0).all()


def test_write_in_place(dev):
    """out as qkv's own q columns gives the same q."""
    from connex_b200 import ops
    s = _write_case(dev, [(0, 40), (9, 3)], 6, 2, 61)
    a = ops.rope_cache_int4(s["qkv"], s["pos"], s["cs"], 6, 2, s["slots"], s["k"], s["v"])
    ops.rope_cache_int4(s["qkv"], s["pos"], s["cs"], 6, 2, s["slots"], s["k"], s["v"], out=s["qkv"][:, :6 * D])
    assert torch.equal(s["qkv"][:, :6 * D], a)


def test_decode_bad_pages_and_lengths(dev):
    """A block id out of range is left out, a length beyond the table cut; both recorded."""
    from connex_b200 import ops
    from connex_b200.ops import reference as R
    hq, hkv = 8, 2
    k, v = _cache(20, hkv, dev, 91), _cache(20, hkv, dev, 92)
    q = torch.randn(2, hq * D, generator=_g(dev, 93), device=dev).to(torch.bfloat16)
    ws = ops.decode_workspace_int4(2, hq, hkv, dev)
    i = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    for table, lens, like in (([[3, 20, 5], [1, 2, 4]], [48, 48], ([[3, 5, 5], [1, 2, 4]], [32, 48])),
                              ([[3, -5, 5], [1, 2, 4]], [48, 20], ([[3, 5, 5], [1, 2, 4]], [32, 20])),
                              ([[3, 2**31 - 1, -2**31], [1, 2, 4]], [48, 20], ([[3, 5, 5], [1, 2, 4]], [16, 20])),
                              ([[3, 4, 5], [1, 2, 6]], [49, -3], ([[3, 4, 5], [1, 2, 6]], [48, 0]))):
        st = ops.new_status(dev)
        out = ops.decode_attention_int4(q, k, v, i(table), i(lens), hq, ws, status=st)
        with pytest.raises(RuntimeError, match="bounds"):
            ops.check_status(st)
        t, n = like
        ref, mag = R.paged_attention_int4(q.view(2, hq, D), k, v, i(t), [x - 1 if x else 0 for x in n], [1, 1])
        for b in range(2):
            if n[b] == 0:
                assert not out[b].any()
            else:
                err = (out[b].view(hq, D).double() - ref[b]).abs()
                assert (err <= U_BF16 * ref[b].abs() + (mag[b] + 8) * 2.0 ** -9 + 1e-6).all()
    # no block at all: zeros
    st = ops.new_status(dev)
    assert not ops.decode_attention_int4(q, k, v, i([[-1, 99]] * 2), i([32, 7]), hq, ws, status=st).any()


def test_prefill_bad_pages_and_tiles(dev):
    """A block id out of range reads as zeros; a tile that fits neither the rows nor the tables is left out."""
    from connex_b200 import ops
    hq, hkv, nb = 4, 2, 12
    k, v = _cache(nb, hkv, dev, 121), _cache(nb, hkv, dev, 122)
    q = torch.randn(40, hq * D, generator=_g(dev, 123), device=dev).to(torch.bfloat16)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    table = i32([[3, 4, 1], [5, 6, 2]])
    good = [(0, 20, 0, 28, 0), (20, 20, 0, 10, 1)]
    st = ops.new_status(dev)
    ref = ops.prefill_attention_paged_int4(q, k, v, table, i32(good), hq, hkv, status=st, n_blocks=5)
    ops.check_status(st)
    for bad in ((20, 20, 0, 29, 1), (21, 20, 0, 10, 1), (20, 20, 0, 10, 2), (20, 20, 0, 2**31 - 1, 1)):
        st = ops.new_status(dev)
        out = torch.full_like(ref, 7.0)
        ops.prefill_attention_paged_int4(q, k, v, table, i32([good[0], bad]), hq, hkv, out=out, status=st)
        with pytest.raises(RuntimeError, match="bounds"):
            ops.check_status(st)
        assert torch.equal(out[:20], ref[:20]) and (out[20:] == 7.0).all()
    for bad in (nb, -1, 2**31 - 1):
        st = ops.new_status(dev)
        t = table.clone()
        t[1, 1] = bad
        out = ops.prefill_attention_paged_int4(q, k, v, t, i32(good), hq, hkv, status=st)
        with pytest.raises(RuntimeError, match="bounds"):
            ops.check_status(st)
        k0, v0 = k.clone(), v.clone()
        k0[6] = v0[6] = 0
        want = ops.prefill_attention_paged_int4(q, k0, v0, table, i32(good), hq, hkv)
        assert torch.equal(out, want)


def test_decode_nan_and_extreme_sizes(dev):
    """A NaN key poisons its own head only; logits far apart, q's and v's of any size stay exact enough."""
    from connex_b200 import ops
    from connex_b200.ops import reference as R
    hq, hkv = 4, 2
    table, nb = _table([100, 60], dev, 101)
    k = _cache(nb, hkv, dev, 102)
    ws = ops.decode_workspace_int4(2, hq, hkv, dev)
    lens = torch.tensor([100, 60], dtype=torch.int32, device=dev)
    for size, vsize in ((1e-30, 1.0), (1e-3, 1e-30), (100.0, 1e30), (1e37, 1.0), (1.0, 1e-37)):
        v = R.int4_rows((torch.randn(nb, hkv, BS, D, generator=_g(dev, 103), device=dev) * vsize).to(torch.bfloat16))
        q = (torch.randn(2, hq * D, generator=_g(dev, 104), device=dev) * size).to(torch.bfloat16)
        out = ops.decode_attention_int4(q, k, v, table, lens, hq, ws).view(2, hq, D).double()
        ref, mag = R.paged_attention_int4(q.view(2, hq, D), k, v, table, [99, 59], [1, 1])
        tol = _attention_tolerance(ref, mag, q.view(2, hq, D), k, v, table, [99, 59], [1, 1], U_F16)
        assert ((out - ref).abs() <= tol).all(), (size, vsize)
    v = _cache(nb, hkv, dev, 106)
    q = torch.randn(2, hq * D, generator=_g(dev, 105), device=dev).to(torch.bfloat16)
    # one half of a value row: only those dims
    v0 = v.clone()
    v0[table[1, 1].long(), 0, 3, 64:68] = 0xFF
    out = ops.decode_attention_int4(q, k, v0, table, lens, hq, ws).view(2, hq, D)
    bad = torch.isnan(out.float())
    assert bad[1, :2, :64].all() and int(bad.sum()) == 2 * 64
    assert torch.equal(out[~bad], ops.decode_attention_int4(q, k, v, table, lens, hq, ws).view(2, hq, D)[~bad])
    k[table[0, 2].long(), 1, 5, 64:] = 0x7F
    k[table[0, 2].long(), 1, 5, 65] = 0xFF
    k[table[0, 2].long(), 1, 5, 67] = 0xFF
    out = ops.decode_attention_int4(q, k, v, table, lens, hq, ws).view(2, hq, D)
    assert torch.isnan(out[0, 2:].float()).all()
    assert torch.isfinite(out[0, :2].float()).all() and torch.isfinite(out[1].float()).all()


def test_constant_values(dev):
    """Values whose scale is zero (every element of a half the same) are their minimum."""
    from connex_b200 import ops
    from connex_b200.ops import reference as R
    hq, hkv = 8, 2
    table, nb = _table([70, 3000], dev, 111)
    k = _cache(nb, hkv, dev, 112)
    v = R.int4_rows(torch.full((nb, hkv, BS, D), -2.5, dtype=torch.bfloat16, device=dev))
    q = torch.randn(2, hq * D, generator=_g(dev, 113), device=dev).to(torch.bfloat16)
    out = ops.decode_attention_int4(q, k, v, table, torch.tensor([70, 3000], dtype=torch.int32, device=dev), hq,
                                    ops.decode_workspace_int4(2, hq, hkv, dev))
    assert ((out.float() + 2.5).abs() <= 2.5 * U_BF16).all()


def test_empty_calls(dev):
    """No rows, no sequences, no tiles, no table: nothing is written and nothing fails."""
    from connex_b200 import ops
    hq, hkv, nb = 8, 2, 6
    k, v = _cache(nb, hkv, dev, 131), _cache(nb, hkv, dev, 132)
    was = [t.clone() for t in (k, v)]
    i32 = lambda *n: torch.zeros(*n, dtype=torch.int32, device=dev)  # noqa: E731
    st = ops.new_status(dev)
    qkv = torch.zeros(0, (hq + 2 * hkv) * D, dtype=torch.bfloat16, device=dev)
    out = ops.rope_cache_int4(qkv, i32(0), ops.rope_cos_sin(64, D, 5e5, dev), hq, hkv,
                              torch.zeros(0, dtype=torch.int64, device=dev), k, v, status=st)
    assert out.shape == (0, hq * D)
    ws = ops.decode_workspace_int4(3, hq, hkv, dev)
    q = torch.ones(3, hq * D, dtype=torch.bfloat16, device=dev)
    assert ops.decode_attention_int4(q[:0], k, v, i32(0, 4), i32(0), hq, ws, status=st).shape == (0, hq * D)
    assert (ops.decode_attention_int4(q, k, v, i32(3, 0), i32(3), hq, ws, status=st) == 0).all()
    tiles = torch.tensor([[0, 3, 0, 0, 0]], dtype=torch.int32, device=dev)
    ops.prefill_attention_paged_int4(q[:0], k, v, i32(1, 4), tiles, hq, hkv, status=st)
    kept = torch.full((3, hq * D), 7.0, dtype=torch.bfloat16, device=dev)
    ops.prefill_attention_paged_int4(q, k, v, i32(1, 4), tiles[:0], hq, hkv, out=kept, status=st)
    assert (kept == 7.0).all()
    with pytest.raises(RuntimeError, match="no block table"):
        ops.prefill_attention_paged_int4(q, k, v, i32(0, 4), tiles, hq, hkv, status=st)
    ops.check_status(st)
    assert torch.equal(k, was[0]) and torch.equal(v, was[1])
    assert (ops.decode_attention_int4(q, k, v, i32(3, 0), i32(3) + 5, hq, ws, status=st) == 0).all()
    with pytest.raises(RuntimeError, match="bounds"):
        ops.check_status(st)


def test_write_many_rows_as_few(dev):
    """Calls of many rows (another division of the work) and of few give the same bits."""
    from connex_b200 import ops
    for hq, hkv, T, norm in ((32, 8, 3000, False), (20, 4, 4100, True), (2, 1, 20000, False)):
        nb = -(-T // BS)
        qkv = torch.randn(T, (hq + 2 * hkv) * D, generator=_g(dev, 301), device=dev).to(torch.bfloat16)
        w = (torch.rand(D, generator=_g(dev, 302), device=dev) + 0.5).to(torch.bfloat16) if norm else None
        cs = ops.rope_cos_sin(T, D, 5e5, dev)
        pos, slots = torch.arange(T, dtype=torch.int32, device=dev), torch.randperm(T, generator=_g(dev, 303), device=dev)
        got = []
        for step in (T, 250):
            k, v = (torch.zeros(nb, hkv, BS, ROW, dtype=torch.uint8, device=dev) for _ in range(2))
            st = ops.new_status(dev)
            q = torch.cat([ops.rope_cache_int4(qkv[i:i + step], pos[i:i + step], cs, hq, hkv, slots[i:i + step], k, v,
                                               status=st, q_norm=w, k_norm=w) for i in range(0, T, step)])
            ops.check_status(st)
            got.append((q, k, v))
        assert all(torch.equal(a, b) for a, b in zip(*got))


def test_decode_workspace_for_any_batch(dev):
    """4096 sequences, then batches of other sizes and lengths with the same workspace, rows of a wider tensor, a
    negative scale: each as a call with a workspace of its own."""
    from connex_b200 import ops
    hq, hkv = 8, 2
    big = ops.decode_workspace_int4(4096, hq, hkv, dev)
    k, v = _cache(300, hkv, dev, 311), _cache(300, hkv, dev, 312)
    g = _g(dev, 313)
    for B, top in ((4096, 40), (3, 4000), (1, 1), (700, 300), (4096, 1), (64, 0), (2, 4800)):
        width = max(1, -(-top // BS))
        # blocks shared between sequences, some twice in a table
        table = torch.randint(0, 300, (B, width), generator=g, device=dev).to(torch.int32)
        lens = torch.randint(0, top + 1, (B,), generator=g, device=dev).to(torch.int32)
        lens[0] = top
        q = torch.randn(B, hq * D + 64, generator=g, device=dev).to(torch.bfloat16)
        st = ops.new_status(dev)
        out = ops.decode_attention_int4(q, k, v, table, lens, hq, big, status=st)
        own = ops.decode_attention_int4(q[:, :hq * D].contiguous(), k, v, table, lens, hq, ops.decode_workspace_int4(B, hq, hkv, dev))
        turned = ops.decode_attention_int4(-q, k, v, table, lens, hq, big, scale=-1 / math.sqrt(D), status=st)
        ops.check_status(st)
        assert torch.equal(out, own) and torch.equal(out, turned) and torch.isfinite(out).all()
        assert not out[lens == 0].any()
    with pytest.raises(RuntimeError, match="at most 4096 sequences"):
        ops.decode_attention_int4(torch.zeros(4097, hq * D, dtype=torch.bfloat16, device=dev), k, v,
                                  torch.zeros(4097, 1, dtype=torch.int32, device=dev),
                                  torch.zeros(4097, dtype=torch.int32, device=dev), hq, big)


def test_prefill_of_shared_blocks(dev):
    """Two prompts over the same blocks, one of them twice in a table: as over copies of the blocks."""
    from connex_b200 import ops
    hq, hkv, n = 8, 2, 40
    k, v = _cache(60, hkv, dev, 321), _cache(60, hkv, dev, 322)
    shared = torch.randint(0, 20, (2, n), generator=_g(dev, 323), device=dev).to(torch.int32)
    kc, vc = (x[shared.view(-1).long()].contiguous() for x in (k, v))
    apart = torch.arange(2 * n, dtype=torch.int32, device=dev).view(2, n)
    q = torch.randn(150 + 30, hq * D, generator=_g(dev, 324), device=dev).to(torch.bfloat16)
    ti = ops.prefill_tile_info([150, 30], dev, ctx=[490, 600])
    st = ops.new_status(dev)
    a = ops.prefill_attention_paged_int4(q, k, v, shared, ti, hq, hkv, status=st)
    b = ops.prefill_attention_paged_int4(q, kc, vc, apart, ti, hq, hkv, status=st)
    ops.check_status(st)
    assert torch.equal(a, b)
