"""Decode attention over the 4-bit cache where its numbers lie far apart: weights far below the largest, halves of V of
very different sizes, logits far from zero.  Against a 64-bit statement, with tolerances for each half by itself.

One rounding to a type t is off by at most eps(t) / 2 of the value: bf16 2^-8, f16 2^-11, fp32 2^-24."""
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


def _paged(rows, dev, seed):
    """Sequences' rows (bf16 [n, Hkv, D] each) in a 4-bit cache of shuffled blocks; (cache, table)."""
    from connex_b200.ops import reference as R
    need = [-(-len(r) // BS) for r in rows]
    perm = torch.randperm(sum(need) + 2, generator=_g(dev, seed), device=dev).to(torch.int32)
    cache = torch.full((sum(need) + 2, rows[0].shape[1], BS, ROW), 0xFF, dtype=torch.uint8, device=dev)
    table, at = torch.full((len(rows), max(need)), -1, dtype=torch.int32, device=dev), 0
    for b, (r, n) in enumerate(zip(rows, need)):
        table[b, :n] = perm[at:at + n]
        at += n
        p = torch.arange(len(r), device=dev)
        R.int4_append(cache, r, table[b].long()[p // BS] * BS + p % BS)
    return cache, table


def _check(out, q, k, v, table, lens, hkv):
    """bf16 of the result, twice f16 of each weight (weight and sum), fp32 sums of 128 products in the logits and of n in
    the result, with sizes of code * scale and of the minimum taken by themselves; and a weight times scale held to
    2^-33 of the half's largest at least, which is the largest scale's share at most."""
    from connex_b200.ops import reference as R
    hq = q.shape[1]
    ctx, one = [n - 1 for n in lens], [1] * len(lens)
    ref, mag = R.paged_attention_int4(q, k, v, table, ctx, one)
    size = v.clone()
    size[..., :64] = 0xFF
    size[..., 67] &= 0x7F
    size[..., 71] &= 0x7F
    span = R.paged_attention_int4(q, k, size, table, ctx, one)[0]       # sums of weight * (|minimum| + 15 scale)
    least, logit = torch.zeros_like(ref), torch.zeros(*ref.shape[:2], 1, dtype=torch.float64, device=q.device)
    for b, n in enumerate(lens):
        ids = table[b, :-(-n // BS)].long()
        kp, vp = (x[ids].transpose(0, 1).reshape(hkv, -1, ROW)[:, :n, 64:].contiguous().view(torch.bfloat16).double()
                  for x in (k, v))
        big = (15 * kp[..., 0::2] + kp[..., 1::2].abs()).amax(1).repeat_interleave(64, -1).repeat_interleave(hq // hkv, 0)
        logit[b, :, 0] = (q[b].double().abs() * big).sum(-1) / math.sqrt(D) * D * U_F32
        top = vp[..., 0::2].amax(1).repeat_interleave(64, -1).repeat_interleave(hq // hkv, 0)
        least[b] = n * 15 * 2.0 ** -33 * top
    n = max(lens)
    tol = U_BF16 * ref.abs() + (mag + span) * (2 * U_F16 + 4 * logit + n * U_F32 + 2.0 ** -20) + least
    err = (out.view(ref.shape).double() - ref).abs()
    assert (err <= tol).all(), float((err / tol).max())
    return ref


@pytest.mark.parametrize("heads", [(8, 2), (16, 1), (5, 1)])
@pytest.mark.parametrize("ratio", [-12, 0, 20])
@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("lens", [[5000, 3, 900], [2400] * 120], ids=["few", "many"])
def test_many_small_weights_beside_a_large_one(dev, heads, ratio, first, lens):
    """One token holds most of the weight, thousands have 2^-16 to 2^-22 of its weight each, some hundredths of it
    together; V's second half is 2^ratio of the first.  With many sequences a warp reads a pair to a quarter."""
    from connex_b200 import ops
    hq, hkv = heads
    rows_k, rows_v = [], []
    g = _g(dev, 1)
    for n in lens:
        # keys: one dim counts, its value is the logit; minimum and maximum of a half are stored exactly
        k = torch.zeros(n, hkv, D, device=dev)
        k[..., 0] = -math.log(2.0) * (16 + 6 * torch.rand(n, hkv, generator=g, device=dev) ** 2)
        k[0 if first else n - 1, :, 0] = 0
        v = torch.randn(n, hkv, D, generator=g, device=dev) + 2
        v[..., 64:] *= 2.0 ** ratio
        rows_k.append(k.to(torch.bfloat16)), rows_v.append(v.to(torch.bfloat16))
    k, table = _paged(rows_k, dev, 2)
    v, _ = _paged(rows_v, dev, 2)
    B = len(lens)
    q = torch.zeros(B, hq, D, dtype=torch.bfloat16, device=dev)
    q[..., 0] = math.sqrt(D)
    out = ops.decode_attention_int4(q.view(B, -1), k, v, table, torch.tensor(lens, dtype=torch.int32, device=dev), hq,
                                    ops.decode_workspace_int4(B, hq, hkv, dev))
    _check(out, q, k, v, table, lens, hkv)


@pytest.mark.parametrize("ratio", [-12, 24])
@pytest.mark.parametrize("n", [1, 40, 3000])
def test_halves_of_different_sizes(dev, ratio, n):
    from connex_b200 import ops
    hq, hkv = 12, 3
    k, table = _paged([torch.randn(n, hkv, D, generator=_g(dev, 3), device=dev).to(torch.bfloat16)], dev, 4)
    x = torch.randn(n, hkv, D, generator=_g(dev, 5), device=dev)
    x[..., 64:] *= 2.0 ** ratio
    v, _ = _paged([x.to(torch.bfloat16)], dev, 4)
    q = torch.randn(1, hq, D, generator=_g(dev, 6), device=dev).to(torch.bfloat16)
    out = ops.decode_attention_int4(q.view(1, -1), k, v, table, torch.tensor([n], dtype=torch.int32, device=dev), hq,
                                    ops.decode_workspace_int4(1, hq, hkv, dev))
    _check(out, q, k, v, table, [n], hkv)


@pytest.mark.parametrize("logit", [-400.0, -100.0, 100.0, 400.0])
@pytest.mark.parametrize("step", [0.0, 3.0])
@pytest.mark.parametrize("constant", [False, True])
def test_logits_far_from_zero(dev, logit, step, constant):
    """All logits near one number, rising by ``step`` from block to block; one half of V is a constant (its scale is
    zero), the other tiny, or a constant as well."""
    from connex_b200 import ops
    hq, hkv, n = 8, 2, 700
    kr = torch.zeros(n, hkv, D, device=dev)
    kr[..., 0] = logit + step * (torch.arange(n, device=dev) // BS)[:, None]
    k, table = _paged([kr.to(torch.bfloat16)], dev, 7)
    x = torch.randn(n, hkv, D, generator=_g(dev, 8), device=dev) * 2.0 ** -110
    x[..., :64] = -2.5
    if constant:
        x[..., 64:] = 7.0
    v, _ = _paged([x.to(torch.bfloat16)], dev, 7)
    q = torch.zeros(1, hq, D, dtype=torch.bfloat16, device=dev)
    q[..., 0] = math.sqrt(D)
    out = ops.decode_attention_int4(q.view(1, -1), k, v, table, torch.tensor([n], dtype=torch.int32, device=dev), hq,
                                    ops.decode_workspace_int4(1, hq, hkv, dev))
    _check(out, q, k, v, table, [n], hkv)
    assert ((out.view(hq, D)[:, :64].float() + 2.5).abs() <= 2.5 * U_BF16).all()


@pytest.mark.parametrize("bits", [0x7F80, 0x7F7F, 0x7F00])
@pytest.mark.parametrize("step", [0.0, 5.0])
def test_scales_that_no_write_leaves(dev, bits, step):
    """An infinite scale of V, the largest number and 2^127 in one half of one token: that half of its heads is not finite
    or the sum of what fp32 holds, everything else as without it."""
    from connex_b200 import ops
    hq, hkv, n = 8, 2, 300
    kr = torch.zeros(n, hkv, D, device=dev)
    kr[..., 0] = step * (torch.arange(n, device=dev) // 32)[:, None]
    k, table = _paged([kr.to(torch.bfloat16)], dev, 9)
    v, _ = _paged([torch.randn(n, hkv, D, generator=_g(dev, 10), device=dev).to(torch.bfloat16)], dev, 9)
    q = torch.zeros(1, hq, D, dtype=torch.bfloat16, device=dev)
    q[..., 0] = math.sqrt(D)
    lens = torch.tensor([n], dtype=torch.int32, device=dev)

    def call():
        return ops.decode_attention_int4(q.view(1, -1), k, v, table, lens, hq,
                                         ops.decode_workspace_int4(1, hq, hkv, dev)).view(hq, D)
    want = call()
    at = v[int(table[0, 250 // BS]), 1, 250 % BS]
    at[68], at[69] = bits & 0xFF, bits >> 8                      # the second half's scale of KV head 1
    at[32:64] = 0xF1                                             # codes 1 and 15
    got = call()
    assert torch.equal(got[:4], want[:4]) and torch.equal(got[4:, :64], want[4:, :64])
    # codes of 15 leave fp32's range; those of 1 hold weight * 2^127 where that is the scale
    from connex_b200.ops import reference as R
    logits = R.int4_values(k[table[0].long(), 1]).view(-1, D)[:n, 0]       # of the keys as they are cached: 15 * bf16(x / 15)
    weight = torch.softmax(logits, 0)[250]
    assert not torch.isfinite(got[4:, 65::2]).any() or weight * 15 * 2.0 ** 127 < 3e38
    if bits == 0x7F00:
        high = got[4:, 64::2].double()
        assert (torch.isnan(high) | ((high - weight * 2.0 ** 127).abs() <= 2.0 ** -6 * weight * 2.0 ** 127)).all()
    else:
        assert bits != 0x7F80 or not torch.isfinite(got[4:, 64:]).any()
