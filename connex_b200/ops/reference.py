"""Plain PyTorch fp32 re-statements of every kernel in :mod:`connex_b200.ops`.

These are the numerics oracles of the test-suite (and of ``smoke()``); no
production code path calls them.  Each takes the same arguments as its
kernel counterpart and returns fp32 results computed from the bf16 inputs.
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F


def gemm(a, b, residual=None):
    out = a.float() @ b.float().t()
    if residual is not None:
        out = out + residual.float()
    return out


def silu_mul_gemm(a, w_interleaved, tile=256):
    from connex_b200.ops import deinterleave_gate_up  # noqa: WPS433 (pure torch helper)
    g, u = deinterleave_gate_up(w_interleaved, tile)
    return F.silu(a.float() @ g.float().t()) * (a.float() @ u.float().t())


def rmsnorm(x, w, eps, residual=None):
    xf = x.float()
    if residual is not None:
        xf = (xf + residual.float()).to(torch.bfloat16).float()
    var = xf.pow(2).mean(-1, keepdim=True)
    return xf * torch.rsqrt(var + eps) * w.float()


def rope(x, positions, cos_sin):
    """x: [T, H, 128] -> rotated (rotate-half convention)."""
    d = x.shape[-1]
    cs = cos_sin[positions.long()]
    cos, sin = cs[:, None, : d // 2], cs[:, None, d // 2:]
    x1, x2 = x[..., : d // 2].float(), x[..., d // 2:].float()
    return torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], dim=-1)


def causal_attention(q, k, v, seq_lens, scale=None):
    """q [T, Hq, D], k/v [T, Hkv, D] packed by sequence -> [T, Hq, D] fp32."""
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    out = torch.empty(T, Hq, D, dtype=torch.float32, device=q.device)
    s = 0
    for n in seq_lens:
        qs = q[s:s + n].float().transpose(0, 1)  # [Hq, n, D]
        ks = k[s:s + n].float().transpose(0, 1).repeat_interleave(Hq // Hkv, 0)
        vs = v[s:s + n].float().transpose(0, 1).repeat_interleave(Hq // Hkv, 0)
        att = (qs @ ks.transpose(1, 2)) * scale
        mask = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1)
        att = att.masked_fill(mask, float("-inf")).softmax(-1)
        out[s:s + n] = (att @ vs).transpose(0, 1)
        s += n
    return out


def paged_decode_attention(q, k_cache, v_cache, block_tables, ctx_lens, scale=None):
    """q [B, Hq, D]; caches [blocks, Hkv, BS, D] -> [B, Hq, D] fp32."""
    B, Hq, D = q.shape
    Hkv, BS = k_cache.shape[1], k_cache.shape[2]
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    out = torch.empty(B, Hq, D, dtype=torch.float32, device=q.device)
    for b in range(B):
        n = int(ctx_lens[b])
        nb = (n + BS - 1) // BS
        blocks = block_tables[b, :nb].long()
        k = k_cache[blocks].float().permute(1, 0, 2, 3).reshape(Hkv, nb * BS, D)[:, :n]
        v = v_cache[blocks].float().permute(1, 0, 2, 3).reshape(Hkv, nb * BS, D)[:, :n]
        k = k.repeat_interleave(Hq // Hkv, 0)
        v = v.repeat_interleave(Hq // Hkv, 0)
        att = (q[b].float()[:, None, :] @ k.transpose(1, 2)) * scale  # [Hq, 1, n]
        out[b] = (att.softmax(-1) @ v)[:, 0]
    return out


def paged_prefill_attention(q, k_cache, v_cache, block_tables, ctx, n_new, scale=None):
    """Chunks that continue cached sequences: q [T, Hq, D] packed by sequence
    (``n_new[i]`` rows each); K/V of positions [0, ctx[i] + n_new[i]) from the
    caches [blocks, Hkv, BS, D] through ``block_tables``; query j of sequence
    i sits at position ctx[i] + j -> [T, Hq, D] fp32."""
    T, Hq, D = q.shape
    Hkv, BS = k_cache.shape[1], k_cache.shape[2]
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    out = torch.empty(T, Hq, D, dtype=torch.float32, device=q.device)
    s = 0
    for b, (c, n) in enumerate(zip(ctx, n_new)):
        tot = c + n
        nb = (tot + BS - 1) // BS
        blocks = block_tables[b, :nb].long()
        k = k_cache[blocks].float().permute(1, 0, 2, 3).reshape(Hkv, nb * BS, D)[:, :tot]
        v = v_cache[blocks].float().permute(1, 0, 2, 3).reshape(Hkv, nb * BS, D)[:, :tot]
        k = k.repeat_interleave(Hq // Hkv, 0)
        v = v.repeat_interleave(Hq // Hkv, 0)
        qs = q[s:s + n].float().transpose(0, 1)                        # [Hq, n, D]
        att = (qs @ k.transpose(1, 2)) * scale                         # [Hq, n, tot]
        keys = torch.arange(tot, device=q.device)[None, :]
        pos = (c + torch.arange(n, device=q.device))[:, None]
        att = att.masked_fill(keys > pos, float("-inf")).softmax(-1)
        out[s:s + n] = (att @ v).transpose(0, 1)
        s += n
    return out


# ---- 8-bit KV cache (64-bit arithmetic)
def fp8_values(cache, scale):
    """What an 8-bit cache [blocks, Hkv, BS, D] with scales [blocks, Hkv] stands for."""
    return cache.double() * scale.double()[..., None, None]


def fp8_scale(amax):
    """The smallest power of two s >= 2^-100 with amax <= 448 s."""
    m, p = torch.frexp(amax.double())
    e = (p - 9 + (m > 0.875).to(p.dtype)).clamp(min=-100)
    return torch.ldexp(torch.ones_like(m), torch.where(amax > 0, e, torch.full_like(e, -100)))


def fp8_append(cache, scale, rows, slots):
    """In place: ``rows`` [T, Hkv, D] (bf16) into their slots; a block whose row
    0 is written starts anew, any other keeps at least its scale and its
    other rows; the later of two rows for a slot wins, slots < 0 are skipped."""
    BS = cache.shape[2]
    by = {}
    for t, s in enumerate(slots.tolist()):
        if s >= 0:
            by.setdefault(s // BS, {})[s % BS] = t
    for b, at in by.items():
        off, tok = torch.tensor(list(at), device=rows.device), torch.tensor(list(at.values()), device=rows.device)
        x = rows[tok].double()                                          # [n, Hkv, D]
        amax = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax((0, 2))
        new = fp8_scale(amax)
        if 0 not in at:
            old = scale[b].double()
            new = torch.maximum(new, old)
            cache[b] = (cache[b].double() * (old / new)[:, None, None]).float().to(cache.dtype)
        x = torch.where(torch.isfinite(x), x, torch.full_like(x, math.nan)) / new[None, :, None]
        cache[b].view(torch.uint8)[:, off] = x.float().to(cache.dtype).view(torch.uint8).transpose(0, 1)
        scale[b] = new.float()


def paged_attention_fp8(q, k_cache, v_cache, k_scale, v_scale, block_tables, ctx, n_new, scale=None):
    """Causal attention of ``n_new[i]`` query rows of each sequence behind
    ``ctx[i]`` cached tokens: q [T, Hq, D] -> [T, Hq, D] fp64, and the same
    sums over |v| (the size that rounding errors of the weights act on)."""
    T, Hq, D = q.shape
    Hkv, BS = k_cache.shape[1], k_cache.shape[2]
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    out = torch.zeros(T, Hq, D, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    s = 0
    for b, (c, n) in enumerate(zip(ctx, n_new)):
        tot = c + n
        if tot > 0 and n > 0:
            ids = block_tables[b, :(tot + BS - 1) // BS].long()
            k, v = (fp8_values(x.view(torch.uint8)[ids].view(x.dtype), z[ids]).transpose(0, 1).reshape(Hkv, -1, D)[:, :tot]
                    .repeat_interleave(Hq // Hkv, 0) for x, z in ((k_cache, k_scale), (v_cache, v_scale)))
            a = (q[s:s + n].double().transpose(0, 1) @ k.transpose(1, 2)) * scale
            late = torch.arange(tot, device=q.device) > (c + torch.arange(n, device=q.device))[:, None]
            p = a.masked_fill(late, float("-inf")).softmax(-1)
            out[s:s + n] = (p @ v).transpose(0, 1)
            mag[s:s + n] = (p @ v.abs()).transpose(0, 1)
        s += n
    return out, mag


# ---- block-scaled fp8 (64-bit arithmetic)
def fp8_block_values(q, scale):
    """What e4m3 [R, K] with scales [R or ceil(R / 128), ceil(K / 128)] stands for."""
    R, K = q.shape
    if scale.shape[0] != R:
        scale = scale.repeat_interleave(128, 0)[:R]
    return q.double() * scale.double().repeat_interleave(128, 1)[:, :K]


def fp8_block_scale(x, rows=1):
    """Scales of ``x`` [R, K] in blocks of ``rows`` x 128: largest finite magnitude / 448, of at least 2^-100."""
    R, K = x.shape
    f = torch.zeros(-(-R // rows) * rows, -(-K // 128) * 128, dtype=torch.float64, device=x.device)
    f[:R, :K] = torch.where(torch.isfinite(x), x.double().abs(), torch.zeros_like(x, dtype=torch.float64))
    return f.view(f.shape[0] // rows, rows, -1, 128).amax((1, 3)).clamp(min=2.0 ** -100) / 448


def gemm_fp8(a, a_scale, b, b_scale, residual=None):
    y = fp8_block_values(a, a_scale) @ fp8_block_values(b, b_scale).t()
    return y if residual is None else y + residual.double()


def silu_mul_columns(y, tile=256):
    """SiLU(gate) * up of columns [.., N] that alternate in blocks of tile / 2."""
    g, u = (t.flatten(-2) for t in y.unflatten(-1, (-1, 2, tile // 2)).unbind(-2))
    return g * torch.sigmoid(g) * u


# ---- 4-bit KV cache (64-bit arithmetic)
def int4_values(rows):
    """uint8 [..., 72] -> fp64 [..., 128]."""
    code = torch.stack([rows[..., :64] & 15, rows[..., :64] >> 4], -1).flatten(-2).double().unflatten(-1, (2, 64))
    par = rows[..., 64:].contiguous().view(torch.bfloat16).double()
    return (code * par[..., 0::2, None] + par[..., 1::2, None]).flatten(-2)


def int4_rows(x):
    """bf16 [..., 128] -> uint8 [..., 72]."""
    h = x.double().unflatten(-1, (2, 64))
    lo, hi = h.amin(-1), h.amax(-1)
    scale = ((hi - lo) / 15).to(torch.bfloat16)
    s = scale.double()[..., None]
    code = torch.where(s > 0, (h - lo[..., None]) / s.clamp(min=1e-300), torch.zeros_like(h)).round().clamp(0, 15)
    code = code.nan_to_num(0.0).to(torch.uint8).flatten(-2)
    bad = ~torch.isfinite(scale.float()) | ~torch.isfinite(h).all(-1)
    par = torch.stack([scale, lo.to(torch.bfloat16)], -1)
    par = torch.where(bad[..., None], torch.full_like(par, math.nan), par)
    code = torch.where(bad.repeat_interleave(64, -1), torch.zeros_like(code), code)
    return torch.cat([code[..., 0::2] | code[..., 1::2] << 4, par.flatten(-2).contiguous().view(torch.uint8)], -1)


def int4_append(cache, rows, slots):
    """In place: ``rows`` [T, Hkv, 128] (bf16) into their slots of [blocks, Hkv, 16, 72]; slots < 0 are skipped."""
    keep = slots >= 0
    s = slots[keep]
    cache[s // 16, :, s % 16] = int4_rows(rows[keep])


def paged_attention_int4(q, k_cache, v_cache, block_tables, ctx, n_new, scale=None):
    """:func:`paged_attention_fp8` over a 4-bit cache: outputs and the same sums over |v|, fp64."""
    T, Hq, D = q.shape
    Hkv = k_cache.shape[1]
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    out = torch.zeros(T, Hq, D, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    s = 0
    for b, (c, n) in enumerate(zip(ctx, n_new)):
        tot = c + n
        if tot > 0 and n > 0:
            ids = block_tables[b, :(tot + 15) // 16].long()
            k, v = (int4_values(x[ids]).transpose(0, 1).reshape(Hkv, -1, D)[:, :tot].repeat_interleave(Hq // Hkv, 0)
                    for x in (k_cache, v_cache))
            a = (q[s:s + n].double().transpose(0, 1) @ k.transpose(1, 2)) * scale
            late = torch.arange(tot, device=q.device) > (c + torch.arange(n, device=q.device))[:, None]
            p = a.masked_fill(late, float("-inf")).softmax(-1)
            out[s:s + n] = (p @ v).transpose(0, 1)
            mag[s:s + n] = (p @ v.abs()).transpose(0, 1)
        s += n
    return out, mag


def kv_copy_blocks(kv, pairs, scales=None):
    """In-place reference of kv_copy_blocks on plain tensors."""
    src, dst = pairs[:, 0].long(), pairs[:, 1].long()
    raw = kv.view(torch.uint8) if kv.element_size() == 1 else kv
    raw[:, :, dst] = raw[:, :, src]
    if scales is not None:
        scales[:, :, dst] = scales[:, :, src]


def kv_push(src_k, src_v, dst_k, dst_v, pairs, src_h0=0, dst_h0=0, n_heads=None):
    """In-place reference of kv_push_layer on plain tensors."""
    nh = n_heads if n_heads is not None else src_k.shape[1]
    for sb, db in pairs.tolist():
        dst_k[db, dst_h0:dst_h0 + nh] = src_k[sb, src_h0:src_h0 + nh]
        dst_v[db, dst_h0:dst_h0 + nh] = src_v[sb, src_h0:src_h0 + nh]
