// The 8-bit paged KV cache: quantising write, decode attention over it, block
// copies.
//
// Values are e4m3 with one power-of-two scale per (block of 16 tokens, KV
// head).  e4m3 is a floating format, so the scale's mantissa would buy no
// accuracy; as a power of two, raising a block's scale for a later, larger
// token moves exponents only (exact except for values that fall under the
// smallest e4m3 step), and every cached value is an exact bf16 number.
#include <algorithm>
#include <stdexcept>
#include <type_traits>

#include "common.cuh"
#include "kv_fp8.h"

namespace cx {

namespace kvq {
constexpr int D = 128, BS = 16;
constexpr int MIN_EXP = -100, MAX_EXP = 120;   // 448 * 2^120 covers every finite bf16
constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int SMEM = BS * D * 4 + WARPS * BS * D * 2;   // cos / sin rows, each warp's rows
}  // namespace kvq

// 2^e for e of [-126, 127]
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// The smallest e >= MIN_EXP with a <= 448 * 2^e = 1.75 * 2^(e + 8), for finite a >= 0.
__device__ __forceinline__ int fp8_exp_for(float a) {
  const uint32_t u = __float_as_uint(a);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(e, kvq::MIN_EXP);
}
__device__ __forceinline__ int fp8_exp_of(float scale) {
  return min(max((int)((__float_as_uint(scale) >> 23) & 255u) - 127, kvq::MIN_EXP), kvq::MAX_EXP);
}
// two fp32 -> two e4m3 bytes (lo in the low byte), nearest even, NaN kept
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// two e4m3 bytes -> f16x2, exact
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
  return r;
}
__device__ __forceinline__ float f16_lo(uint32_t v) {
  float f;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.f32.f16 %0, l;\n\t}" : "=f"(f) : "r"(v));
  return f;
}
__device__ __forceinline__ float f16_hi(uint32_t v) {
  float f;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.f32.f16 %0, h;\n\t}" : "=f"(f) : "r"(v));
  return f;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float finite_or_zero(float a) {   // |a| of a finite value, 0 of Inf and NaN
  const uint32_t u = __float_as_uint(a) & 0x7fffffffu;
  return u < 0x7f800000u ? __uint_as_float(u) : 0.f;
}
// x * mul as e4m3 would hold it: e4m3 has no infinities, so Inf becomes NaN
__device__ __forceinline__ float scaled_or_nan(float x, float mul) {
  return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u ? __uint_as_float(0x7fffffffu) : x * mul;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ u128 lds16(uint32_t a) {
  u128 r;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a) : "memory");
  return r;
}
__device__ __forceinline__ void sts16(uint32_t a, const u128& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint64_t unpack_bf16x2(uint32_t w) { return f32x2(bf16_lo(w), bf16_hi(w)); }
// larger magnitudes of two bf16 pairs, signs undefined; NaN only where both are
__device__ __forceinline__ uint32_t max_abs_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// a cos + b sin of a pair of dims, rounded to bf16
__device__ __forceinline__ uint32_t turn_bf16x2(uint32_t a, uint32_t b, uint64_t co, uint64_t si) {
  const uint64_t r = fma_f32x2(unpack_bf16x2(b), si, mul_f32x2(unpack_bf16x2(a), co));
  return pack_bf16x2(lo_f32(r), hi_f32(r));
}
struct alignas(16) f32x4 {        // two pairs of fp32
  uint64_t a, b;
};

// ------------------------------------------------- RoPE + quantising write
// CTAs of two kinds.  Block CTAs write the cache.  A block's scale depends on
// every row that the call puts there, so one CTA collects them: the one whose
// token is the first to fall into the block scans the call's slots, which
// keeps the result independent of the rows' order (of two rows for one slot
// the later wins).  Each of its warps takes K or V of one KV head on its own:
// all rows' loads in flight together, K rotated, the largest magnitude, the
// scale, the block's older rows requantised if the scale grew, the new rows.
// A block whose row 0 is written starts anew; otherwise its scale never
// shrinks.  Tokens are dealt to these CTAs with an odd stride: the first rows
// of blocks, every 16th token of a prompt, then spread over all of them, and
// so do the rows of decode steps.  Rotation CTAs take the q heads, eight of a
// token per warp at a time.
// 8192 rows of 32/8 heads take 42 us: rotating q alone 25 (134 MB at 5.3
// TB/s), and on the same SMs the scans 6, the blocks' stores 3.5 and their
// arithmetic 4.  A bf16 cache's write takes 65.  One row each of many
// sequences is a block CTA and a scan per row: 4.4, 6.3, 18.6 and 75 us for
// 64, 256, 1024 and 4096 rows, where the bf16 write takes 2.4, 3.5, 8.3 and 27.
__device__ __forceinline__ void write_block(const __nv_bfloat16* qkv, int ldq, const int* pos, const float* cos_sin,
                                            const int64_t* slots, const KvFp8& c, int t, int blk, int group, int T,
                                            int Hq, int max_pos, const __nv_bfloat16* kn, float eps) {
  using namespace kvq;
  __shared__ int row_of[BS];      // the token of each row of the block (-1: not written by this call)
  __shared__ int first;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // which rows the call writes, and whether t is the first of their tokens
  auto scan = [&](bool check) {
    __syncthreads();
    if (tid < BS) row_of[tid] = -1;
    if (tid == 0) first = 0x7fffffff;
    __syncthreads();
    auto take = [&](int i, int64_t si) {
      if ((si >> 4) != blk) return;                     // below 0: not cached
      atomicMin(&first, i);
      if (!check || (pos[i] >= 0 && pos[i] < max_pos)) atomicMax(&row_of[(int)(si & 15)], i);
    };
    if ((reinterpret_cast<uintptr_t>(slots) & 15) == 0) {
#pragma unroll 8
      for (int i = 2 * tid; i < (T & ~1); i += 2 * THREADS) {
        const longlong2 s2 = *reinterpret_cast<const longlong2*>(slots + i);
        take(i, s2.x);
        take(i + 1, s2.y);
      }
      if ((T & 1) && tid == 0) take(T - 1, slots[T - 1]);
    } else {
      for (int i = tid; i < T; i += THREADS) take(i, slots[i]);
    }
    __syncthreads();
  };
  scan(false);
  if (first != t) return;         // uniform over the CTA
  int tok = row_of[lane & 15], ptok = tok >= 0 ? pos[tok] : 0;     // lane r (and r + 16): row r
  if (__any_sync(0xffffffffu, ptok < 0 || ptok >= max_pos)) {      // positions out of range: those rows do not count
    scan(true);
    tok = row_of[lane & 15];
    ptok = tok >= 0 ? pos[tok] : 0;
  }
  const uint32_t rows = __ballot_sync(0xffffffffu, tok >= 0) & 0xffffu;
  if (rows == 0) return;
  // A warp: K or V of one head; step i: rows 2i and 2i + 1, 16 lanes of 8 dims
  // each.  The rows pass through shared memory: asynchronous copies, all in
  // flight at once.  (Kept in registers instead, with the loops unrolled, the
  // same rows took 47 us of 8192 where this takes 43, and 5.3 us of 64 decode
  // rows where this takes 4.1: the code is long for what each CTA runs once.)
  extern __shared__ __align__(16) uint8_t smem[];
  const int half = lane >> 4, j = lane & 15;
  const uint32_t table = smem_u32(smem), mine = table + BS * D * 4 + warp * (BS * D * 2) + half * (D * 2) + j * 16;
  __syncthreads();                // the previous block is done with the table
  for (int r = warp; r < BS; r += WARPS) {              // cos / sin: a row per warp at a time
    const int pr = __shfl_sync(0xffffffffu, ptok, r);
    if (rows >> r & 1) cp_async16(table + r * (D * 4) + lane * 16, cos_sin + (size_t)pr * D + lane * 4);
  }
  const int h = (group * WARPS + warp) >> 1;            // K in the even warps, V in the odd ones
  const bool on = h < c.Hkv, is_v = warp & 1;
  float* scale = (is_v ? c.vs : c.ks) + (size_t)blk * c.Hkv + h;
  float old = 1.f;
  if (on) {
    old = *scale;
    const __nv_bfloat16* src = qkv + (size_t)(Hq + (is_v ? c.Hkv : 0) + h) * D + 8 * j;
#pragma unroll 4
    for (int i = 0; i < 8; ++i) {
      const int tr = __shfl_sync(0xffffffffu, tok, 2 * i + half);
      if (tr >= 0) cp_async16(mine + i * (D * 4), src + (size_t)tr * ldq);
    }
  }
  cp_async_commit();
  cp_async_wait<0>();
  __syncthreads();                                    // the table
  if (!on) return;
  uint32_t top = 0;
#pragma unroll 2
  for (int i = 0; i < 8; ++i) {
    if (!(rows >> 2 * i & 3)) continue;               // uniform over the warp
    const bool here = rows >> (2 * i + half) & 1;
    u128 x = here ? lds16(mine + i * (D * 4)) : u128{0, 0, 0, 0};
    uint32_t* w = reinterpret_cast<uint32_t*>(&x);
    if (!is_v) {
      u128 y = here ? lds16(mine + (j < 8 ? D : -D) + i * (D * 4)) : u128{0, 0, 0, 0};   // the partner dims, 64 away
      uint32_t* z = reinterpret_cast<uint32_t*>(&y);
      __syncwarp();                                   // both halves of a row are read before one is written
      if (kn != nullptr) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) ss += bf16_lo(w[e]) * bf16_lo(w[e]) + bf16_hi(w[e]) * bf16_hi(w[e]);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float n = rsqrtf(ss * (1.0f / D) + eps);
        const u128 nw = ld_v4(kn + 8 * j), nz = ld_v4(kn + 8 * (j ^ 8));
        const uint32_t *pw = reinterpret_cast<const uint32_t*>(&nw), *pz = reinterpret_cast<const uint32_t*>(&nz);
        // bf16 between the norm and the rotation, like a norm layer of its own
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] = pack_bf16x2(bf16_lo(w[e]) * n * bf16_lo(pw[e]), bf16_hi(w[e]) * n * bf16_hi(pw[e]));
          z[e] = pack_bf16x2(bf16_lo(z[e]) * n * bf16_lo(pz[e]), bf16_hi(z[e]) * n * bf16_hi(pz[e]));
        }
      }
      const uint32_t flip = j < 8 ? 0x80008000u : 0u; // first half: a cos - b sin; second: a cos + b sin
      const uint32_t cs = table + (2 * i + half) * (D * 4) + (j & 7) * 32;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const u128 co = lds16(cs + 16 * e), si = lds16(cs + 2 * D + 16 * e);
        const f32x4 &c4 = reinterpret_cast<const f32x4&>(co), &s4 = reinterpret_cast<const f32x4&>(si);
        // rounded to bf16 before e4m3: what a bf16 cache would hold is what is quantised
        w[2 * e] = turn_bf16x2(w[2 * e], z[2 * e] ^ flip, c4.a, s4.a);
        w[2 * e + 1] = turn_bf16x2(w[2 * e + 1], z[2 * e + 1] ^ flip, c4.b, s4.b);
      }
      if (here) sts16(mine + i * (D * 4), x);
      else x = u128{0, 0, 0, 0};
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) top = max_abs_bf16x2(top, w[e]);
  }
  top &= 0x7fff7fffu;
  float amax = fmaxf(bf16_lo(top), bf16_hi(top));
  // Inf or NaN among the new rows: they have no part in the scale
  const bool special = __any_sync(0xffffffffu, (top & 0xffffu) >= 0x7f80u || top >= 0x7f800000u);
  if (special) {
    amax = 0.f;
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      const u128 x = rows >> (2 * i + half) & 1 ? lds16(mine + i * (D * 4)) : u128{0, 0, 0, 0};
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&x);
#pragma unroll
      for (int e = 0; e < 4; ++e) amax = fmaxf(amax, fmaxf(finite_or_zero(bf16_lo(w[e])), finite_or_zero(bf16_hi(w[e]))));
    }
  }
  amax = warp_max(amax);
  uint8_t* dst = (is_v ? c.v : c.k) + ((size_t)blk * c.Hkv + h) * (BS * D) + half * D + 8 * j;
  int e = fp8_exp_for(amax);
  if (!(rows & 1)) {            // the block's rows so far stay
    const int was = fp8_exp_of(old);
    if (e <= was) {
      e = was;
    } else {
      const float f = exp2_int(max(was - e, -126));
      uint2 w[8];                                     // all loads before the first store
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = *reinterpret_cast<const uint2*>(dst + 2 * i * D);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (rows >> (2 * i + half) & 1) continue;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t& v = k ? w[i].y : w[i].x;
          const uint32_t a = e4m3x2_to_f16x2((uint16_t)v), b = e4m3x2_to_f16x2((uint16_t)(v >> 16));
          v = to_e4m3x2(f16_lo(a) * f, f16_hi(a) * f) | to_e4m3x2(f16_lo(b) * f, f16_hi(b) * f) << 16;
        }
        *reinterpret_cast<uint2*>(dst + 2 * i * D) = w[i];
      }
    }
  }
  __syncwarp();                 // every lane has read the old scale
  if (lane == 0) *scale = exp2_int(e);
  const float mul = exp2_int(-e);
  const uint64_t mul2 = f32x2(mul, mul);
  auto store = [&](auto inf) {
#pragma unroll 2
    for (int i = 0; i < 8; ++i) {
      if (!(rows >> (2 * i + half) & 1)) continue;
      const u128 x = lds16(mine + i * (D * 4));
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&x);
      uint32_t q[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint64_t r = mul_f32x2(unpack_bf16x2(w[k]), mul2);
        q[k] = inf ? to_e4m3x2(scaled_or_nan(bf16_lo(w[k]), mul), scaled_or_nan(bf16_hi(w[k]), mul))
                   : to_e4m3x2(lo_f32(r), hi_f32(r));
      }
      *reinterpret_cast<uint2*>(dst + 2 * i * D) = make_uint2(q[0] | q[1] << 16, q[2] | q[3] << 16);
    }
  };
  if (special) store(std::true_type{});
  else store(std::false_type{});
}

// Heads [8 hu, 8 hu + 8) of token t's q: a lane holds dims [8 j, 8 j + 8) of four of them.
__device__ __forceinline__ void rotate_q(const __nv_bfloat16* qkv, int ldq, const int* pos, const float* cos_sin,
                                         __nv_bfloat16* out, int ldo, int t, int hu, int Hq, int max_pos,
                                         const __nv_bfloat16* qn, float eps) {
  using namespace kvq;
  const int lane = threadIdx.x & 31, j = lane & 15, h0 = 8 * hu + (lane >> 4);
  u128 raw[4];
#pragma unroll
  for (int k = 0; k < 4; ++k)
    raw[k] = h0 + 2 * k < Hq ? ld_v4(qkv + (size_t)t * ldq + (size_t)(h0 + 2 * k) * D + 8 * j) : u128{0, 0, 0, 0};
  const int p = pos[t];
  const bool pos_ok = p >= 0 && p < max_pos;
  f32x4 co[2], si[2];                                   // sin negated in the first half: a cos - b sin
  co[0] = co[1] = si[0] = si[1] = f32x4{0ull, 0ull};
  if (pos_ok) {
    const f32x4* cs = reinterpret_cast<const f32x4*>(cos_sin + (size_t)p * D + 8 * (j & 7));
    const uint64_t flip = j < 8 ? 0x8000000080000000ull : 0ull;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      co[e] = cs[e];
      si[e] = cs[D / 8 + e];
      si[e].a ^= flip;
      si[e].b ^= flip;
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&raw[k]);
    if (qn != nullptr) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) ss += bf16_lo(w[e]) * bf16_lo(w[e]) + bf16_hi(w[e]) * bf16_hi(w[e]);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float n = rsqrtf(ss * (1.0f / D) + eps);
      const u128 nw = ld_v4(qn + 8 * j);
      const uint32_t* pw = reinterpret_cast<const uint32_t*>(&nw);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = pack_bf16x2(bf16_lo(w[e]) * n * bf16_lo(pw[e]), bf16_hi(w[e]) * n * bf16_hi(pw[e]));
    }
    u128 r;
    uint32_t* pr = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t b0 = __shfl_xor_sync(0xffffffffu, w[2 * e], 8), b1 = __shfl_xor_sync(0xffffffffu, w[2 * e + 1], 8);
      pr[2 * e] = turn_bf16x2(w[2 * e], b0, co[e].a, si[e].a);
      pr[2 * e + 1] = turn_bf16x2(w[2 * e + 1], b1, co[e].b, si[e].b);
    }
    if (!pos_ok) r = u128{0, 0, 0, 0};                  // a position out of range: zeros
    if (h0 + 2 * k < Hq) st_v4(out + (size_t)t * ldo + (size_t)(h0 + 2 * k) * D + 8 * j, r);
  }
}

// CTAs 0, 2, 4, .. write blocks (n_block for each group of WARPS of a block's
// K and V heads), the others rotate q; once one kind is used up the rest is
// the other.
__global__ void __launch_bounds__(kvq::THREADS, 4)
    rope_cache_fp8_kernel(const __nv_bfloat16* qkv, int ldq, const int* __restrict__ pos,
                          const float* __restrict__ cos_sin, const int64_t* __restrict__ slots, KvFp8 c,
                          __nv_bfloat16* out, int ldo, int T, int Hq, int max_pos, int* status,
                          const __nv_bfloat16* __restrict__ qn, const __nv_bfloat16* __restrict__ kn, float eps,
                          int n_block, int groups, int n_rot) {
  using namespace kvq;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n_b = n_block * groups, both = 2 * min(n_b, n_rot), i = blockIdx.x;
  const bool block_cta = i < both ? (i & 1) == 0 : n_b > n_rot;
  int k = i < both ? i >> 1 : i - both / 2;             // its number among its kind
  if (!block_cta) {
    const uint32_t hus = (Hq + 7) / 8;
    const uint32_t units = (uint32_t)T * hus;           // T <= KVQ_MAX_ROWS
    for (uint32_t u = k * WARPS + warp; u < units; u += n_rot * WARPS) {
      const uint32_t t = u / hus;
      rotate_q(qkv, ldq, pos, cos_sin, out, ldo, t, u - t * hus, Hq, max_pos, qn, eps);
    }
    return;
  }
  const int group = k / n_block;
  k -= group * n_block;
  for (int base = k; base < T; base += 32 * n_block) {  // 32 of the CTA's tokens at a time, one per lane
    const int64_t tl = base + (int64_t)lane * n_block;
    bool cand = false;
    int block = -1;
    if (tl < T) {
      const int64_t slot = slots[tl], before = tl > 0 ? slots[tl - 1] : -1;
      const int p = pos[tl];
      const bool in = slot >= 0 && (slot >> 4) < c.num_blocks;
      if (warp == 0 && group == 0 && ((slot >= 0 && !in) || p < 0 || p >= max_pos)) record_status(status, CX_ERR_BOUNDS);
      cand = in && (before < 0 || (before >> 4) != (slot >> 4));   // most tokens of a prompt follow one of the same block
      block = (int)(slot >> 4);
    }
    for (uint32_t m = __ballot_sync(0xffffffffu, cand); m != 0; m &= m - 1) { // the same in every warp
      const int blk = __shfl_sync(0xffffffffu, block, __ffs(m) - 1);
      write_block(qkv, ldq, pos, cos_sin, slots, c, base + (__ffs(m) - 1) * n_block, blk, group, T, Hq, max_pos, kn, eps);
    }
  }
}

void rope_cache_fp8(const void* qkv, int ldq, const int* pos, const float* cos_sin, const int64_t* slots,
                    const KvFp8& c, void* out, int ldo, int T, int Hq, int max_pos, int sms, int* status,
                    cudaStream_t s, const void* q_norm, const void* k_norm, float eps) {
  static bool attr[64] = {};
  int dev;
  cudaGetDevice(&dev);
  if (!attr[dev & 63]) {
    cudaFuncSetAttribute(rope_cache_fp8_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kvq::SMEM);
    attr[dev & 63] = true;
  }
  // Each block's first row scans the call's slots, so rows are taken
  // KVQ_MAX_ROWS at a time to keep the scan linear in T.
  for (int t0 = 0; t0 < T; t0 += KVQ_MAX_ROWS) {
    const int n = std::min(KVQ_MAX_ROWS, T - t0);
    // tokens per CTA: few enough that two first rows rarely meet in one (8192 rows:
    // 43 us with n / 14 and with n / 8; five 613-row prompts: 22 and 17 us)
    const int n_block = std::min(n, std::max(n / 8, 2 * sms) | 1);
    const int64_t units = (int64_t)n * ((Hq + 7) / 8);
    const int groups = (2 * c.Hkv + kvq::WARPS - 1) / kvq::WARPS;
    const int n_rot = (int)std::min<int64_t>((units + kvq::WARPS - 1) / kvq::WARPS, 6 * sms);
    rope_cache_fp8_kernel<<<n_block * groups + n_rot, kvq::THREADS, kvq::SMEM, s>>>(
        reinterpret_cast<const __nv_bfloat16*>(qkv) + (size_t)t0 * ldq, ldq, pos + t0, cos_sin, slots + t0, c,
        reinterpret_cast<__nv_bfloat16*>(out) + (size_t)t0 * ldo, ldo, n, Hq, max_pos, status,
        reinterpret_cast<const __nv_bfloat16*>(q_norm), reinterpret_cast<const __nv_bfloat16*>(k_norm), eps, n_block,
        groups, n_rot);
  }
}

// ------------------------------------------------------- decode attention
// S = q.K^T and O^T = V^T.W^T on mma.sync m16n8k16 (f16 in, fp32 out).  The
// cached bytes are turned into f16 (exact) in registers, in the fragments'
// layout as they come from the cache; the block scales stay out of the
// operands.  (mma.sync takes e4m3 operands too.  With them the kernel executed
// 61 million warp instructions at 64 x 4096, with f16 ones 43 million, and q,
// made f16 once, has to be converted no further: 103 us with e4m3, 101 with
// f16, ragged lengths 38 and 34.)
//   K: lane (g = lane / 4, c = lane % 4) takes bytes [16 c, 16 c + 16) of both
//      64-byte halves of tokens g and g + 8.  The contraction may take the
//      dims in any order as long as q uses the same one, so each word of a
//      piece is the four k-values a lane holds of an MMA step.
//   V: the lane takes bytes [16 g, 16 g + 16) of tokens 2c, 2c + 1, 2c + 8,
//      2c + 9 of each block -- the tokens whose weights S leaves in this lane --
//      and interleaves the bytes of two tokens.
// q is scaled by a power of two per head into f16's range: exact but for
// elements 2^29 times smaller than the head's largest.  K's scale multiplies
// the logits.  V's is part of the weights 2^(x - mv) v, which have a running
// maximum mv of their own next to the one of the softmax sum, so that f16
// holds them (2^-11 of each) whatever the ratio of the blocks' scales.
//
// Loads: cp.async into three slots per warp, each K or V of two blocks, in the
// order of their use: one is read while two are under way, without barriers
// between warps.  Block ids and scales come 32 blocks at a time, one per lane.
//
// Work split: the blocks of all (sequence, KV head) pairs, laid end to end
// with PAIR_COST blocks' worth for the fixed cost of a pair, are cut into
// equal shares, one per CTA, from the lengths themselves -- the same launch (a
// graph replay) is balanced for any lengths.  A pair that spans several CTAs
// leaves partial results in the workspace, and the CTA that arrives last
// merges them (a counter that wraps to zero by itself).  64 x 4096 tokens of
// 32/8 heads take 100 us, 0.82 of the rate of a copy (the loads alone 95, a
// fixed 10 of it before the first byte and after the last).  Where no pair is
// longer than two shares, cuts move by up to SLACK blocks' worth to the pair's
// start or end: a part more costs a CTA more than that (64 x 128 tokens 7.7 us,
// 14.3 with the cuts where they fall; 64 x 500 15.2 and 19.5; with twice the
// slack 100 x 2048 takes 84, not 80; ragged lengths gain nothing).
namespace dec8 {
// Two CTAs of eight warps took 99 us of 2 x 131072 (102 with four of four) and 32.5 of ragged lengths (34), but
// 18.2 of 64 x 500 (15.2) and 9.5 of 64 x 16 (6.0): a pair's start and end wait for all the CTA's warps.
constexpr int D = kvq::D, BS = kvq::BS, WARPS = 4, THREADS = 32 * WARPS;
// CTAs that an SM holds at a time, by the registers of the variant for nt tiles of query heads
constexpr int ctas_per_sm(int nt) { return nt == 1 ? 4 : 3; }
constexpr int MIN_UNITS = 2 * WARPS;    // blocks' worth of a CTA, at least (500 tokens alone: 6.6 us; 7.5 with 16)
constexpr int PAIR_COST = 4 * WARPS;    // measured on ragged lengths: 41 us with 8, 34 with 16 and with 32
constexpr int SLACK = 2 * PAIR_COST;    // see the work split above
constexpr float RESCALE = 8.f;          // O is rescaled once mv has grown by this much: weights stay under 2^9
constexpr int SLOT = 2 * BS * D;        // K (or V) of two blocks
constexpr int SLOTS = 3;                // per warp: one in use, two on their way
constexpr int RING = WARPS * SLOTS * SLOT;
constexpr int O_ROW = D + 4;            // floats of a head's row of O: eight lanes' stores fall on eight banks
template <int NT>
struct Smem {                           // rings, later the warps' O | their (m, l, mv) | q fragments | prefix sums
  static constexpr int STATS = RING;
  static_assert(WARPS * 8 * NT * O_ROW * 4 <= RING, "O fits in the drained rings");
  static constexpr int Q = STATS + WARPS * 8 * NT * 16;
  static constexpr int PRE = Q + NT * 4 * 32 * 16;
  static constexpr int bytes(int B) { return PRE + (B + 1) * 4; }
};
}  // namespace dec8

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a));
  return r;
}
__device__ __forceinline__ uint32_t word(const u128& v, int i) { return reinterpret_cast<const uint32_t*>(&v)[i]; }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// NT: tiles of 8 query heads per KV head (1: groups up to 8, 2: up to 16).
template <int NT>
__global__ void __launch_bounds__(dec8::THREADS, dec8::ctas_per_sm(NT))
    decode_attn_fp8_kernel(const __nv_bfloat16* __restrict__ q, int ldq, KvFp8 c, const int* __restrict__ tables,
                           int max_blocks, const int* __restrict__ ctx_lens, __nv_bfloat16* __restrict__ out, int ldo,
                           int B, int Hq, float scale_log2, float* __restrict__ part, uint32_t* __restrict__ counters,
                           int* status) {
  using namespace dec8;
  extern __shared__ __align__(16) uint8_t smem[];
  float* so = reinterpret_cast<float*>(smem);                           // [WARPS][8 NT][O_ROW], once the rings are drained
  float* sm = reinterpret_cast<float*>(smem + Smem<NT>::STATS);         // [WARPS][8 NT][m, l, mv]
  uint4* sq = reinterpret_cast<uint4*>(smem + Smem<NT>::Q);             // [NT][4 steps][32 lanes]
  int* pre = reinterpret_cast<int*>(smem + Smem<NT>::PRE);              // [B + 1] units of the pairs before sequence b
  __shared__ int wsum[WARPS], wtop[WARPS];
  __shared__ int2 share[2];
  __shared__ uint32_t ticket;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gq = lane >> 2, qd = lane & 3;
  const int Hkv = c.Hkv, G = Hq / Hkv;

  auto len_of = [&](int b) { return min(max(ctx_lens[b], 0), max_blocks * BS); };
  // ---- prefix sums of the pairs' units
  if (tid == 0) pre[0] = 0;
  int run = 0, top = 0;                                         // all units; the longest sequence's
  for (int b0 = 0; b0 < B; b0 += THREADS) {
    const int b = b0 + tid;
    int n = 0;
    if (b < B) {
      if (ctx_lens[b] > max_blocks * BS && blockIdx.x == 0) record_status(status, CX_ERR_BOUNDS);
      const int len = len_of(b);
      n = len > 0 ? ((len + BS - 1) / BS + PAIR_COST) * Hkv : 0;
    }
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    const int longest = __reduce_max_sync(0xffffffffu, n);
    if (lane == 31) {
      wsum[warp] = x;
      wtop[warp] = longest;
    }
    __syncthreads();
    int add = run;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) add += wsum[w];
      run += wsum[w];
      top = max(top, wtop[w]);
    }
    if (b < B) pre[b + 1] = add + x;
    __syncthreads();
  }
  const int total = run;
  // rows without tokens: zeros
  for (int b = blockIdx.x; b < B; b += gridDim.x)
    if (pre[b + 1] == pre[b])
      for (int i = tid; i < Hq * D / 8; i += THREADS) st_v4(out + (size_t)b * ldo + 8 * i, u128{0, 0, 0, 0});
  const int n_cta = max(1, min((int)gridDim.x, (total + MIN_UNITS - 1) / MIN_UNITS));
  const int per = (total + n_cta - 1) / n_cta;
  // blocks' worth by which a cut moves to the start or the end of the pair it falls into
  const int most = top <= 2 * per * Hkv ? SLACK : 0;
  auto slack_of = [&](int units) { return min((units - PAIR_COST) / 2, most); };
  const int x = (blockIdx.x + (tid & 1)) * per;          // thread 0 finds the share's start, thread 1 its end
  int lo = 0, end = total;
  if (x < total) {
    int hi = B;                                         // the sequence that holds x: the last b with pre[b] <= x
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= x) lo = mid;
      else hi = mid;
    }
    const int units = (pre[lo + 1] - pre[lo]) / Hkv, into = (x - pre[lo]) % units, slack = slack_of(units);
    end = into <= PAIR_COST + slack ? x - into : units - into <= slack ? x - into + units : x;
  }
  // (through shared memory, not shuffles: the compiler then knows that they are the same in all
  // lanes; 64 x 4096 took 115 us otherwise)
  if (tid < 2) share[tid] = make_int2(end, lo);
  __syncthreads();
  const int u0 = share[0].x, u1 = share[1].x;
  int b = share[0].y;
  // Both land row by row, 512 contiguous bytes per instruction (measured: with
  // every lane fetching the pieces it reads back, K in 64-byte halves and V
  // in every other row, the loads alone took 122 us of 64 x 4096 where these
  // take 96).  16-byte pieces are permuted inside a row so that the fragment
  // reads meet no bank twice: K by the row's lowest bit (two rows at a time
  // are read), V by the two above it (rows 2c, c = 0 .. 3).
  const uint32_t ring = smem_u32(smem) + warp * (SLOTS * SLOT);
  const uint32_t kput = (lane >> 3) * D + (((lane & 7) ^ (lane >> 3 & 1) * 4) << 4);
  const uint32_t kget = gq * D + ((qd ^ (gq & 1) * 4) << 4);
  const int khalf = gq & 1 ? -64 : 64;
  const uint32_t vput = (lane >> 3) * D + (((lane & 7) ^ (lane >> 4) * 2) << 4);   // rows 0-3; ^ 64 in rows 4-7
  const uint32_t vget = 2 * qd * D + ((gq ^ qd * 2) << 4);
  const int vhalf = gq >> 1 & 1;       // 8-byte half of the piece that comes first (bank conflicts again)

  for (int u = u0; u < u1;) {
    // ---- the blocks [j0, j1) of KV head h of sequence b
    while (pre[b + 1] <= u) ++b;
    const int units = (pre[b + 1] - pre[b]) / Hkv;
    const int h = (u - pre[b]) / units;
    const int pair0 = pre[b] + h * units;                      // first unit of the pair
    const int j0 = max(0, u - pair0 - PAIR_COST), j1 = min(units, u1 - pair0) - PAIR_COST;
    u = min(pair0 + units, u1);
    if (j1 <= 0) continue;                                     // none but the pair's fixed cost
    const int len = len_of(b);

    // ---- the warp's loads, two blocks at a time: K and V of it, K and V of the next, ...
    int fj = j0 + 2 * warp, fcount = 0, ids = -1, id0 = -1, id1 = -1;
    float lks = 0.f, lvs = 0.f;
    auto fetch_k = [&](uint32_t slot) {
      id0 = id1 = -1;
      if (fj < j1) {
        if ((fcount & 15) == 0) {                              // ids of the next 32 blocks, one per lane
          const int mine = fj + (lane >> 1) * (2 * WARPS) + (lane & 1);
          ids = -1;
          if (mine < j1) {
            ids = tables[(size_t)b * max_blocks + mine];
            if (ids < 0 || ids >= c.num_blocks) {
              record_status(status, CX_ERR_BOUNDS);
              ids = -1;
            }
          }
        }
        id0 = __shfl_sync(0xffffffffu, ids, 2 * (fcount & 15));
        id1 = __shfl_sync(0xffffffffu, ids, 2 * (fcount & 15) + 1);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int id = i ? id1 : id0;
          if (id < 0) continue;
          const uint8_t* p = c.k + ((size_t)id * Hkv + h) * (BS * D) + lane * 16;
#pragma unroll
          for (int e = 0; e < 4; ++e) cp_async16(slot + kput + (4 * i + e) * 512, p + e * 512);
        }
        if ((fcount & 15) == 0) {                              // their scales: needed when the blocks are used
          lks = ids >= 0 ? c.ks[(size_t)ids * Hkv + h] : -1.f; // below 0: no block
          lvs = ids >= 0 ? c.vs[(size_t)ids * Hkv + h] : 0.f;
        }
        fj += 2 * WARPS;
        ++fcount;
      }
      cp_async_commit();
    };
    auto fetch_v = [&](uint32_t slot) {                        // of the blocks whose K was fetched last
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int id = i ? id1 : id0;
        if (id < 0) continue;
        const uint8_t* p = c.v + ((size_t)id * Hkv + h) * (BS * D) + lane * 16;
#pragma unroll
        for (int e = 0; e < 4; ++e) cp_async16(slot + (4 * i + e) * 512 + (vput ^ (e & 1) * 64), p + e * 512);
      }
      cp_async_commit();
    };
    float ks0, ks1, vs0, vs1;                                  // scales of the two blocks in use
    auto scales = [&](int n) {                                 // of the warp's n-th two blocks
      const int at = 2 * (n & 15);
      ks0 = __shfl_sync(0xffffffffu, lks, at);
      ks1 = __shfl_sync(0xffffffffu, lks, at + 1);
      vs0 = __shfl_sync(0xffffffffu, lvs, at);
      vs1 = __shfl_sync(0xffffffffu, lvs, at + 1);
    };
    // ---- q fragments: two words' dims of the pieces at a time; warp i makes [.][i]
    float qf[NT];
    u128 raw[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i)                              // 8 dims at (i / 2) * 64 + qd * 16 + (i % 2) * 8
        raw[nt][i] = gq + 8 * nt < G ? ld_v4(q + (size_t)b * ldq + (size_t)(h * G + gq + 8 * nt) * D + (i >> 1) * 64 +
                                             qd * 16 + (i & 1) * 8)
                                     : u128{0, 0, 0, 0};
    uint32_t s0 = ring, s1 = ring + SLOT, s2 = ring + 2 * SLOT;   // K in use, V in use, the next K
    fetch_k(s0);
    fetch_v(s1);
    fetch_k(s2);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float am = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          am = fmaxf(am, fmaxf(finite_or_zero(bf16_lo(word(raw[nt][i], e))), finite_or_zero(bf16_hi(word(raw[nt][i], e)))));
      am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 1));
      am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 2));
      // am * 2^-eq in [2^14, 2^15)
      const int eq = am > 0.f ? max((int)(__float_as_uint(am) >> 23) - 127 - 14, -126) : 0;
      const float down = exp2_int(-eq);
      qf[nt] = exp2_int(eq) * scale_log2;
      static_assert(WARPS == 4, "a warp per two words");
      const u128 mine = warp == 0 ? raw[nt][0] : warp == 1 ? raw[nt][1] : warp == 2 ? raw[nt][2] : raw[nt][3];
      uint32_t f[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = pack_f16x2(bf16_lo(word(mine, e)) * down, bf16_hi(word(mine, e)) * down);
      sq[(nt * 4 + warp) * 32 + lane] = make_uint4(f[0], f[1], f[2], f[3]);
    }
    __syncthreads();

    float o[NT][8][4];
    float m[NT], l[NT], mv[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt] = mv[nt] = -INFINITY;
      l[nt] = 0.f;
#pragma unroll
      for (int mt = 0; mt < 8; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][mt][e] = 0.f;
    }
    scales(0);
    for (int j = j0 + 2 * warp; j < j1; j += 2 * WARPS) {
      cp_async_wait<2>();                                      // K of these blocks
      __syncwarp();                                            // of every lane
      float s[2][2][4];                                        // [block][tokens 0-7, 8-15]
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][0][e] = s[i][1][e] = 0.f;
#pragma unroll
      for (int p = 0; p < 2; ++p) {                            // pieces: 64 dims each
        u128 kr[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int tt = 0; tt < 2; ++tt) kr[i][tt] = lds16(s0 + kget + p * khalf + i * (BS * D) + tt * 8 * D);
#pragma unroll
        for (int w2 = 0; w2 < 2; ++w2) {                       // two words
          uint4 qa[NT];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) qa[nt] = sq[(nt * 4 + 2 * p + w2) * 32 + lane];
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
              const uint32_t wa = word(kr[i][tt], 2 * w2), wb = word(kr[i][tt], 2 * w2 + 1);
              mma_f16(s[i][tt], qa[0].x, NT == 2 ? qa[NT - 1].x : 0u, qa[0].y, NT == 2 ? qa[NT - 1].y : 0u,
                      e4m3x2_to_f16x2((uint16_t)wa), e4m3x2_to_f16x2((uint16_t)(wa >> 16)));
              mma_f16(s[i][tt], qa[0].z, NT == 2 ? qa[NT - 1].z : 0u, qa[0].w, NT == 2 ? qa[NT - 1].w : 0u,
                      e4m3x2_to_f16x2((uint16_t)wb), e4m3x2_to_f16x2((uint16_t)(wb >> 16)));
            }
        }
      }
      __syncwarp();                                            // K has been read by all
      fetch_v(s0);                                             // of the next blocks
      float x[NT][8];                                          // logits: 4 of each block
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float f0 = qf[nt] * ks0, f1 = qf[nt] * ks1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[nt][e] = ks0 < 0.f ? -INFINITY : s[0][e >> 1][2 * nt + (e & 1)] * f0;   // below 0: no block
          x[nt][4 + e] = ks1 < 0.f ? -INFINITY : s[1][e >> 1][2 * nt + (e & 1)] * f1;
        }
      }
      const int tok0 = j * BS + 2 * qd;                        // this lane's tokens: + {0, 1, 8, 9} of each block
      const bool tail = (j + 2) * BS > len;
      if (tail) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (tok0 + (e & 1) + ((e >> 1) & 1) * 8 + (e >> 2) * BS >= len)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) x[nt][e] = -INFINITY;
      }
      const float e0 = (float)((int)(__float_as_uint(vs0) >> 23) - 127);
      const float e1 = (float)((int)(__float_as_uint(vs1) >> 23) - 127);
      uint32_t wb[NT][4];                                      // weights: B fragments of the second product
      float alpha[NT];
      bool grow = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float a0 = fmaxf(fmaxf(x[nt][0], x[nt][1]), fmaxf(x[nt][2], x[nt][3]));
        float a1 = fmaxf(fmaxf(x[nt][4], x[nt][5]), fmaxf(x[nt][6], x[nt][7]));
        a0 = fmaxf(a0, __shfl_xor_sync(0xffffffffu, a0, 1));
        a1 = fmaxf(a1, __shfl_xor_sync(0xffffffffu, a1, 1));
        a0 = fmaxf(a0, __shfl_xor_sync(0xffffffffu, a0, 2));
        a1 = fmaxf(a1, __shfl_xor_sync(0xffffffffu, a1, 2));
        const float m_new = fmaxf(m[nt], fmaxf(a0, a1)), base = m_new == -INFINITY ? 0.f : m_new;
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = ex2(x[nt][e] - base);
        l[nt] = l[nt] * ex2(m[nt] - base) + (((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7])));
        m[nt] = m_new;
        const float mt = fmaxf(a0 + e0, a1 + e1);              // of x + log2 of V's scale
        alpha[nt] = 1.f;
        if (mt > mv[nt] + RESCALE || mv[nt] == -INFINITY) {
          alpha[nt] = mt == -INFINITY ? 1.f : ex2(mv[nt] - mt);
          mv[nt] = mt;
          grow = true;
        }
        // p 2^(e + m - mv); the bound keeps blocks whose scales are 2^126 apart finite
        const float vb = base - (mv[nt] == -INFINITY ? 0.f : mv[nt]);
        const float c0 = ex2(fminf(e0 + vb, 126.f)), c1 = ex2(fminf(e1 + vb, 126.f));
#pragma unroll
        for (int i = 0; i < 4; ++i) wb[nt][i] = pack_f16x2(p[2 * i] * (i < 2 ? c0 : c1), p[2 * i + 1] * (i < 2 ? c0 : c1));
      }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {                      // O^T's columns are heads 2 qd, 2 qd + 1
          const float a0 = __shfl_sync(0xffffffffu, alpha[nt], 8 * qd), a1 = __shfl_sync(0xffffffffu, alpha[nt], 8 * qd + 4);
#pragma unroll
          for (int mt = 0; mt < 8; ++mt) {
            o[nt][mt][0] *= a0;
            o[nt][mt][1] *= a1;
            o[nt][mt][2] *= a0;
            o[nt][mt][3] *= a1;
          }
        }
      }
      cp_async_wait<2>();                                      // V of these blocks
      __syncwarp();
      const bool gaps = tail || ks0 < 0.f || ks1 < 0.f;
#pragma unroll
      for (int w2 = 0; w2 < 2; ++w2) {                         // 8 dims of each token: MMA tiles 4 w2 ..
        uint2 vr[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) vr[e] = lds8(s1 + vget + (e >> 2) * (BS * D) + ((e >> 1 & 1) * 8 + (e & 1)) * D + 8 * (w2 ^ vhalf));
        if (gaps) {                                            // rows never written: 0 x NaN would poison O
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (tok0 + (e & 1) + ((e >> 1) & 1) * 8 + (e >> 2) * BS >= len || (e < 4 ? ks0 : ks1) < 0.f)
              vr[e] = make_uint2(0, 0);
        }
#pragma unroll
        for (int w = 0; w < 2; ++w) {                          // 4 dims: two tiles
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t t0 = w ? vr[4 * i].y : vr[4 * i].x, t1 = w ? vr[4 * i + 1].y : vr[4 * i + 1].x,
                           t2 = w ? vr[4 * i + 2].y : vr[4 * i + 2].x, t3 = w ? vr[4 * i + 3].y : vr[4 * i + 3].x;
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {                   // bytes of two tokens side by side: dims 2 hf, 2 hf + 1
              const uint32_t y = __byte_perm(t0, t1, hf ? 0x7362 : 0x5140), z = __byte_perm(t2, t3, hf ? 0x7362 : 0x5140);
              const uint32_t a0 = e4m3x2_to_f16x2((uint16_t)y), a1 = e4m3x2_to_f16x2((uint16_t)(y >> 16));
              const uint32_t a2 = e4m3x2_to_f16x2((uint16_t)z), a3 = e4m3x2_to_f16x2((uint16_t)(z >> 16));
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma_f16(o[nt][4 * w2 + 2 * w + hf], a0, a1, a2, a3, wb[nt][2 * i], wb[nt][2 * i + 1]);
            }
          }
        }
      }
      __syncwarp();                                            // V has been read by all
      scales(fcount - 1);                                      // before the fetch may replace them
      fetch_k(s1);
      const uint32_t t = s0;                                   // next: K in s2, V in s0, the K after it in s1
      s0 = s2;
      s2 = s1;
      s1 = t;
    }
    cp_async_wait<0>();
    __syncthreads();                                           // every warp has drained its ring

    // ---- the warps' results of this run
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float ls = l[nt];
      ls += __shfl_xor_sync(0xffffffffu, ls, 1);
      ls += __shfl_xor_sync(0xffffffffu, ls, 2);
      if (qd == 0) *reinterpret_cast<float4*>(sm + (warp * 8 * NT + nt * 8 + gq) * 4) = make_float4(m[nt], ls, mv[nt], 0.f);
      // dim gq * 16 + k of a head in column k * 8 + gq
#pragma unroll
      for (int mt = 0; mt < 8; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          so[(warp * 8 * NT + nt * 8 + 2 * qd + (e & 1)) * O_ROW + (2 * (mt ^ 4 * vhalf) + (e >> 1)) * 8 + gq] = o[nt][mt][e];
    }
    __syncthreads();
    // the CTAs that share the pair: those of the cuts left inside it, and the one before
    const int slack = slack_of(units), c0 = (pair0 + PAIR_COST + slack) / per, c1 = (pair0 + units - slack - 1) / per;
    // two heads at a time, a thread for two dims of one
    for (int hh = tid >> 6; hh < G; hh += 2) {
      const int d16 = tid & 7, d2 = tid >> 3 & 7, dim = d16 * 16 + 2 * d2;
      float4 st[WARPS];
      float M = -INFINITY, MV = -INFINITY;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        st[w] = *reinterpret_cast<const float4*>(sm + (w * 8 * NT + hh) * 4);
        M = fmaxf(M, st[w].x);
        MV = fmaxf(MV, st[w].z);
      }
      const float mb = M == -INFINITY ? 0.f : M, vb = MV == -INFINITY ? 0.f : MV;
      float2 num = make_float2(0.f, 0.f);
      float den = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float* p = so + (w * 8 * NT + hh) * O_ROW + 16 * d2 + d16;
        const float f = ex2(st[w].z - vb);
        num.x += p[0] * f;
        num.y += p[8] * f;
        den += st[w].y * ex2(st[w].x - mb);
      }
      if (c0 >= c1) {
        const float inv = den == 0.f ? 0.f : ex2(vb - mb) / den;
        *reinterpret_cast<uint32_t*>(out + (size_t)b * ldo + (size_t)(h * G + hh) * D + dim) =
            pack_bf16x2(num.x * inv, num.y * inv);
      } else {   // slot 1 for the pair that goes on in the next CTA, 0 for one that began before
        float* p = part + ((size_t)(blockIdx.x * 2 + ((int)blockIdx.x == c0)) * G + hh) * DEC8_ROW;
        *reinterpret_cast<float2*>(p + dim) = num;
        if ((tid & 63) == 0) {
          *reinterpret_cast<float4*>(p + D) = make_float4(M, den, MV, 0.f);
        }
      }
    }
    if (c0 < c1) {
      __threadfence();
      __syncthreads();
      if (tid == 0) ticket = atomicInc(&counters[b * Hkv + h], (uint32_t)(c1 - c0));
      __syncthreads();
      if (ticket == (uint32_t)(c1 - c0)) {
        __threadfence();
        // a warp per head: lanes over the CTAs for the statistics, over the dims for the sums
        for (int hh = warp; hh < G; hh += WARPS) {
          auto slot = [&](int cc) {
            return part + ((size_t)(cc * 2 + (cc == c0)) * G + hh) * DEC8_ROW;
          };
          float m_all = -INFINITY, mv_all = -INFINITY, den = 0.f;
          float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int cb = c0; cb <= c1; cb += 32) {              // 32 CTAs at a time, rescaled as the maxima grow
            const int n = min(32, c1 - cb + 1);
            const float4 st = lane < n ? __ldcg(reinterpret_cast<const float4*>(slot(cb + lane) + D))
                                       : make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
            float4 x[8];
            auto rows = [&](int i) {
#pragma unroll
              for (int k = 0; k < 8; ++k)
                x[k] = i + k < n ? __ldcg(reinterpret_cast<const float4*>(slot(cb + i + k)) + lane)
                                 : make_float4(0.f, 0.f, 0.f, 0.f);
            };
            rows(0);                                           // on their way while the maxima are found
            const float m_new = fmaxf(m_all, warp_max(st.x)), mv_new = fmaxf(mv_all, warp_max(st.z));
            const float mb = m_new == -INFINITY ? 0.f : m_new, vb = mv_new == -INFINITY ? 0.f : mv_new;
            const float fv = ex2(mv_all - vb);
            den = den * ex2(m_all - mb) + st.y * ex2(st.x - mb);
            num.x *= fv;
            num.y *= fv;
            num.z *= fv;
            num.w *= fv;
            m_all = m_new;
            mv_all = mv_new;
            const float f = ex2(st.z - vb);
            for (int i = 0; i < n; i += 8) {
              float4 y[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) y[k] = x[k];
              if (i + 8 < n) rows(i + 8);
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const float g = __shfl_sync(0xffffffffu, f, (i + k) & 31);
                if (i + k < n) {
                  num.x += y[k].x * g;
                  num.y += y[k].y * g;
                  num.z += y[k].z * g;
                  num.w += y[k].w * g;
                }
              }
            }
          }
          const float mb = m_all == -INFINITY ? 0.f : m_all, vb = mv_all == -INFINITY ? 0.f : mv_all;
          den = warp_sum(den);
          const float inv = den == 0.f ? 0.f : ex2(vb - mb) / den;
          uint2 w;
          w.x = pack_bf16x2(num.x * inv, num.y * inv);
          w.y = pack_bf16x2(num.z * inv, num.w * inv);
          *reinterpret_cast<uint2*>(out + (size_t)b * ldo + (size_t)(h * G + hh) * D + 4 * lane) = w;
        }
      }
    }
    __syncthreads();                                           // O and the statistics have been read
  }
}

int decode_fp8_ctas(int sms) { return sms * dec8::ctas_per_sm(1); }
// The shares are equal, so one more CTA than an SM holds would run a whole share after the others: the
// grid counts what fits, by registers and beside the prefix sums (four up to about 1400 sequences, then
// three).  64 x 4096 tokens of 128/8 heads take 103 us, 131 with four CTAs' shares on an SM; of 16/1 heads
// 25 and 41; 2000 x 128 of 32/8 heads 163 and 205, 4096 x 64 of 8/2 heads 89 and 119.
int decode_fp8_resident(int B, int G) {
  const int nt = G > 8 ? 2 : 1;
  const int smem = nt == 2 ? dec8::Smem<2>::bytes(B) : dec8::Smem<1>::bytes(B);
  constexpr int PER_SM = 228 * 1024, OTHER = 1024 + 256;      // of a CTA: the system's, and the static variables
  return std::min(dec8::ctas_per_sm(nt), PER_SM / (smem + OTHER));
}
long decode_fp8_rows(int sms, int B, int Hkv, int G) {
  const long row = (long)G * DEC8_ROW;
  return 2L * decode_fp8_ctas(sms) + ((long)B * Hkv + row - 1) / row;
}

void decode_attention_fp8(const void* q, int ldq, const KvFp8& c, const int* block_tables, int max_blocks,
                          const int* ctx_lens, void* out, int ldo, int B, int Hq, float scale, float* ws, long ws_rows,
                          int sms, int* status, cudaStream_t s) {
  if (B == 0) return;
  const int G = Hq / c.Hkv;
  const int ctas = decode_fp8_ctas(sms);
  // the partial results (room for the largest grid) sit at the front, the counters behind them: neither
  // moves with the batch
  uint32_t* counters = reinterpret_cast<uint32_t*>(ws + 2L * ctas * G * DEC8_ROW);
  const int nt = G > 8 ? 2 : 1;
  const long most = ((long)B * c.Hkv * (max_blocks + dec8::PAIR_COST) + dec8::MIN_UNITS - 1) / dec8::MIN_UNITS;
  const int grid = (int)std::max(1L, std::min((long)sms * decode_fp8_resident(B, G), most));
  const int smem = nt == 2 ? dec8::Smem<2>::bytes(B) : dec8::Smem<1>::bytes(B);
  auto kern = nt == 2 ? decode_attn_fp8_kernel<2> : decode_attn_fp8_kernel<1>;
  static bool attr[64][2] = {};
  int dev;
  cudaGetDevice(&dev);
  if (!attr[dev & 63][nt - 1]) {
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                         nt == 2 ? dec8::Smem<2>::bytes(DEC8_MAX_BATCH) : dec8::Smem<1>::bytes(DEC8_MAX_BATCH));
    cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
    attr[dev & 63][nt - 1] = true;
  }
  kern<<<grid, dec8::THREADS, smem, s>>>(reinterpret_cast<const __nv_bfloat16*>(q), ldq, c, block_tables, max_blocks,
                                         ctx_lens, reinterpret_cast<__nv_bfloat16*>(out), ldo, B, Hq,
                                         scale * 1.4426950408889634f, ws, counters, status);
}

// ------------------------------------------------------------ block copies
// A CTA moves one pair's block in a run of planes.  A pair whose destination
// is another pair's source, or the destination of another source, has no
// defined result: it is left out and recorded.  The check is a scan of the
// pairs while the first vectors are in flight.
namespace kvc {
constexpr int THREADS = 256;
}
__global__ void __launch_bounds__(kvc::THREADS)
    kv_copy_blocks_kernel(uint8_t* kv, float* scales, const int* __restrict__ pairs, int n, int planes, int per,
                          int num_blocks, int64_t block_bytes, int Hkv, int* status) {
  const int i = blockIdx.x, tid = threadIdx.x;
  const int src = pairs[2 * i], dst = pairs[2 * i + 1];
  const int p0 = blockIdx.y * per, p1 = min(planes, p0 + per);
  if (src < 0 || src >= num_blocks || dst < 0 || dst >= num_blocks) {
    if (tid == 0) record_status(status, CX_ERR_BOUNDS);
    return;
  }
  if (src == dst) return;
  // the planes' vectors end to end, eight of a thread in flight
  const int nv = (int)(block_bytes >> 4);
  const int64_t plane = (int64_t)num_blocks * block_bytes;
  const uint8_t* a = kv + p0 * plane + src * block_bytes;
  uint8_t* b = kv + p0 * plane + dst * block_bytes;
  const int total = (p1 - p0) * nv;
  int v = tid;                    // the thread's next vector of plane `at`
  int64_t at = 0;
  u128 r[8];
  int64_t off[8];
  auto load = [&](int i) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      while (v >= nv) {
        v -= nv;
        at += plane;
      }
      off[e] = at + (int64_t)v * 16;
      if (i + e * kvc::THREADS < total) r[e] = ld_nc_v4(a + off[e]);
      v += kvc::THREADS;
    }
  };
  load(tid);
  bool bad = false;
  for (int k = tid; k < n; k += kvc::THREADS) {
    const int s = pairs[2 * k], d = pairs[2 * k + 1];
    bad |= (s == dst && d != dst) || (d == dst && s != src);
  }
  if (__syncthreads_or(bad)) {
    if (tid == 0) record_status(status, CX_ERR_BOUNDS);
    return;
  }
  for (int i = tid; i < total;) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (i + e * kvc::THREADS < total) st_cs_v4(b + off[e], r[e]);
    i += 8 * kvc::THREADS;
    if (i < total) load(i);
  }
  if (scales != nullptr)
    for (int i = tid; i < (p1 - p0) * Hkv; i += kvc::THREADS) {
      const int64_t row = (int64_t)(p0 + i / Hkv) * num_blocks;
      scales[(row + dst) * Hkv + i % Hkv] = scales[(row + src) * Hkv + i % Hkv];
    }
}

void kv_copy_blocks(void* kv, float* scales, const int* pairs, int n, int planes, int num_blocks, int64_t block_bytes,
                    int Hkv, int sms, int* status, cudaStream_t s) {
  if (n == 0 || planes == 0) return;
  const long want = 8L * sms;
  const int per = (int)std::max(1L, std::min((long)planes, (long)n * planes / want));
  kv_copy_blocks_kernel<<<dim3(n, (planes + per - 1) / per), kvc::THREADS, 0, s>>>(
      reinterpret_cast<uint8_t*>(kv), scales, pairs, n, planes, per, num_blocks, block_bytes, Hkv, status);
}

// --------------------------------------------------------- dequantised blocks
// The blocks that the tiles of a chunked prefill read, as bf16 (exact: the
// scales are powers of two), sequence after sequence, and the tables that find
// them there.  Bound by memory and short next to the attention that
// follows: 12 of 211 us for 2048 rows at 6144.  (Converting inside the
// attention kernel, by four more warps between the copies and the MMAs, took
// 302 us where two launches took 225: the thread that issues the MMAs is busy
// 83 % of its time, and a converter on its SM quarter slows it.)
// One CTA per block: all heads of K, then of V, 16 bytes of a lane each.  The
// first CTA also hands on the tiles that fit the rows and the tables -- the
// attention kernel takes them as they are -- and divides their work.
//
// The work: an item is 256 rows (tokens of a tile by query heads) for each CTA
// of a team, its length its key tiles and ITEM_COST for its fixed cost.  The
// items, laid end to end, are cut into equal shares, one per team; a cut within
// CUT_SLACK of an item's start or end moves there.  Against one item per CTA at a time, the conversion
// not counted in the latter: 256 rows at 7936 60 and 121 us, 2 x 256 at 32256
// 263 and 465, 2048 rows at 6144 201 and 211; eight prompts of 2048, whose items
// balance by themselves, 295 and 271: there the cuts only cost.
namespace kvd {
constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int ROWS = 256, KEYS = 128;                   // of a tile of the attention
constexpr int ITEM_COST = 2;                            // 4 x 512 rows at 8192: 302 us, 311 with 1, 320 with 4
constexpr int CUT_SLACK = 1;                            // 2048 rows at 6144: 210 us, 215 with 3
constexpr int MIN_SHARE = 3;                            // less is all fixed cost: 131 rows at 2000 31 us, 34 with 4
}
__device__ __forceinline__ bool tile_fits(const int* ti, int T, int B, int width) {
  const int start = ti[0], n = ti[1], q0 = ti[2], ctx = ti[3], seq = ti[4];
  return seq >= 0 && seq < B && n > 0 && q0 >= 0 && q0 < n && ctx >= 0 && start >= 0 && (int64_t)start + n <= T &&
         (int64_t)ctx + n <= (int64_t)width * kvq::BS;
}
// key tiles of `tokens` queries from q0
__device__ __forceinline__ int tile_keys(const int* ti, int q0, int tokens) {
  return (min(ti[3] + ti[1], ti[3] + q0 + tokens) + kvd::KEYS - 1) / kvd::KEYS;
}
__device__ __forceinline__ void kv_prefill_plan(const int* __restrict__ tile_info, int n_tiles, int T, int B, int width,
                                                int Hq, const KvChunks& o, int* status) {
  using namespace kvd;
  __shared__ int64_t wlen[WARPS];
  __shared__ int wfit[WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, tokens = ROWS >> o.pack;
  int64_t len = 0;                                      // of the tiles so far, for one set of heads
  int kept = 0;
  __shared__ int longest;
  if (tid == 0) longest = 0;
  __syncthreads();
  for (int t0 = 0; t0 < n_tiles; t0 += THREADS) {
    const int t = t0 + tid;
    const int* ti = tile_info + 5 * (int64_t)t;
    const bool fits = t < n_tiles && tile_fits(ti, T, B, width);
    if (t < n_tiles && !fits) record_status(status, CX_ERR_BOUNDS);
    int parts = 0;                                      // items of the tile for one set of heads
    int64_t n = 0;                                      // their length
    if (fits)
      for (int q0 = ti[2], q1 = min(ti[1], ti[2] + ROWS); q0 < q1; q0 += tokens, ++parts)
        n += tile_keys(ti, q0, tokens) + ITEM_COST;
    if (fits) atomicMax(&longest, tile_keys(ti, ti[2], ROWS));
    int64_t x = n;
    int y = parts;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t xu = __shfl_up_sync(0xffffffffu, x, d);
      const int yu = __shfl_up_sync(0xffffffffu, y, d);
      if (lane >= d) {
        x += xu;
        y += yu;
      }
    }
    if (lane == 31) {
      wlen[warp] = x;
      wfit[warp] = y;
    }
    __syncthreads();
    int64_t at = len + x - n;
    int to = kept + y - parts;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) {
        at += wlen[w];
        to += wfit[w];
      }
      len += wlen[w];
      kept += wfit[w];
    }
    for (int k = 0; k < parts; ++k, ++to) {
      for (int e = 0; e < 5; ++e) o.tiles[5 * (int64_t)to + e] = ti[e] + (e == 2 ? k * tokens : 0);
      o.before[to] = at;
      at += tile_keys(ti, ti[2] + k * tokens, tokens) + ITEM_COST;
    }
    __syncthreads();
  }
  for (int i = tid; i < 2 * o.n_cta; i += THREADS) o.arrived[i] = 0;
  const int teams = o.n_cta / o.team, each = (Hq >> o.pack) / o.team;     // items of a tile
  // A piece costs its item's merge about what a key tile costs its CTA: shares of at least sqrt(length)
  // (chunks of 131, 45, 3, 4 and 1 rows: 34 us, 36 with 1.4 times that, 38 with 1.8; 48 rows at 30000 with
  // 8/1 heads 68, 72 with 0.7 times, 119 without).
  const int least = max(MIN_SHARE, (int)sqrtf((float)longest));
  const int64_t total = len * each, per = max((int64_t)least, (total + teams - 1) / teams);
  for (int i = tid; i <= teams; i += THREADS) {
    const int64_t x = i * per;
    int2 cut = make_int2(kept * each, 0);
    if (x < total) {
      int lo = 0, hi = kept;                            // the tile that holds x
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (o.before[mid] * each <= x) lo = mid;
        else hi = mid;
      }
      const int n = tile_keys(o.tiles + 5 * (int64_t)lo, o.tiles[5 * (int64_t)lo + 2], tokens) + ITEM_COST;
      const int64_t in = x - o.before[lo] * each;
      const int h = (int)(in / n), p = (int)(in - (int64_t)h * n);
      const int slack = min((n - ITEM_COST) / 2, CUT_SLACK);
      cut = p <= ITEM_COST + slack ? make_int2(lo * each + h, 0)
            : n - p <= slack       ? make_int2(lo * each + h + 1, 0)
                                   : make_int2(lo * each + h, p - ITEM_COST);
    }
    o.cuts[i] = cut;
  }
}
__global__ void __launch_bounds__(kvd::THREADS)
    kv_dequant_kernel(KvFp8 c, const int* __restrict__ tables, int B, int width, const int* __restrict__ tile_info,
                      int n_tiles, int T, int Hq, KvChunks out, int* status) {
  using namespace kvq;
  extern __shared__ int from[];                         // [B + 1]: blocks of the sequences before b
  __shared__ int wsum[kvd::WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int b = tid; b <= B; b += kvd::THREADS) from[b] = 0;
  __syncthreads();
  // blocks of a sequence: any of its tiles tells
  for (int t = tid; t < n_tiles; t += kvd::THREADS) {
    const int* ti = tile_info + 5 * (int64_t)t;
    if (tile_fits(ti, T, B, width)) atomicMax(&from[1 + ti[4]], (ti[1] + ti[3] + BS - 1) / BS);
  }
  __syncthreads();
  int total = 0;
  for (int b0 = 0; b0 < B; b0 += kvd::THREADS) {
    const int b = b0 + tid;
    int x = b < B ? from[1 + b] : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += y;
    }
    if (lane == 31) wsum[warp] = x;
    __syncthreads();
    int add = total;
#pragma unroll
    for (int w = 0; w < kvd::WARPS; ++w) {
      if (w < warp) add += wsum[w];
      total += wsum[w];
    }
    if (b < B) from[1 + b] = add + x;
    __syncthreads();
  }
  auto entry = [&](int i) {                             // of the tables: the i-th that is read
    int lo = 0, hi = B;                                 // the sequence: the last one with from[lo] <= i
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (from[mid] <= i) lo = mid;
      else hi = mid;
    }
    return (int64_t)lo * width + i - from[lo];
  };
  if (blockIdx.x == 0) {
    kv_prefill_plan(tile_info, n_tiles, T, B, width, Hq, out, status);
    if (total > out.blocks && tid == 0) record_status(status, CX_ERR_BOUNDS);
    for (int i = out.blocks + tid; i < total; i += kvd::THREADS) out.tables[entry(i)] = 0;   // no room: any block
  }
  const int i = blockIdx.x;
  if (i >= min(total, out.blocks)) return;
  const int64_t at = entry(i);
  if (tid == 0) out.tables[at] = i;
  const int id = tables[at];
  const bool in = id >= 0 && id < c.num_blocks;
  if (!in && tid == 0) record_status(status, CX_ERR_BOUNDS);
  __nv_bfloat16 *ko = reinterpret_cast<__nv_bfloat16*>(out.k), *vo = reinterpret_cast<__nv_bfloat16*>(out.v);
  const int per = c.Hkv * (BS * D / 16);                // 16-byte pieces of K, and of V
#pragma unroll 4
  for (int v = tid; v < 2 * per; v += kvd::THREADS) {
    const bool is_v = v >= per;
    const int e = (is_v ? v - per : v) * 16, h = e / (BS * D);
    u128 raw{0, 0, 0, 0};                               // an id out of range reads as zeros
    float f = 0.f;
    if (in) {
      raw = ld_nc_v4((is_v ? c.v : c.k) + (size_t)id * c.Hkv * (BS * D) + e);
      f = (is_v ? c.vs : c.ks)[(size_t)id * c.Hkv + h];
    }
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw);
    u128 o[2];
    uint32_t* po = reinterpret_cast<uint32_t*>(o);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t a = e4m3x2_to_f16x2((uint16_t)w[k]), b = e4m3x2_to_f16x2((uint16_t)(w[k] >> 16));
      po[2 * k] = pack_bf16x2(f16_lo(a) * f, f16_hi(a) * f);
      po[2 * k + 1] = pack_bf16x2(f16_lo(b) * f, f16_hi(b) * f);
    }
    __nv_bfloat16* d = (is_v ? vo : ko) + (size_t)i * c.Hkv * (BS * D) + e;
    st_v4(d, o[0]);
    st_v4(d + 8, o[1]);
  }
}

void kv_dequant_blocks(const KvFp8& c, const int* tables, int B, int width, const int* tile_info, int n_tiles, int T,
                       int Hq, const KvChunks& o, int* status, cudaStream_t s) {
  if (B == 0 || width == 0) return;
  kv_dequant_kernel<<<std::max(1, o.blocks), kvd::THREADS, (B + 1) * sizeof(int), s>>>(c, tables, B, width, tile_info,
                                                                                       n_tiles, T, Hq, o, status);
}

}  // namespace cx
