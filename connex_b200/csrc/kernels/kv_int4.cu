// The 4-bit paged KV cache: quantising write, its values, decode attention over
// it.  (Chunked prefill turns the blocks into bf16, as for the 8-bit cache.)
//
//   minimum = min x,  scale = (max x - min x) / 15,  code = round((x - minimum) / scale)
//
// over the 64 dims of a half of a token's head: the halves that RoPE rotates
// with one another.  With a minimum, all 16 levels lie between the extremes
// also for keys whose channels have a mean.  Scale and minimum are bf16 and lie
// in the token's own row: a token is written without reading its block, and a
// block is copied, shared or moved as bytes.
#include <algorithm>
#include <stdexcept>

#include "decode_split.cuh"
#include "fewbit.cuh"
#include "kv_int4.h"

namespace cx {

namespace kv4 {
constexpr int D = 128, BS = 16, ROW = KV4_ROW;
constexpr int THREADS = 256, WARPS = THREADS / 32;
// Up to two rounds of warps of eight heads on 148 SMs, warps of four: 64 rows of 32/8 heads take 2.6 us (3.4), 1024 rows
// 7.4 (8.1); beyond, the positions and angles that each warp reads again cost more: 8192 rows 44.7 (41.3).
constexpr int64_t FEW_UNITS = 9472;
constexpr uint32_t NAN_PAIR = 0x7fff7fffu;     // scale and minimum of a half without finite range
}  // namespace kv4

// --------------------------------------------------- RoPE + quantising write
// Eight bf16 dims of a lane, eight lanes to a half: scale | minimum << 16, and
// the lane's codes.
__device__ __forceinline__ uint32_t quant4(const uint32_t (&w)[4], uint32_t& codes) {
  float v[8], lo, hi;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = bf16_lo(w[i]);
    v[2 * i + 1] = bf16_hi(w[i]);
    odd |= (w[i] & 0x7f80u) == 0x7f80u || (w[i] & 0x7f800000u) == 0x7f800000u;
  }
  lo = hi = v[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = fminf(lo, v[i]);
    hi = fmaxf(hi, v[i]);
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  const __nv_bfloat16 sb = __float2bfloat16_rn(__fdiv_rn(hi - lo, 15.f));
  const float s = __bfloat162float(sb);
  odd |= !(s < INFINITY);                                // the range is no finite number
  const uint32_t mates = 0xffu << (threadIdx.x & 24);
  odd = (__ballot_sync(0xffffffffu, odd) & mates) != 0;
  codes = 0;
  if (odd) return kv4::NAN_PAIR;
  const float inv = s > 0.f ? fminf(__fdiv_rn(1.f, s), 3.4028234e38f) : 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) codes |= min(__float2uint_rn((v[i] - lo) * inv), 15u) << (4 * i);
  return (uint32_t)__bfloat16_as_ushort(sb) | (__float_as_uint(lo) & 0xffff0000u);   // lo is one of the bf16 values
}

// A warp: 2 PAIRS heads of a token, two at a time, eight dims of a lane.  q's
// heads are rotated, k's rotated and quantised, v's quantised.
// What bounds it: instructions.  8192 rows of 32/8 heads take 41 us, 177 MB at 4.3 TB/s (more warps on an SM, with fewer
// registers each, 44 to 60; the rotation's products one by one and 64-bit divisions 44); 64 rows 2.6, a launch and
// three dependent loads.
template <int PAIRS>
__global__ void __launch_bounds__(kv4::THREADS)
    rope_cache_int4_kernel(const __nv_bfloat16* qkv, int ldq, const int* __restrict__ pos,
                           const float* __restrict__ cos_sin, const int64_t* __restrict__ slots, KvInt4 c,
                           __nv_bfloat16* out, int ldo, uint32_t units, uint32_t per_token, int Hq, int max_pos, int* status,
                           const __nv_bfloat16* __restrict__ qn, const __nv_bfloat16* __restrict__ kn, float eps) {
  using namespace kv4;
  const int lane = threadIdx.x & 31, j = lane & 15;
  const uint32_t u = blockIdx.x * WARPS + (threadIdx.x >> 5);
  if (u >= units) return;
  const int64_t t = u / per_token;
  const int Hkv = c.Hkv, heads = Hq + 2 * Hkv, h0 = 2 * PAIRS * (int)(u - (uint32_t)t * per_token) + (lane >> 4);
  u128 raw[PAIRS];
#pragma unroll
  for (int k = 0; k < PAIRS; ++k)
    raw[k] = h0 + 2 * k < heads ? ld_v4(qkv + t * ldq + (int64_t)(h0 + 2 * k) * D + 8 * j) : u128{0, 0, 0, 0};
  const int p = pos[t];
  const int64_t slot = slots[t];
  const bool pos_ok = p >= 0 && p < max_pos, cached = pos_ok && slot >= 0 && (slot >> 4) < c.num_blocks;
  if (h0 == 0 && j == 0 && (!pos_ok || (slot >= 0 && !cached))) record_status(status, CX_ERR_BOUNDS);
  uint64_t co[4], si[4];                    // pairs
#pragma unroll
  for (int e = 0; e < 4; ++e) co[e] = si[e] = 0;
  if (pos_ok) {
    const ulonglong2* cs = reinterpret_cast<const ulonglong2*>(cos_sin + (int64_t)p * D + 8 * (j & 7));
    const uint64_t sign = j < 8 ? 0x8000000080000000ull : 0;         // a cos - b sin in the first half, a cos + b sin
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const ulonglong2 c2 = __ldg(cs + e), s2 = __ldg(cs + D / 8 + e);
      co[2 * e] = c2.x;
      co[2 * e + 1] = c2.y;
      si[2 * e] = s2.x ^ sign;
      si[2 * e + 1] = s2.y ^ sign;
    }
  }
#pragma unroll
  for (int k = 0; k < PAIRS; ++k) {
    const int h = h0 + 2 * k;
    uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
    const bool turned = h < Hq + Hkv;
    const __nv_bfloat16* nw = h < Hq ? qn : kn;
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) ss += bf16_lo(w[e]) * bf16_lo(w[e]) + bf16_hi(w[e]) * bf16_hi(w[e]);
    if (qn != nullptr || kn != nullptr) {
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      if (turned && nw != nullptr) {
        // bf16 between the norm and the rotation, like a norm layer of its own
        const float n = rsqrtf(ss * (1.0f / D) + eps);
        const u128 g = ld_v4(nw + 8 * j);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          w[e] = pack_bf16x2(bf16_lo(w[e]) * n * bf16_lo(word(g, e)), bf16_hi(w[e]) * n * bf16_hi(word(g, e)));
      }
    }
    uint32_t r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t b = __shfl_xor_sync(0xffffffffu, w[e], 8);      // the partner dims, 64 away
      // products and sums rounded each, as a bf16 cache's write rotates (a sum in pairs is made one with its product)
      const uint64_t x = mul_f32x2(unpack_bf16x2(w[e]), co[e]), y = mul_f32x2(unpack_bf16x2(b), si[e]);
      r[e] = pack_bf16x2(__fadd_rn(lo_f32(x), lo_f32(y)), __fadd_rn(hi_f32(x), hi_f32(y)));
    }
    if (h < Hq) {
      st_v4(out + t * ldo + (int64_t)h * D + 8 * j, u128{r[0], r[1], r[2], r[3]});   // a position out of range: zeros
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = turned ? r[e] : w[e];         // what a bf16 cache would hold is quantised
    if (!__any_sync(0xffffffffu, h >= Hq)) continue;
    uint32_t codes;
    const uint32_t par = quant4(w, codes);
    if (!cached || h < Hq || h >= heads) continue;
    const bool is_v = h >= Hq + Hkv;
    uint8_t* row = (is_v ? c.v : c.k) +
                   (((slot >> 4) * Hkv + (h - Hq - (is_v ? Hkv : 0))) * BS + (slot & 15)) * ROW;
    *reinterpret_cast<uint32_t*>(row + 4 * j) = codes;
    if ((j & 7) == 0) *reinterpret_cast<uint32_t*>(row + D / 2 + 4 * (j >> 3)) = par;
  }
}

void rope_cache_int4(const void* qkv, int ldq, const int* pos, const float* cos_sin, const int64_t* slots,
                     const KvInt4& c, void* out, int ldo, int T, int Hq, int max_pos, int* status, cudaStream_t s,
                     const void* q_norm, const void* k_norm, float eps) {
  if (T == 0) return;
  const int heads = Hq + 2 * c.Hkv;
  const bool few = (int64_t)T * ((heads + 7) / 8) <= kv4::FEW_UNITS;
  const int per_token = few ? (heads + 3) / 4 : (heads + 7) / 8;
  const int64_t units = (int64_t)T * per_token;
  if (units > UINT32_MAX - 64) throw std::runtime_error("rope_cache_int4: too many rows for one call");
  const unsigned ctas = (unsigned)((units + kv4::WARPS - 1) / kv4::WARPS);
  (few ? rope_cache_int4_kernel<2> : rope_cache_int4_kernel<4>)<<<ctas, kv4::THREADS, 0, s>>>(
      reinterpret_cast<const __nv_bfloat16*>(qkv), ldq, pos, cos_sin, slots, c, reinterpret_cast<__nv_bfloat16*>(out), ldo,
      (uint32_t)units, per_token, Hq, max_pos, status, reinterpret_cast<const __nv_bfloat16*>(q_norm),
      reinterpret_cast<const __nv_bfloat16*>(k_norm), eps);
}

// ------------------------------------------------------------------- values
// Eight dims of a lane: one word of codes, 16 bytes out.  Bytes bound it, nearly all of them written: 4096 blocks of 8
// heads take 32.6 us, 5.3 TB/s.
__global__ void __launch_bounds__(kv4::THREADS)
    kv_values_int4_kernel(const uint8_t* __restrict__ cache, __nv_bfloat16* __restrict__ out, int64_t words) {
  using namespace kv4;
  for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < words; i += (int64_t)gridDim.x * THREADS) {
    const uint8_t* row = cache + (i >> 4) * ROW;
    const int j = (int)(i & 15);
    st_v4(out + i * 8, int4_values(*reinterpret_cast<const uint32_t*>(row + 4 * j),
                                   *reinterpret_cast<const uint32_t*>(row + D / 2 + 4 * (j >> 3))));
  }
}

void kv_values_int4(const void* cache, void* out, int64_t rows, int sms, cudaStream_t s) {
  const int64_t words = rows * 16;
  if (words == 0) return;
  const int64_t ctas = std::min<int64_t>((words + kv4::THREADS - 1) / kv4::THREADS, (int64_t)sms * 8);
  kv_values_int4_kernel<<<(unsigned)ctas, kv4::THREADS, 0, s>>>(reinterpret_cast<const uint8_t*>(cache),
                                                                reinterpret_cast<__nv_bfloat16*>(out), words);
}

// ---------------------------------------------------------- decode attention
// S^T = K.q^T and O^T = V^T.W^T on mma.sync m16n8k16 (f16 in, fp32 out), the
// query heads of a KV head being an MMA's eight columns: bytes decide, and the
// instructions that take them apart, not tensor work.  A code needs no
// conversion: four bits under a mask are an f16 number already, the subnormal
// code * 2^-24 (the low half of a byte) or code * 2^-20 (the high half), exact in
// the product.  The factor 2^4 between the two kinds is part of q for K, and of
// O's rows for V.
//   K: lane (g = lane / 4, t = lane % 4) takes bytes [8 t, 8 t + 8) of a half of
//      tokens g and g + 8: 16 dims, two words.  The contraction may take the
//      dims in any order as long as q uses the same one.  S of each half comes
//      out by itself, heads 2t and 2t + 1 of the lane's two tokens; scale and
//      minimum are applied to it in fp32: x = sum_halves scale * S + minimum *
//      sum(q).
//   V: the weights, scale included (weight * scale, held in f16 relative to a running maximum of their own for each
//      half: see TOP_W), are turned round by movmatrix: the
//      lane then holds head g of tokens 2t, 2t + 1, 2t + 8, 2t + 9, of which it
//      takes word g of a half (8 dims), two tokens side by side.  The minimum's
//      part, sum of weight * minimum, is one fp32 number per half.
// q is scaled by a power of two per head into f16's range.  The running maxima
// move only once a weight has outgrown them by 2^8 and more, and the warp votes
// on that: the steps in between have no shuffles and no rescaling.
//
// Loads: a block of a head is 1152 contiguous bytes, one asynchronous bulk copy.
// A warp has K and V of two blocks in each of two stages, one read while the
// other is under way, without barriers between warps.
// What bounds it: 64 x 4096 tokens of 32/8 heads take 74.6 us, 302 MB at 4.05
// TB/s or 0.63 of a copy's rate.  42.6 million warp instructions keep the
// schedulers 57 % busy with 14 warps on an SM (128 registers each), the integer
// pipe 56 %, tensor cores 22 %: the masks and shifts that take the codes apart,
// in chains that four warps of a scheduler do not hide.  Tokens as columns of
// the first product, with a shuffle per maximum, took 99 us.  16 query heads of
// one KV head take 29.0 us for 64 x 4096, of four 69.3 (2.2 TB/s: twice the
// products for the bytes, three CTAs on an SM).
namespace dec4 {
struct Cfg {
  static constexpr int WARPS = 4, THREADS = 32 * WARPS, BS = kv4::BS;
  static constexpr int MIN_UNITS = 2 * WARPS, PAIR_COST = 4 * WARPS, SLACK = 2 * PAIR_COST;
};
constexpr int WARPS = Cfg::WARPS, THREADS = Cfg::THREADS, D = kv4::D, BS = kv4::BS, ROW = kv4::ROW;
constexpr int ctas_per_sm(int nt) { return nt == 1 ? 4 : 3; }
constexpr float LATE = 8.f;             // a logit may be this far above the running maximum: weights stay under 2^8
// The products weight * scale of a half are held in f16, times a power of two that makes the largest so far 2^TOP_W at
// least and lets it grow to MOST_W (a pair of 2^15) before it is chosen anew: each to 2^-11 of itself from 2^-22 of the
// largest up, and to 2^-33 of the largest below.  The power is at most 2^START: a weight (2^LATE at most) times that is
// finite.
constexpr int TOP_W = 8, START = 119;
constexpr uint32_t MOST_W = 0x78007800u;
constexpr int BLOCK = BS * ROW;         // of one head
constexpr int STAGE = 4 * BLOCK;        // K of two blocks, V of two blocks
constexpr int STAGES = 2;
constexpr int RING = WARPS * STAGES * STAGE;
constexpr int O_ROW = D + 4;            // floats of a head's row of O: eight lanes' stores fall on eight banks
template <int NT>
struct Smem {                           // rings, later the warps' O | their statistics | q fragments | barriers | sums
  static constexpr int STATS = RING;
  static_assert(WARPS * 8 * NT * O_ROW * 4 <= RING, "O fits in the drained rings");
  static constexpr int Q = STATS + WARPS * 8 * NT * 32;
  static constexpr int BAR = Q + NT * 4 * 32 * 16;
  static constexpr int PRE = BAR + WARPS * STAGES * 8;
  static constexpr int bytes(int B) { return PRE + (B + 1) * 4; }
};
}  // namespace dec4

// contiguous 16-byte multiples from global memory; completes `bytes` on `bar`
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ uint32_t lds4(uint32_t a) {
  uint32_t r;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// the 8 x 8 matrix of 16-bit elements that a warp holds in rows, transposed
__device__ __forceinline__ uint32_t turned8x8(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ uint32_t max_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ bool any_above_f16x2(uint32_t a, uint32_t b) {     // in either half
  uint32_t r;
  asm("set.gt.u32.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r != 0;
}
__device__ __forceinline__ float min_or_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// the largest over the lanes of the same t: tokens
__device__ __forceinline__ float tokens_max(float a) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
  return a;
}
__device__ __forceinline__ float tokens_sum(float a) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  return a;
}

// NT: tiles of 8 query heads per KV head (1: groups up to 8, 2: up to 16).
template <int NT>
__global__ void __launch_bounds__(dec4::THREADS, dec4::ctas_per_sm(NT))
    decode_attn_int4_kernel(const __nv_bfloat16* __restrict__ q, int ldq, KvInt4 c, const int* __restrict__ tables,
                            int max_blocks, const int* __restrict__ ctx_lens, __nv_bfloat16* __restrict__ out, int ldo,
                            int B, int Hq, float scale_log2, float* __restrict__ part, uint32_t* __restrict__ counters,
                            int* status, uint64_t wait_ns) {
  using namespace dec4;
  extern __shared__ __align__(16) uint8_t smem[];
  float* so = reinterpret_cast<float*>(smem);                           // [WARPS][8 NT][O_ROW], once the rings are drained
  float* sm = reinterpret_cast<float*>(smem + Smem<NT>::STATS);         // [WARPS][8 NT][m, l, mv0, mv1, z0, z1, -, -]
  uint4* sq = reinterpret_cast<uint4*>(smem + Smem<NT>::Q);             // [NT][4 words][32 lanes]
  int* pre = reinterpret_cast<int*>(smem + Smem<NT>::PRE);              // [B + 1] units of the pairs before sequence b
  __shared__ uint32_t ticket;
  __shared__ __align__(16) float sqf[8 * NT][4];                        // of a head: factor of the logits, sums of q
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int gq = lane >> 2, qd = lane & 3;
  const int Hkv = c.Hkv, G = Hq / Hkv;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Smem<NT>::BAR) + warp * STAGES;
  if (lane == 0) {
    for (int i = 0; i < STAGES; ++i) mbar_init(&bars[i], 1);
    fence_barrier_init();
  }
  const DecodeShare share = decode_share<Cfg>(ctx_lens, B, max_blocks, Hkv, pre, status);   // (its barriers order the init)
  // rows without tokens: zeros
  for (int b = blockIdx.x; b < B; b += gridDim.x)
    if (pre[b + 1] == pre[b])
      for (int i = tid; i < Hq * D / 8; i += THREADS) st_v4(out + (size_t)b * ldo + 8 * i, u128{0, 0, 0, 0});

  const uint32_t ring = smem_u32(smem) + warp * (STAGES * STAGE);
  const uint32_t kget = gq * ROW + 8 * qd;             // + 32 for the second half, + 8 ROW for token g + 8
  const uint32_t vget = 2 * qd * ROW + 4 * gq;
  const uint32_t pget = gq * ROW + D / 2;              // scales and minima of token g
  uint32_t turn = 0;                                   // pairs of blocks that the warp has consumed
  // false once a wait of the CTA ran out (recorded): it then loads nothing more, but walks its share to the end and
  // takes its turn in every pair, so that the counters are zero again and the pair's rows come out as NaN
  bool alive = true;

  int b = share.b;
  for (int u = share.u0; u < share.u1;) {
    // ---- the blocks [j0, j1) of KV head h of sequence b
    while (pre[b + 1] <= u) ++b;
    const int units = (pre[b + 1] - pre[b]) / Hkv;
    const int h = (u - pre[b]) / units;
    const int pair0 = pre[b] + h * units;                      // first unit of the pair
    const int j0 = max(0, u - pair0 - Cfg::PAIR_COST), j1 = min(units, share.u1 - pair0) - Cfg::PAIR_COST;
    u = min(pair0 + units, share.u1);
    if (j1 <= 0) continue;                                     // none but the pair's fixed cost
    const int len = min(max(ctx_lens[b], 0), max_blocks * BS);

    // ---- the warp's loads, two blocks at a time
    const int mine0 = j0 + 2 * warp;                           // the warp's first block
    const int turns = alive && mine0 < j1 ? (j1 - mine0 + 2 * WARPS - 1) / (2 * WARPS) : 0;
    int fcount = 0, ids = -1;
    uint32_t valid = 0, given = 0;          // blocks of `ids` that there are; of the stages' two blocks, 2 bits a stage
    const uint8_t* mycache = (lane & 2 ? c.v : c.k) + (size_t)h * BLOCK;      // lanes 0..3: K, K, V, V
    auto fetch = [&](uint32_t stage) {
      if ((fcount & 15) == 0) {                                // ids of the next 32 blocks, one per lane
        const int mine = mine0 + (fcount + (lane >> 1)) * (2 * WARPS) + (lane & 1);
        ids = -1;
        if (mine < j1) {
          ids = tables[(size_t)b * max_blocks + mine];
          if (ids < 0 || ids >= c.num_blocks) {
            record_status(status, CX_ERR_BOUNDS);
            ids = -1;
          }
        }
        valid = __ballot_sync(0xffffffffu, ids >= 0);
      }
      const int at = 2 * (fcount & 15);
      const int id = __shfl_sync(0xffffffffu, ids, at + (lane & 1));
      const uint32_t two = valid >> at & 3;
      given = (given & ~(3u << 2 * stage)) | two << 2 * stage;
      if (lane == 0) mbar_arrive_expect_tx(&bars[stage], __popc(two) * 2 * BLOCK);
      __syncwarp();
      if (lane < 4 && id >= 0)
        bulk_load(ring + stage * STAGE + lane * BLOCK, mycache + (size_t)id * Hkv * BLOCK, BLOCK, &bars[stage]);
      ++fcount;
    };
    fence_proxy_async_smem();                                  // O of the run before was written to the rings
#pragma unroll
    for (uint32_t i = 0; i < STAGES; ++i)
      if ((int)i < turns) fetch((turn + i) & 1);
    // ---- q fragments: a word's dims 8w + {0, 4}, {2, 6}, {1, 5}, {3, 7}; warp i makes [.][i]
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const bool on = gq + 8 * nt < G;
      u128 raw[4];                                             // [half][word]: dims half * 64 + qd * 16 + word * 8 ..
#pragma unroll
      for (int i = 0; i < 4; ++i)
        raw[i] = on ? ld_v4(q + (size_t)b * ldq + (size_t)(h * G + gq + 8 * nt) * D + (i >> 1) * 64 + qd * 16 + (i & 1) * 8)
                    : u128{0, 0, 0, 0};
      float am = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          am = fmaxf(am, fmaxf(finite_or_zero(bf16_lo(word(raw[i], e))), finite_or_zero(bf16_hi(word(raw[i], e)))));
      am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 1));
      am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 2));
      // am * 2^-eq in [2^14, 2^15)
      const int eq = am > 0.f ? max((int)(__float_as_uint(am) >> 23) - 127 - 14, -126) : 0;
      const float down = exp2_int(-eq);
      if (warp == 0) {
        float qs[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float a = 0.f;
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) a += (bf16_lo(word(raw[2 * half + i], e)) + bf16_hi(word(raw[2 * half + i], e))) * down;
          a += __shfl_xor_sync(0xffffffffu, a, 1);
          a += __shfl_xor_sync(0xffffffffu, a, 2);
          qs[half] = a * 5.9604645e-8f;                        // S counts in 2^-24
        }
        if (qd == 0) *reinterpret_cast<float4*>(sqf[8 * nt + gq]) = make_float4(exp2_int(eq) * scale_log2, qs[0], qs[1], 0.f);
      }
      static_assert(WARPS == 4, "a warp per word");
      const u128 w = warp == 0 ? raw[0] : warp == 1 ? raw[1] : warp == 2 ? raw[2] : raw[3];
      const float d16 = down * 0.0625f;
      sq[(nt * 4 + warp) * 32 + lane] =
          make_uint4(pack_f16x2(bf16_lo(w.x) * down, bf16_lo(w.z) * down), pack_f16x2(bf16_lo(w.y) * down, bf16_lo(w.w) * down),
                     pack_f16x2(bf16_hi(w.x) * d16, bf16_hi(w.z) * d16), pack_f16x2(bf16_hi(w.y) * d16, bf16_hi(w.w) * d16));
    }
    __syncthreads();

    // of heads 8 nt + 2 qd + {0, 1}: the logits' factor, sums of q, running maximum m of the logits, sum l; of their
    // halves: sums z of weight * minimum, the power of two f of the weights times scales
    float o[NT][8][4], z[NT][2][2], m[NT][2], l[NT][2], f[NT][2][2], qf[NT][2], qs[NT][2][2];
    auto power = [&](int nt, int cc, int half) { return (int)(__float_as_uint(f[nt][cc][half]) >> 23) - 127; };
    auto scale_o = [&](int nt, int cc, int half, float by) {
#pragma unroll
      for (int k = 4 * half; k < 4 * half + 4; ++k) {
        o[nt][k][cc] *= by;
        o[nt][k][2 + cc] *= by;
      }
    };
    bool far = false;                                          // q beyond 2^100: 2^24 is not folded into its factor
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int cc = 0; cc < 2; ++cc) {
        const float4 t = *reinterpret_cast<const float4*>(sqf[8 * nt + 2 * qd + cc]);
        qf[nt][cc] = t.x;
        qs[nt][cc][0] = t.y;
        qs[nt][cc][1] = t.z;
        far |= fabsf(t.x) > 1e30f;
        m[nt][cc] = -INFINITY;
        f[nt][cc][0] = f[nt][cc][1] = exp2_int(START);
        l[nt][cc] = z[nt][cc][0] = z[nt][cc][1] = 0.f;
      }
#pragma unroll
      for (int mt = 0; mt < 8; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][mt][e] = 0.f;
    }
    far = __any_sync(0xffffffffu, far);
    if (!far)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        qf[nt][0] *= 16777216.f;
        qf[nt][1] *= 16777216.f;
      }
    int i0 = 0;
    bool ok = alive;
    for (; i0 < turns; ++i0, ++turn) {
      const uint32_t stage = turn & 1;
      const uint32_t sk = ring + stage * STAGE, sv = sk + 2 * BLOCK;
      const int j = mine0 + i0 * 2 * WARPS;
      const uint32_t here = given >> 2 * stage & 3;
      const bool full = here == 3 && (j + 2) * BS <= len;      // the same for the whole warp
      if (wait_ns != 0) ok = mbar_wait(&bars[stage], turn >> 1 & 1, status, wait_ns);
      else if (here != 0) ok = wait_lost(status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      // ---- logits of tokens g and g + 8 of both blocks: x[nt][block][token][head]
      float x[NT][2][2][2];
      uint2 kp[2][2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) kp[i][tt] = lds8(sk + pget + i * BLOCK + tt * 8 * ROW);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float s[NT][2][4];
        uint2 kw[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int tt = 0; tt < 2; ++tt) kw[i][tt] = lds8(sk + kget + half * 32 + i * BLOCK + tt * 8 * ROW);
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint4 qa = sq[(nt * 4 + 2 * half + w) * 32 + lane];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t a = w ? kw[i][0].y : kw[i][0].x, a8 = a >> 8, e = w ? kw[i][1].y : kw[i][1].x, e8 = e >> 8;
              if (w == 0)
                mma_f16_first(s[nt][i], a & 0x000f000fu, e & 0x000f000fu, a8 & 0x000f000fu, e8 & 0x000f000fu, qa.x, qa.y);
              else
                mma_f16(s[nt][i], a & 0x000f000fu, e & 0x000f000fu, a8 & 0x000f000fu, e8 & 0x000f000fu, qa.x, qa.y);
              mma_f16(s[nt][i], a & 0x00f000f0u, e & 0x00f000f0u, a8 & 0x00f000f0u, e8 & 0x00f000f0u, qa.z, qa.w);
            }
          }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int tt = 0; tt < 2; ++tt) {
            const uint32_t pr = half ? kp[i][tt].y : kp[i][tt].x;
            const float ps = bf16_lo(pr), pm = bf16_hi(pr);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int cc = 0; cc < 2; ++cc)
                x[nt][i][tt][cc] = fmaf(ps, s[nt][i][2 * tt + cc],
                                        half ? fmaf(pm, qs[nt][cc][1], x[nt][i][tt][cc]) : pm * qs[nt][cc][0]);
          }
      }
      float vs[2][2][2], vm[2][2][2];                          // [half][block][token]
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
          const uint2 pr = lds8(sv + pget + i * BLOCK + tt * 8 * ROW);
          vs[0][i][tt] = bf16_lo(pr.x);
          vm[0][i][tt] = bf16_hi(pr.x);
          vs[1][i][tt] = bf16_lo(pr.y);
          vm[1][i][tt] = bf16_hi(pr.y);
        }
      if (far)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 8; ++e) x[nt][e >> 2][e >> 1 & 1][e & 1] *= 16777216.f;
      // ---- weights: y = logit - m
      float y[NT][2][2][2], top = -INFINITY;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          y[nt][e >> 2][e >> 1 & 1][e & 1] = fmaf(x[nt][e >> 2][e >> 1 & 1][e & 1], qf[nt][e & 1], -m[nt][e & 1]);
      if (!full) {
        // tokens behind the end, blocks that are not there: no weight, and what their rows hold does not count
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int tt = 0; tt < 2; ++tt)
            if (!(here >> i & 1) || (j + i) * BS + tt * 8 + gq >= len) {
              vs[0][i][tt] = vs[1][i][tt] = vm[0][i][tt] = vm[1][i][tt] = 0.f;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                y[nt][i][tt][0] = y[nt][i][tt][1] = -INFINITY;
            }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, y[nt][e >> 2][e >> 1 & 1][e & 1]);
      if (__any_sync(0xffffffffu, top > LATE)) {               // m moves (from -inf: y is infinite, or not a number)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            float most = -INFINITY;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (y[nt][e >> 1][e & 1][cc] != -INFINITY) most = fmaxf(most, x[nt][e >> 1][e & 1][cc] * qf[nt][cc]);
            const float now = fmaxf(m[nt][cc], tokens_max(most)), base = now == -INFINITY ? 0.f : now;
            const float keep = ex2(m[nt][cc] - base);
            l[nt][cc] *= keep;
            z[nt][cc][0] *= keep;
            z[nt][cc][1] *= keep;
            // O counts in 2^(m - power): the products so far are smaller next to the new maximum, and so the power may rise
            const float rise = fminf(base - m[nt][cc], 1000.f);           // 1000: from no maximum at all
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const int p = power(nt, cc, half), up = min((int)ceilf(rise), START - p);
              f[nt][cc][half] = exp2_int(p + up);
              scale_o(nt, cc, half, ex2((float)up - rise));
            }
            m[nt][cc] = now;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (y[nt][e >> 1][e & 1][cc] != -INFINITY)       // (the product is rounded in `now` and not here)
                y[nt][e >> 1][e & 1][cc] = min_or_nan(fmaf(x[nt][e >> 1][e & 1][cc], qf[nt][cc], -base), 0.f);
          }
      }
      uint32_t wb[NT][2][2][2];                                // [half][block][token]: heads 2 qd, 2 qd + 1
      uint32_t big = 0;
      auto weights = [&](int nt, int half, int e) {
        const float s = vs[half][e >> 1][e & 1];
        return pack_f16x2(y[nt][e >> 1][e & 1][0] * f[nt][0][half] * s, y[nt][e >> 1][e & 1][1] * f[nt][1][half] * s);
      };
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[nt][e >> 2][e >> 1 & 1][e & 1] = ex2(y[nt][e >> 2][e >> 1 & 1][e & 1]);
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          l[nt][cc] += (y[nt][0][0][cc] + y[nt][0][1][cc]) + (y[nt][1][0][cc] + y[nt][1][1][cc]);
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int e = 0; e < 4; ++e) z[nt][cc][half] = fmaf(y[nt][e >> 1][e & 1][cc], vm[half][e >> 1][e & 1], z[nt][cc][half]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            wb[nt][half][e >> 1][e & 1] = weights(nt, half, e);
            big = max_f16x2(big, wb[nt][half][e >> 1][e & 1]);
          }
      }
      if (__any_sync(0xffffffffu, any_above_f16x2(big, MOST_W))) {              // the powers sink
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int cc = 0; cc < 2; ++cc) {
              float most = 0.f;                                // (2^-16 of it: the product may be beyond fp32)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                most = fmaxf(most, y[nt][e >> 1][e & 1][cc] * (vs[half][e >> 1][e & 1] * 1.52587890625e-5f));
              const float room = TOP_W - 16.f - lg2(fmaxf(tokens_max(most), 1e-37f));
              const int p = power(nt, cc, half), to = min(p, (int)fmaxf(ceilf(room), -126.f));
              f[nt][cc][half] = exp2_int(to);
              scale_o(nt, cc, half, ex2((float)(to - p)));
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) wb[nt][half][e >> 1][e & 1] = weights(nt, half, e);
          }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int e = 0; e < 4; ++e) wb[nt][half][e >> 1][e & 1] = turned8x8(wb[nt][half][e >> 1][e & 1]);
      // ---- O^T
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int i = 0; i < 2; ++i) {                          // blocks
          uint32_t vw[4];                                      // tokens 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
          for (int e = 0; e < 4; ++e) vw[e] = lds4(sv + vget + half * 32 + i * BLOCK + ((e >> 1) * 8 + (e & 1)) * ROW);
#pragma unroll
          for (int hw = 0; hw < 2; ++hw) {                     // dims 4 hw .. of the word, two tokens side by side
            const uint32_t y = __byte_perm(vw[0], vw[1], hw ? 0x7632 : 0x5410), y8 = y >> 8;
            const uint32_t w = __byte_perm(vw[2], vw[3], hw ? 0x7632 : 0x5410), w8 = w >> 8;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_f16(o[nt][4 * half + 2 * hw], y & 0x000f000fu, y8 & 0x000f000fu, w & 0x000f000fu, w8 & 0x000f000fu,
                      wb[nt][half][i][0], wb[nt][half][i][1]);
              mma_f16(o[nt][4 * half + 2 * hw + 1], y & 0x00f000f0u, y8 & 0x00f000f0u, w & 0x00f000f0u, w8 & 0x00f000f0u,
                      wb[nt][half][i][0], wb[nt][half][i][1]);
            }
          }
        }
      __syncwarp();                                            // the stage has been read by all
      if (i0 + STAGES < turns) fetch(stage);
    }
    if (!ok)   // the copies under way get a bounded time to land before the rings are written to
      for (uint32_t i = 0; i < STAGES && i0 + (int)i < turns; ++i)
        mbar_wait(&bars[(turn + i) & 1], (turn + i) >> 1 & 1, nullptr, 100000000ull);
    alive = !__syncthreads_or(!ok);                            // every warp has drained its ring
    if (!alive)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          l[nt][cc] = __uint_as_float(0x7fffffffu);
          m[nt][cc] = -INFINITY;
        }

    // ---- the warps' results of this run
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int cc = 0; cc < 2; ++cc) {
        const float ls = tokens_sum(l[nt][cc]), z0 = tokens_sum(z[nt][cc][0]), z1 = tokens_sum(z[nt][cc][1]);
        if (gq == 0) {
          float4* st = reinterpret_cast<float4*>(sm + (warp * 8 * NT + nt * 8 + 2 * qd + cc) * 8);
          st[0] = make_float4(m[nt][cc], ls, m[nt][cc] - power(nt, cc, 0), m[nt][cc] - power(nt, cc, 1));
          st[1] = make_float4(z0, z1, 0.f, 0.f);
        }
      }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
      // dim half * 64 + 8 g + n in column (half * 8 + n) * 8 + g
#pragma unroll
      for (int mt = 0; mt < 8; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int n = (mt >> 1 & 1) * 4 + (mt & 1) + 2 * (e >> 1);
          so[(warp * 8 * NT + nt * 8 + 2 * qd + (e & 1)) * O_ROW + ((mt >> 2) * 8 + n) * 8 + gq] =
              o[nt][mt][e] * (mt & 1 ? 1048576.f : 16777216.f);
        }
    __syncthreads();
    // the CTAs that share the pair: those of the cuts left inside it, and the one before
    const int slack = decode_slack<Cfg>(units, share.most);
    const int c0 = (pair0 + Cfg::PAIR_COST + slack) / share.per, c1 = (pair0 + units - slack - 1) / share.per;
    // two heads at a time, a thread for two dims of one
    for (int hh = tid >> 6; hh < G; hh += 2) {
      const int d8 = tid & 7, d2 = tid >> 3 & 7, half = d2 >> 2, dim = half * 64 + 8 * d8 + 2 * (d2 & 3);
      float M = -INFINITY, MV0 = -INFINITY, MV1 = -INFINITY;   // (the units are infinite where the maximum is)
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        M = fmaxf(M, sm[(w * 8 * NT + hh) * 8]);
        MV0 = fmaxf(MV0, sm[(w * 8 * NT + hh) * 8 + 2]);
        MV1 = fmaxf(MV1, sm[(w * 8 * NT + hh) * 8 + 3]);
      }
      const float mb = M == -INFINITY ? 0.f : M, vb = M == -INFINITY ? 0.f : half ? MV1 : MV0;
      float2 num = make_float2(0.f, 0.f), zz = make_float2(0.f, 0.f);
      float den = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float* p = so + (w * 8 * NT + hh) * O_ROW + 16 * d2 + d8;
        const float* st = sm + (w * 8 * NT + hh) * 8;
        const float f = ex2(st[2 + half] - vb), fm = ex2(st[0] - mb);
        num.x += p[0] * f;
        num.y += p[8] * f;
        den += st[1] * fm;
        zz.x += st[4] * fm;
        zz.y += st[5] * fm;
      }
      if (c0 >= c1) {
        const float inv = den == 0.f ? 0.f : 1.f / den, f = ex2(vb - mb), zh = half ? zz.y : zz.x;
        *reinterpret_cast<uint32_t*>(out + (size_t)b * ldo + (size_t)(h * G + hh) * D + dim) =
            pack_bf16x2(fmaf(num.x, f, zh) * inv, fmaf(num.y, f, zh) * inv);
      } else {   // slot 1 for the pair that goes on in the next CTA, 0 for one that began before
        float* p = part + ((size_t)(blockIdx.x * 2 + ((int)blockIdx.x == c0)) * G + hh) * DEC4_ROW;
        *reinterpret_cast<float2*>(p + dim) = num;
        if ((tid & 63) == 0) {
          *reinterpret_cast<float4*>(p + D) = make_float4(M, den, MV0, MV1);
          *reinterpret_cast<float4*>(p + D + 4) = make_float4(zz.x, zz.y, 0.f, 0.f);
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
            return part + ((size_t)(cc * 2 + (cc == c0)) * G + hh) * DEC4_ROW;
          };
          const int of = lane & 16, at = lane & 15;            // a half-warp for each half of the dims
          float m_all = -INFINITY, mv_all = -INFINITY, den = 0.f, zh = 0.f;
          float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
          auto largest = [](float a) {
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
            return a;
          };
          auto total = [](float a) {
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
            return a;
          };
          for (int cb = c0; cb <= c1; cb += 16) {              // 16 CTAs at a time, rescaled as the maxima grow
            const int n = min(16, c1 - cb + 1);
            float4 st = make_float4(-INFINITY, 0.f, -INFINITY, -INFINITY);
            float2 zs = make_float2(0.f, 0.f);
            if (at < n) {
              st = __ldcg(reinterpret_cast<const float4*>(slot(cb + at) + D));
              zs = __ldcg(reinterpret_cast<const float2*>(slot(cb + at) + D + 4));
            }
            const float mv = of ? st.w : st.z;
            const float m_new = fmaxf(m_all, largest(st.x)), mb = m_new == -INFINITY ? 0.f : m_new;
            const float mv_new = fmaxf(mv_all, largest(mv)), vb = m_new == -INFINITY ? 0.f : mv_new;
            const float fv = ex2(mv_all - vb), fm = ex2(m_all - mb), mine = ex2(st.x - mb);
            den = den * fm + st.y * mine;
            zh = zh * fm + (of ? zs.y : zs.x) * mine;
            num.x *= fv;
            num.y *= fv;
            num.z *= fv;
            num.w *= fv;
            m_all = m_new;
            mv_all = mv_new;
            const float f = ex2(mv - vb);
            for (int i = 0; i < n; i += 8) {
              float4 y[8];
#pragma unroll
              for (int k = 0; k < 8; ++k)
                y[k] = i + k < n ? __ldcg(reinterpret_cast<const float4*>(slot(cb + i + k)) + lane)
                                 : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const float g = __shfl_sync(0xffffffffu, f, of + (i + k & 15));
                if (i + k < n) {
                  num.x += y[k].x * g;
                  num.y += y[k].y * g;
                  num.z += y[k].z * g;
                  num.w += y[k].w * g;
                }
              }
            }
          }
          const float mb = m_all == -INFINITY ? 0.f : m_all, vb = m_all == -INFINITY ? 0.f : mv_all;
          den = total(den);
          zh = total(zh);
          const float inv = den == 0.f ? 0.f : 1.f / den, f = ex2(vb - mb);
          uint2 w;
          w.x = pack_bf16x2(fmaf(num.x, f, zh) * inv, fmaf(num.y, f, zh) * inv);
          w.y = pack_bf16x2(fmaf(num.z, f, zh) * inv, fmaf(num.w, f, zh) * inv);
          *reinterpret_cast<uint2*>(out + (size_t)b * ldo + (size_t)(h * G + hh) * D + 4 * lane) = w;
        }
      }
    }
    fence_proxy_async_smem();                                  // the rings are copied into again
    __syncthreads();                                           // O and the statistics have been read
  }
}

static int decode_int4_resident(int B, int nt) {
  const int smem = nt == 2 ? dec4::Smem<2>::bytes(B) : dec4::Smem<1>::bytes(B);
  constexpr int PER_SM = 228 * 1024, OTHER = 1024 + 256;      // of a CTA: the system's, and the static variables
  return std::min(dec4::ctas_per_sm(nt), PER_SM / (smem + OTHER));
}
long decode_int4_rows(int sms, int B, int Hkv, int G) {
  const long row = (long)G * DEC4_ROW;
  return 2L * sms * dec4::ctas_per_sm(1) + ((long)B * Hkv + row - 1) / row;
}

void decode_attention_int4(const void* q, int ldq, const KvInt4& c, const int* block_tables, int max_blocks,
                           const int* ctx_lens, void* out, int ldo, int B, int Hq, float scale, float* ws, int sms,
                           int* status, int64_t wait_ns, cudaStream_t s) {
  if (B == 0) return;
  const int G = Hq / c.Hkv, nt = G > 8 ? 2 : 1;
  // the partial results (room for the largest grid) sit at the front, the counters behind them: neither
  // moves with the batch
  uint32_t* counters = reinterpret_cast<uint32_t*>(ws + 2L * sms * dec4::ctas_per_sm(1) * G * DEC4_ROW);
  const long most = ((long)B * c.Hkv * (max_blocks + dec4::Cfg::PAIR_COST) + dec4::Cfg::MIN_UNITS - 1) / dec4::Cfg::MIN_UNITS;
  const int grid = (int)std::max(1L, std::min((long)sms * decode_int4_resident(B, nt), most));
  const int smem = nt == 2 ? dec4::Smem<2>::bytes(B) : dec4::Smem<1>::bytes(B);
  auto kern = nt == 2 ? decode_attn_int4_kernel<2> : decode_attn_int4_kernel<1>;
  static bool attr[64][2] = {};
  int dev;
  cudaGetDevice(&dev);
  if (!attr[dev & 63][nt - 1]) {
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                         nt == 2 ? dec4::Smem<2>::bytes(DEC4_MAX_BATCH) : dec4::Smem<1>::bytes(DEC4_MAX_BATCH));
    cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
    attr[dev & 63][nt - 1] = true;
  }
  kern<<<grid, dec4::THREADS, smem, s>>>(reinterpret_cast<const __nv_bfloat16*>(q), ldq, c, block_tables, max_blocks,
                                         ctx_lens, reinterpret_cast<__nv_bfloat16*>(out), ldo, B, Hq,
                                         scale * 1.4426950408889634f, ws, counters, status,
                                         wait_ns < 0 ? kDefaultWaitNs : (uint64_t)wait_ns);
}

}  // namespace cx
