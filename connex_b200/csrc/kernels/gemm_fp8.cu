// Products in e4m3 with a scale for each block of 128: the operands' quantisers
// and the GEMM.
//
//   q[r, c] = e4m3(x[r, c] * 448 / top),  scale = top / 448,  top = max |x| of the block
//   D[m, n] = sum_kb sa[m, kb] * sb[n / 128, kb] * sum_{k in kb} a[m, k] * b[n, k]
//
// The scales are any fp32 numbers (a checkpoint's weights come with such), so
// the tensor core adds up one block of 128 columns at a time and the scales are
// applied to those sums outside of it.
#include <algorithm>
#include <stdexcept>

#include "fewbit.cuh"
#include "gemm.h"
#include "gemm_fp8.h"
#include "gemm_tile.cuh"

namespace cx {

namespace q8 {
constexpr int Q = 128;                       // columns of a block
constexpr float TOP = 448.f, TINY = 7.888609052210118e-31f;   // largest e4m3 value; 2^-100, a block's top at least
constexpr int THREADS = 256;
}  // namespace q8

// ------------------------------------------------------------- quantisation
// Eight fp32 values -> e4m3; `mul` = 448 / top.  Infinities and NaN become NaN
// (`scaled` of a finite value is one, |x| mul <= 448).
__device__ __forceinline__ uint32_t quant_pair(float lo, float hi, float mul) {
  auto scaled = [&](float x) {
    return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u ? __uint_as_float(0x7fffffffu) : x * mul;
  };
  return to_e4m3x2(scaled(lo), scaled(hi));
}
__device__ __forceinline__ uint2 quant8(const float (&v)[8], float mul) {
  return make_uint2(quant_pair(v[0], v[1], mul) | quant_pair(v[2], v[3], mul) << 16,
                    quant_pair(v[4], v[5], mul) | quant_pair(v[6], v[7], mul) << 16);
}
__device__ __forceinline__ float top8(const float (&v)[8]) {
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = fmaxf(a, finite_or_zero(v[i]));
  return a;
}
// the largest over a half-warp: the 16 lanes of a block of 128 columns
__device__ __forceinline__ float half_warp_max(float a) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
  return a;
}
__device__ __forceinline__ void unpack8(const u128& r, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = bf16_lo(word(r, i));
    v[2 * i + 1] = bf16_hi(word(r, i));
  }
}

// A half-warp per block, eight columns of a lane, UNROLL blocks in flight.
template <int UNROLL>
__global__ void __launch_bounds__(q8::THREADS)
    quantize_fp8_kernel(const __nv_bfloat16* __restrict__ x, int64_t ldx, uint8_t* __restrict__ q, int64_t ldq,
                        Fp8Scales s, int64_t blocks, int kb, int K) {
  using namespace q8;
  const int lane = threadIdx.x & 31, j = lane & 15;
  const int64_t per = (int64_t)gridDim.x * (THREADS / 16);
  const int64_t first = (int64_t)blockIdx.x * (THREADS / 16) + (threadIdx.x >> 4);
  for (int64_t u0 = first - (lane >> 4); u0 < blocks; u0 += UNROLL * per) {   // the same for the whole warp
    u128 raw[UNROLL];
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      const int64_t u = u0 + (lane >> 4) + i * per, row = u / kb;
      const int c = (int)(u - row * kb) * Q + 8 * j;
      raw[i] = u < blocks && c < K ? ld_nc_v4(x + row * ldx + c) : u128{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      const int64_t u = u0 + (lane >> 4) + i * per, row = u / kb;
      const int b = (int)(u - row * kb), c = b * Q + 8 * j;
      float v[8];
      unpack8(raw[i], v);
      const float top = fmaxf(half_warp_max(top8(v)), TINY);
      if (u >= blocks) continue;
      if (c < K) *reinterpret_cast<uint2*>(q + row * ldq + c) = quant8(v, TOP / top);
      if (j == 0) s.p[row * s.row + b * s.col] = top / TOP;
    }
  }
}

// The same behind an RMS norm: a CTA per row, the row in registers.
template <int VPT>
__global__ void __launch_bounds__(q8::THREADS)
    quantize_norm_fp8_kernel(const __nv_bfloat16* __restrict__ x, int64_t ldx, const __nv_bfloat16* __restrict__ w,
                             float eps, uint8_t* __restrict__ q, int64_t ldq, Fp8Scales s, int K) {
  using namespace q8;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  u128 raw[VPT];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (i * THREADS + tid) * 8;
    raw[i] = c < K ? ld_nc_v4(x + row * ldx + c) : u128{0, 0, 0, 0};
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    float v[8];
    unpack8(raw[i], v);
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += v[e] * v[e];
  }
  __shared__ float red[THREADS / 32];
  ss = warp_sum(ss);
  if ((tid & 31) == 0) red[tid >> 5] = ss;
  __syncthreads();
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) sum += red[i];
  const float inv = rsqrtf(sum / (float)K + eps);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (i * THREADS * 8 >= K) break;
    const int c = (i * THREADS + tid) * 8;
    float v[8], g[8];
    unpack8(raw[i], v);
    unpack8(c < K ? ld_v4(w + c) : u128{0, 0, 0, 0}, g);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = v[e] * inv * g[e];
    const float top = fmaxf(half_warp_max(top8(v)), TINY);
    if (c < K) {
      *reinterpret_cast<uint2*>(q + row * ldq + c) = quant8(v, TOP / top);
      if ((tid & 15) == 0) s.p[row * s.row + (c / Q) * s.col] = top / TOP;
    }
  }
}

// A CTA per 128 x 128 block of a weight.
__global__ void __launch_bounds__(q8::THREADS)
    quantize_weight_fp8_kernel(const __nv_bfloat16* __restrict__ w, int64_t ldw, uint8_t* __restrict__ q, int64_t ldq,
                               Fp8Scales s, int N, int K) {
  using namespace q8;
  const int tid = threadIdx.x, c = blockIdx.x * Q + 8 * (tid & 15);
  u128 raw[8];
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t n = (int64_t)blockIdx.y * Q + i * 16 + (tid >> 4);
    raw[i] = n < N && c < K ? ld_nc_v4(w + n * ldw + c) : u128{0, 0, 0, 0};
    float v[8];
    unpack8(raw[i], v);
    top = fmaxf(top, top8(v));
  }
  __shared__ float red[THREADS / 32];
  top = warp_max(top);
  if ((tid & 31) == 0) red[tid >> 5] = top;
  __syncthreads();
  top = TINY;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) top = fmaxf(top, red[i]);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t n = (int64_t)blockIdx.y * Q + i * 16 + (tid >> 4);
    float v[8];
    unpack8(raw[i], v);
    if (n < N && c < K) *reinterpret_cast<uint2*>(q + n * ldq + c) = quant8(v, TOP / top);
  }
  if (tid == 0) s.p[blockIdx.y * s.row + blockIdx.x * s.col] = top / TOP;
}

void quantize_fp8(const void* x, int64_t ldx, const void* w, float eps, void* q, int64_t ldq, const Fp8Scales& s, int T,
                  int K, cudaStream_t stream) {
  using namespace q8;
  if (T == 0 || K == 0) return;
  auto X = reinterpret_cast<const __nv_bfloat16*>(x);
  auto W = reinterpret_cast<const __nv_bfloat16*>(w);
  auto O = reinterpret_cast<uint8_t*>(q);
  const int kb = (K + Q - 1) / Q;
  if (w == nullptr) {
    const int64_t blocks = (int64_t)T * kb;
    const int64_t ctas = std::min<int64_t>((blocks + THREADS / 16 - 1) / (THREADS / 16), 148 * 8);
    quantize_fp8_kernel<4><<<(int)ctas, THREADS, 0, stream>>>(X, ldx, O, ldq, s, blocks, kb, K);
    return;
  }
  const int vpt = (K / 8 + THREADS - 1) / THREADS;
  auto go = [&](auto kern) { kern<<<T, THREADS, 0, stream>>>(X, ldx, W, eps, O, ldq, s, K); };
  if (vpt <= 1) go(quantize_norm_fp8_kernel<1>);
  else if (vpt <= 2) go(quantize_norm_fp8_kernel<2>);
  else if (vpt <= 4) go(quantize_norm_fp8_kernel<4>);
  else if (vpt <= 8) go(quantize_norm_fp8_kernel<8>);
  else throw std::runtime_error("cx quantize_fp8: row too long for the norm");
}

void quantize_weight_fp8(const void* w, int64_t ldw, void* q, int64_t ldq, const Fp8Scales& s, int N, int K,
                         cudaStream_t stream) {
  using namespace q8;
  if (N == 0 || K == 0) return;
  quantize_weight_fp8_kernel<<<dim3((K + Q - 1) / Q, (N + Q - 1) / Q), THREADS, 0, stream>>>(
      reinterpret_cast<const __nv_bfloat16*>(w), ldw, reinterpret_cast<uint8_t*>(q), ldq, s, N, K);
}

// --------------------------------------------------------------------- GEMM
// A persistent CTA per SM, output tiles of 128 x 256:
//   warp 0      TMA: 128 x 128 bytes of A and 256 x 128 of B per stage, 128-byte swizzle
//   warp 1      tcgen05.mma, M = 128, N = 256, K = 32 e4m3, four per stage: one block of 128 columns, into one of
//               two accumulators in TMEM
//   warp 3      the scales of the CTA's rows and of the tile's two blocks of B, up to sixteen blocks of 128 columns ahead (each
//               is a line of its own: fetched one block ahead by the warps that use them they took longer than the MMAs)
//   warps 4-11  promotion: two warpgroups; a thread takes a row, and columns [64 g, 64 g + 64) of both halves of
//               the tile, reads the block's sums from TMEM, multiplies by the scales and adds in registers.  One
//               accumulator is read while the MMAs fill the other.
// What bounds it is the way round: an accumulator's MMAs (513 cycles), the word that it is complete (some 260), its
// promotion by two warps on each SM quarter (350 to 600), the word that it is free (90).  Two accumulators of 256
// columns are all of TMEM, so a block takes 700 cycles at least (an SM by itself, operands in place), 1000 here.
// Measured on 8192 x 28672 x 4096 with SiLU(gate) * up, as variants of this kernel: pairs of CTAs on one tile of 256 x
// 256 (cta_group::2) 1060 us, their way round being longer by two signals between SMs; four warpgroups of half the
// columns 1190; four accumulators of 128 columns 1280 (the issuing thread falls behind); barriers waited for in
// mbarrier.try_wait, which suspends, where single threads poll here, 1150.
// A warpgroup holds gate and up of the same outputs, so SiLU(gate) * up needs no exchange; a row's largest value
// over the tile's 128 outputs, for quantised output, passes through shared memory.
namespace g8 {
constexpr int BM = 128, BN = 256, BK = 128;
constexpr int STAGES = 4;
constexpr int A_BYTES = BM * BK, B_BYTES = BN * BK, STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int EPI_WARPS = 8, THREADS = 128 + 32 * EPI_WARPS;
// 128 fp32 sums of a thread and the block's next 64 need more than an equal share of the registers.  The
// warpgroups' shares add up to no more than the block's at launch, 168 each.
constexpr int REGS_AUX = 64, REGS_EPI = 216;
constexpr int REGS_ALL = 128 * REGS_AUX + 32 * EPI_WARPS * REGS_EPI;
static_assert(REGS_ALL <= THREADS * 168, "register shares");
constexpr int TMEM_COLS = 2 * BN;
// scales of four blocks of columns at a time (one wait for all of them): the rows', then B's two of each
constexpr int SC_SLOTS = 4, SC_KB = 4, SC_ROW = SC_KB * BM + 2 * SC_KB;
constexpr int SMEM = 1024 /* alignment */ + STAGES * STAGE_BYTES + SC_SLOTS * SC_ROW * 4 + 2 * 2 * BM * 4 /* row maxima */ +
                     512 /* barriers */;
constexpr int GROUP = 16;             // tile-rows per raster band
}  // namespace g8

// x / (1 + e^-x) with the approximate quotient (2 ulp; beyond 2^126 it is 0, and so is the value nearly)
__device__ __forceinline__ float silu_fast(float x) { return __fdividef(x, 1.0f + ex2(x * -1.4426950408889634f)); }

template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ void bar_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

template <int EPI, bool QUANT>
__global__ void __launch_bounds__(g8::THREADS, 1)
    gemm_fp8_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, GemmFp8 g,
                    int* status) {
  using namespace g8;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * A_BYTES;
  float* scales = reinterpret_cast<float*>(smem + STAGES * STAGE_BYTES);    // [slot][SC_ROW]
  float* tops = scales + SC_SLOTS * SC_ROW;                                 // [tile parity][warpgroup][row]
  uint64_t* full = reinterpret_cast<uint64_t*>(tops + 2 * 2 * BM);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* sfull = tempty + 2;
  uint64_t* sempty = sfull + SC_SLOTS;
  uint64_t* drain = sempty + SC_SLOTS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);

  const int warp = warp_id(), lane = lane_id();
  const int M = g.M, N = g.N, num_m = (M + BM - 1) / BM, num_n = (N + BN - 1) / BN;
  const int total = num_m * num_n, nk = (g.K + BK - 1) / BK;
  const int first = blockIdx.x, step = gridDim.x;

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], EPI_WARPS);
    }
    for (int i = 0; i < SC_SLOTS; ++i) {
      mbar_init(&sfull[i], 32);
      mbar_init(&sempty[i], EPI_WARPS);
    }
    mbar_init(drain, 1);
    fence_barrier_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  bool ok = true;

  if (warp < 4) {
    regs_dec<REGS_AUX>();
    if (warp == 0 && lane == 0) {
      uint32_t stage = 0, phase = 0;
      for (int t = first; t < total && ok; t += step) {
        int tm, tn;
        tile_coords(t, num_m, num_n, GROUP, tm, tn);
        for (int kb = 0; kb < nk; ++kb) {
          if (!mbar_wait_poll(&empty[stage], phase ^ 1, status)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&full[stage], STAGE_BYTES);
          tma_load_2d(sA + stage * A_BYTES, &tmA, &full[stage], kb * BK, tm * BM);
          tma_load_2d(sB + stage * B_BYTES, &tmB, &full[stage], kb * BK, tn * BN);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok)   // let loads already in flight land before the CTA can exit
        for (int s = 0; s < STAGES; ++s) mbar_wait(&full[s], 0, nullptr, 100000000ull);
    } else if (warp == 1 && lane == 0) {
      constexpr uint32_t IDESC = umma_idesc_e4m3(BM, BN);
      uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
      bool issued = false;
      for (int t = first; t < total && ok; t += step) {
        for (int kb = 0; kb < nk; ++kb) {
          if (!mbar_wait_poll(&tempty[acc], acc_phase ^ 1, status) || !mbar_wait_poll(&full[stage], phase, status)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a0 = smem_u32(sA + stage * A_BYTES), b0 = smem_u32(sB + stage * B_BYTES);
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)
            umma_e4m3(tmem_base + acc * BN, umma_desc_sw128(a0 + k * 32), umma_desc_sw128(b0 + k * 32), IDESC, k != 0);
          issued = true;
          umma_commit(&tfull[acc]);
          umma_commit(&empty[stage]);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
          acc ^= 1;
          if (acc == 0) acc_phase ^= 1;
        }
      }
      if (!ok && issued) {   // wait (bounded) for every issued MMA before TMEM is freed
        umma_commit(drain);
        mbar_wait(drain, 0, nullptr, 100000000ull);
      }
    } else if (warp == 3) {
      uint32_t slot = 0, phase = 0;
      for (int t = first; t < total && ok; t += step) {
        int tm, tn;
        tile_coords(t, num_m, num_n, GROUP, tm, tn);
        const int row0 = tm * BM + lane;
        const float* src = lane < 2 ? g.sb.p + (int64_t)min(2 * tn + lane, (N - 1) / BK) * g.sb.row : nullptr;
        for (int kb = 0; kb < nk; kb += SC_KB) {
          ok = mbar_wait_warp(&sempty[slot], phase ^ 1, status);
          if (!ok) break;
          const uint32_t dst = smem_u32(scales + slot * SC_ROW);
          for (int k = 0; k < min(SC_KB, nk - kb); ++k) {
#pragma unroll
            for (int i = 0; i < BM / 32; ++i) {
              const int row = row0 + 32 * i;
              cp_async4(dst + 4 * (k * BM + 32 * i + lane), g.sa.p + (row < M ? row * g.sa.row + (kb + k) * g.sa.col : 0),
                        row < M);
            }
            if (lane < 2) cp_async4(dst + 4 * (SC_KB * BM + 2 * k + lane), src + (kb + k) * g.sb.col, true);
          }
          cp_async_arrive(&sfull[slot]);
          if (++slot == SC_SLOTS) {
            slot = 0;
            phase ^= 1;
          }
        }
      }
      cp_async_commit();
      cp_async_wait<0>();
    }
  } else {
    regs_inc<REGS_EPI>();
    // A warp reads the TMEM lanes of its number modulo four.  One whose wait ran out takes part in the barriers
    // all the same, so that the others reach their end, and stores nothing.
    const int quad = warp & 3, wg = (warp - 4) >> 2;
    uint32_t acc = 0, acc_phase = 0, slot = 0, sc_phase = 0;
    int parity = 0;
    for (int t = first; t < total; t += step, parity ^= 1) {
      int tm, tn;
      tile_coords(t, num_m, num_n, GROUP, tm, tn);
      const int row_in = quad * 32 + lane, row = tm * BM + row_in;
      const bool in = row < M;
      float sum[128];                         // columns [64 wg, 64 wg + 64) of the tile, then those 128 further on
#pragma unroll
      for (int i = 0; i < 128; ++i) sum[i] = 0.f;
      for (int kb = 0; kb < nk; ++kb) {
        const int k = kb & (SC_KB - 1);
        if (k == 0) ok = ok && mbar_wait_warp(&sfull[slot], sc_phase, status);
        const float* sc = scales + slot * SC_ROW;
        const float sa = sc[k * BM + row_in];
        const float2 sb = *reinterpret_cast<const float2*>(sc + SC_KB * BM + 2 * k);
        const float f0 = sa * sb.x, f1 = sa * sb.y;
        ok = ok && mbar_wait_warp(&tfull[acc], acc_phase, status);
        if (ok) {
          tc_fence_after();
          const uint32_t tb = tmem_base + acc * BN + wg * 64 + ((uint32_t)(quad * 32) << 16);
          // 32 columns are multiplied while the next 32 come
          uint32_t r[2][32];
          tmem_ld32(tb, r[0]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            tmem_ld_wait_for(r[c & 1]);
            if (c < 3) {
              tmem_ld32(tb + ((c + 1) >> 1) * 128 + ((c + 1) & 1) * 32, r[(c + 1) & 1]);
            } else {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&tempty[acc]);
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) sum[c * 32 + i] = fmaf(__uint_as_float(r[c & 1][i]), c < 2 ? f0 : f1, sum[c * 32 + i]);
          }
        }
        if (k == SC_KB - 1 || kb == nk - 1) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&sempty[slot]);
          if (++slot == SC_SLOTS) {
            slot = 0;
            sc_phase ^= 1;
          }
        }
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
      // ---- the tile's outputs
      if constexpr (EPI == EPI_SILU_MUL) {
        float h[64];
#pragma unroll
        for (int i = 0; i < 64; ++i) h[i] = silu_fast(sum[i]) * sum[64 + i];
        const int col = tn * 128 + wg * 64;
        if constexpr (QUANT) {
          float top = 0.f;
#pragma unroll
          for (int i = 0; i < 64; ++i) top = fmaxf(top, fabsf(h[i]));     // (passes over NaN)
          if (!(top < INFINITY)) {              // infinities become NaN and do not count
            top = 0.f;
#pragma unroll
            for (int i = 0; i < 64; ++i) {
              top = fmaxf(top, finite_or_zero(h[i]));
              if (fabsf(h[i]) == INFINITY) h[i] = __uint_as_float(0x7fffffffu);
            }
          }
          float* mine = tops + parity * 2 * BM;
          mine[wg * BM + row_in] = top;
          bar_sync(1, 32 * EPI_WARPS);         // once per tile: the other parity's maxima have been read by then
          top = fmaxf(fmaxf(top, mine[(wg ^ 1) * BM + row_in]), q8::TINY);
          if (ok && in) {
            const float mul = q8::TOP / top;
            uint8_t* d = reinterpret_cast<uint8_t*>(g.d) + (int64_t)row * g.ldd + col;
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              u128 o;
              uint32_t* po = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                po[e] = to_e4m3x2(h[16 * v + 4 * e] * mul, h[16 * v + 4 * e + 1] * mul) |
                        to_e4m3x2(h[16 * v + 4 * e + 2] * mul, h[16 * v + 4 * e + 3] * mul) << 16;
              st_v4(d + 16 * v, o);
            }
            if (wg == 0) g.sd.p[row * g.sd.row + tn * g.sd.col] = top / q8::TOP;
          }
        } else if (ok && in) {
          __nv_bfloat16* d = reinterpret_cast<__nv_bfloat16*>(g.d) + (int64_t)row * g.ldd + col;
#pragma unroll
          for (int v = 0; v < 8; ++v)
            st_v4(d + 8 * v, u128{pack_bf16x2(h[8 * v], h[8 * v + 1]), pack_bf16x2(h[8 * v + 2], h[8 * v + 3]),
                                  pack_bf16x2(h[8 * v + 4], h[8 * v + 5]), pack_bf16x2(h[8 * v + 6], h[8 * v + 7])});
        }
      } else if (ok && in) {
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int col = tn * BN + (v >> 3) * 128 + wg * 64 + (v & 7) * 8;
          if (col >= N) continue;
          u128 o;
          uint32_t* po = reinterpret_cast<uint32_t*>(&o);
          if constexpr (EPI == EPI_ADD) {
            const u128 rv = ld_v4(reinterpret_cast<const __nv_bfloat16*>(g.r) + (int64_t)row * g.ldr + col);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              po[e] = pack_bf16x2(sum[8 * v + 2 * e] + bf16_lo(word(rv, e)), sum[8 * v + 2 * e + 1] + bf16_hi(word(rv, e)));
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) po[e] = pack_bf16x2(sum[8 * v + 2 * e], sum[8 * v + 2 * e + 1]);
          }
          st_v4(reinterpret_cast<__nv_bfloat16*>(g.d) + (int64_t)row * g.ldd + col, o);
        }
      }
    }
  }

  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

template <int EPI, bool QUANT>
static void launch_gemm_fp8(const GemmFp8& g, int sms, int* status, cudaStream_t stream) {
  using namespace g8;
  auto kern = gemm_fp8_kernel<EPI, QUANT>;
  static bool attr[64] = {};
  int dev;
  cudaGetDevice(&dev);
  if (!attr[dev & 63]) {
    cudaFuncAttributes a;
    if (cudaFuncGetAttributes(&a, kern) != cudaSuccess || a.numRegs * THREADS < REGS_ALL)
      throw std::runtime_error("cx gemm_fp8: built with fewer registers than its warpgroups take");   // they would wait
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    attr[dev & 63] = true;
  }
  const CUtensorMap ta = make_tmap_u8_2d(g.a, (uint64_t)g.K, (uint64_t)g.M, (uint64_t)g.lda, BK, BM);
  const CUtensorMap tb = make_tmap_u8_2d(g.b, (uint64_t)g.K, (uint64_t)g.N, (uint64_t)g.ldb, BK, BN);
  const int64_t tiles = (int64_t)((g.M + BM - 1) / BM) * ((g.N + BN - 1) / BN);
  kern<<<(int)std::min<int64_t>(tiles, sms), THREADS, SMEM, stream>>>(ta, tb, g, status);
}

void gemm_fp8(const GemmFp8& g, int sms, int* status, cudaStream_t stream) {
  if (g.M == 0 || g.N == 0) return;
  if (g.epi == EPI_SILU_MUL && g.sd.p != nullptr) launch_gemm_fp8<EPI_SILU_MUL, true>(g, sms, status, stream);
  else if (g.epi == EPI_SILU_MUL) launch_gemm_fp8<EPI_SILU_MUL, false>(g, sms, status, stream);
  else if (g.epi == EPI_ADD) launch_gemm_fp8<EPI_ADD, false>(g, sms, status, stream);
  else launch_gemm_fp8<EPI_STORE, false>(g, sms, status, stream);
}

}  // namespace cx
