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

// A half-warp per block, eight columns of a lane; a CTA takes 2^lc column blocks of 16 / 2^lc rows at a time, four such
// groups of rows in flight.  8192 x 4096 take 22.2 us, 0.72 of a copy's rate.  The grid is at most 1184 CTAs; at 46
// registers an SM holds five of them, 740 on 148, so that many rows run as 1.6 rounds of CTAs: that, and not DRAM, is
// what is left there.  (With a running block number, divided by the row's blocks in 64 bits, 35 us.)
__global__ void __launch_bounds__(q8::THREADS)
    quantize_fp8_kernel(const __nv_bfloat16* __restrict__ x, int64_t ldx, uint8_t* __restrict__ q, int64_t ldq,
                        Fp8Scales s, int T, int K, int lc) {
  using namespace q8;
  constexpr int UNROLL = 4;
  const int hw = threadIdx.x >> 4, j = threadIdx.x & 15;
  const int b = (blockIdx.x << lc) + (hw & ((1 << lc) - 1)), c = b * Q + 8 * j;
  const int64_t step = (int64_t)gridDim.y << (4 - lc), row0 = ((int64_t)blockIdx.y << (4 - lc)) + (hw >> lc);
  for (int64_t r0 = (int64_t)blockIdx.y << (4 - lc); r0 < T; r0 += UNROLL * step) {        // the same for the whole CTA
    const int64_t first = row0 + (r0 - ((int64_t)blockIdx.y << (4 - lc)));
    u128 raw[UNROLL];
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      const int64_t row = first + i * step;
      raw[i] = row < T && c < K ? ld_nc_v4(x + row * ldx + c) : u128{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      const int64_t row = first + i * step;
      // magnitudes as pairs of bf16 (NaN is passed over)
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw[i]);
      const uint32_t m = max_abs_bf16x2(max_abs_bf16x2(w[0], w[1]), max_abs_bf16x2(w[2], w[3])) & 0x7fff7fffu;
      float top = fmaxf(bf16_lo(m), bf16_hi(m));
      const bool odd = !(top < INFINITY);
      if (odd) {
        float v[8];
        unpack8(raw[i], v);
        top = top8(v);
      }
      top = fmaxf(half_warp_max(top), TINY);
      const float mul = TOP / top;
      if (row < T && c < K) {
        uint32_t o[4];
        const uint64_t mul2 = f32x2(mul, mul);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint64_t r = mul_f32x2(unpack_bf16x2(w[e]), mul2);
          o[e] = odd ? quant_pair(bf16_lo(w[e]), bf16_hi(w[e]), mul) : to_e4m3x2(lo_f32(r), hi_f32(r));
        }
        *reinterpret_cast<uint2*>(q + row * ldq + c) = make_uint2(o[0] | o[1] << 16, o[2] | o[3] << 16);
        if (j == 0) s.p[row * s.row + b * s.col] = top / TOP;
      }
    }
  }
}

// The same behind an RMS norm: a CTA per row, the row in registers (read once, where the norm's sum needs all of it
// before the first code).  64 x 4096 take 2.2 us, a launch and a row's read, sum and write; 8192 x 4096 28 to 30 us, 3.5
// TB/s: a row's barrier stands between its reads and its writes, and nothing of a CTA's next row is under way there.
// (Weights read behind the barrier, infinities looked for in every element: 2.5 and 2.7 more than 28.)
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
  // (the weights come from the L2 while the row is on its way; eight words of them would take too many registers)
  constexpr bool EARLY = VPT <= 4;
  u128 gain[EARLY ? VPT : 1];
  if constexpr (EARLY) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (i * THREADS + tid) * 8;
      gain[i] = c < K ? ld_v4(w + c) : u128{0, 0, 0, 0};
    }
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
  const uint64_t inv2 = f32x2(inv, inv);
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if (i * THREADS * 8 >= K) break;
    const int c = (i * THREADS + tid) * 8;
    u128 g;
    if constexpr (EARLY) g = gain[i];
    else g = c < K ? ld_v4(w + c) : u128{0, 0, 0, 0};
    uint64_t v[4];
    float top = 0.f;                           // (a maximum passes over NaN)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = mul_f32x2(mul_f32x2(unpack_bf16x2(word(raw[i], e)), inv2), unpack_bf16x2(word(g, e)));
      top = fmaxf(top, fmaxf(fabsf(lo_f32(v[e])), fabsf(hi_f32(v[e]))));
    }
    const bool odd = !(top < INFINITY);
    if (odd) {
      top = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmaxf(top, fmaxf(finite_or_zero(lo_f32(v[e])), finite_or_zero(hi_f32(v[e]))));
    }
    top = fmaxf(half_warp_max(top), TINY);
    const float mul = TOP / top;
    if (c < K) {
      const uint64_t mul2 = f32x2(mul, mul);
      uint32_t o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint64_t r = mul_f32x2(v[e], mul2);
        o[e] = odd ? quant_pair(lo_f32(v[e]), hi_f32(v[e]), mul) : to_e4m3x2(lo_f32(r), hi_f32(r));
      }
      *reinterpret_cast<uint2*>(q + row * ldq + c) = make_uint2(o[0] | o[1] << 16, o[2] | o[3] << 16);
      if ((tid & 15) == 0) s.p[row * s.row + (c / Q) * s.col] = top / TOP;
    }
  }
}

// A CTA per 128 x 128 block of a weight: 28672 x 4096 take 76 us, 4.6 TB/s (once, as weights are loaded).
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
    int lc = 0;
    while (lc < 4 && 1 << lc < kb) ++lc;
    const int gx = (kb + (1 << lc) - 1) >> lc;
    const int64_t groups = ((int64_t)T + (16 >> lc) - 1) >> (4 - lc);          // of rows
    const int gy = (int)std::max<int64_t>(1, std::min<int64_t>(groups, std::max(1, 148 * 8 / gx)));
    quantize_fp8_kernel<<<dim3(gx, gy), THREADS, 0, stream>>>(X, ldx, O, ldq, s, T, K, lc);
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
//   warp 2      the time limit of the others' waits
//   warp 3      the scales of the CTA's rows and of the tile's two blocks of B, up to sixteen blocks of 128 columns ahead (each
//               is a line of its own: fetched one block ahead by the warps that use them they took longer than the MMAs)
//   warps 4-11  promotion: two warpgroups; a thread takes a row, and columns [64 g, 64 g + 64) of both halves of
//               the tile, reads the block's sums from TMEM, multiplies by the scales and adds in registers.  One
//               accumulator is read while the MMAs fill the other.
// 8192 x 28672 x 4096 with SiLU(gate) * up takes 965 us at full clock (up to 1130 after seconds of load), 6144 columns
// without it 224; the MMAs are half of the time (513 of 1040 cycles of a block, outputs included).  The other half is
// owned in part: the way round of an accumulator is its MMAs, the word that it is complete (some 260), its promotion by
// two warps on each SM quarter (350 to 600), the word that it is free (90), and two accumulators of 256 columns are all
// of TMEM, so a block takes 700 cycles at least (an SM by itself, operands in place).  What takes the rest is not known;
// a block's operands are 48 KB, 47 bytes a cycle, about what comes to an SM in the kernel for few rows, too.
// Variants, timed when the waits had their clocks in each lane and an MMA took 75 cycles to issue, this form then 1020
// us: pairs of CTAs on one tile of 256 x 256 (cta_group::2) 1060; four warpgroups of half the columns 1190; four
// accumulators of 128 columns 1280; barriers waited for in mbarrier.try_wait, which suspends, 1150.  They have not been
// timed since.
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

static_assert(GEMM_FP8_WAIT_NS == kDefaultWaitNs, "one default limit");
// The limit that a CTA's waits have; 0: it loses its operands.
__device__ __forceinline__ uint64_t cta_wait_ns(uint64_t wait_ns) {
  return wait_ns != 0 ? wait_ns : blockIdx.x & 1 ? 0 : kDefaultWaitNs;
}
// What a producer does before its CTA ends: the last load into each stage, of `n` loads into the stages in turn, has a
// bounded time to land.
template <int STAGES>
__device__ __forceinline__ void drain_loads(uint64_t* full, int n) {
  for (int s = 0; s < STAGES && s < n; ++s) mbar_wait(&full[s], (n - 1 - s) / STAGES & 1, nullptr, 100000000ull);
}
// What the warp that issued MMAs does: all of them have a bounded time to end before TMEM is freed.
__device__ __forceinline__ void drain_mmas(uint64_t* drain) {
  __syncwarp();
  if (elect_sync()) umma_commit(drain);
  __syncwarp();
  mbar_wait(drain, 0, nullptr, 100000000ull);
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
  WaitKeeper* keeper = reinterpret_cast<WaitKeeper*>(drain + 1);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(keeper + 1);
  const uint32_t* lost = &keeper->lost;

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
    keeper->init(EPI_WARPS);
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
  // 0 once a wait was lost.  What consumed or filled nothing says so to no other warp, so none takes a result for
  // complete that is not.
  uint32_t ok = 1;

  if (warp < 4) {
    regs_dec<REGS_AUX>();
    // (Whole warps walk through the loops and one thread acts: what the instructions take in uniform registers then
    // lies there.  Left to one thread's branch, an MMA took 75 cycles to issue.)
    if (warp == 0) {
      uint32_t stage = 0, phase = 0;
      int loads = 0;
      for (int t = first; t < total && ok; t += step) {
        int tm, tn;
        tile_coords(t, num_m, num_n, GROUP, tm, tn);
        for (int kb = 0; kb < nk; ++kb) {
          ok = mbar_wait_poll(&empty[stage], phase ^ 1, lost);
          if (!ok) break;
          ++loads;
          if (elect_sync()) {
            mbar_arrive_expect_tx(&full[stage], STAGE_BYTES);
            tma_load_2d(sA + stage * A_BYTES, &tmA, &full[stage], kb * BK, tm * BM);
            tma_load_2d(sB + stage * B_BYTES, &tmB, &full[stage], kb * BK, tn * BN);
          }
          __syncwarp();
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      drain_loads<STAGES>(full, loads);
    } else if (warp == 1) {
      if (cta_wait_ns(g.wait_ns) == 0) ok = 0;
      constexpr uint32_t IDESC = umma_idesc_e4m3(BM, BN);
      const uint32_t a_lo = umma_desc_sw128_lo(smem_u32(sA)), b_lo = umma_desc_sw128_lo(smem_u32(sB));
      uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
      uint32_t blocks = 0;
      for (int t = first; t < total && ok; t += step) {
        for (int kb = 0; kb < nk; ++kb) {
          ok = mbar_wait_poll(&tempty[acc], acc_phase ^ 1, lost) && mbar_wait_poll(&full[stage], phase, lost);
          if (!ok) break;
          tc_fence_after();
          ++blocks;
          if (elect_sync()) {
            const uint32_t al = a_lo + stage * (A_BYTES / 16), bl = b_lo + stage * (B_BYTES / 16);
#pragma unroll
            for (int k = 0; k < BK / 32; ++k)
              umma_e4m3(tmem_base + acc * BN, umma_desc_sw128_of(al + 2 * k), umma_desc_sw128_of(bl + 2 * k), IDESC, k != 0);
            umma_commit(&tfull[acc]);
            umma_commit(&empty[stage]);
            keeper->advance(blocks);
          }
          __syncwarp();
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
          acc ^= 1;
          if (acc == 0) acc_phase ^= 1;
        }
      }
      drain_mmas(drain);
    } else if (warp == 2) {
      if (lane == 0) keeper->keep(cta_wait_ns(g.wait_ns), status);
      __syncwarp();
    } else if (warp == 3) {
      uint32_t slot = 0, phase = 0;
      for (int t = first; t < total && ok; t += step) {
        int tm, tn;
        tile_coords(t, num_m, num_n, GROUP, tm, tn);
        const int row0 = tm * BM + lane;
        const float* src = lane < 2 ? g.sb.p + (int64_t)min(2 * tn + lane, (N - 1) / BK) * g.sb.row : nullptr;
        for (int kb = 0; kb < nk; kb += SC_KB) {
          mbar_wait_warp(&sempty[slot], phase ^ 1, lost, ok);
          if (!ok) break;                        // (nothing here takes the whole warp)
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
    // A warp reads the TMEM lanes of its number modulo four.  A lane that lost a wait reads on all the same, and the warp's
    // outputs from then on are NaN.
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
        if (k == 0) mbar_wait_warp(&sfull[slot], sc_phase, lost, ok);
        const float* sc = scales + slot * SC_ROW;
        const float sa = sc[k * BM + row_in];
        const float2 sb = *reinterpret_cast<const float2*>(sc + SC_KB * BM + 2 * k);
        const float f0 = sa * sb.x, f1 = sa * sb.y;
        mbar_wait_warp(&tfull[acc], acc_phase, lost, ok);
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
            if (lane == 0 && ok) mbar_arrive(&tempty[acc]);
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) sum[c * 32 + i] = fmaf(__uint_as_float(r[c & 1][i]), c < 2 ? f0 : f1, sum[c * 32 + i]);
        }
        if (k == SC_KB - 1 || kb == nk - 1) {
          __syncwarp();
          if (lane == 0 && ok) mbar_arrive(&sempty[slot]);
          if (++slot == SC_SLOTS) {
            slot = 0;
            sc_phase ^= 1;
          }
        }
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
      if (lane == 0 && t + step >= total) mbar_arrive(&keeper->done);   // no wait is left
      // ---- the tile's outputs
      ok = __all_sync(0xffffffffu, ok);
      if (!ok)
#pragma unroll
        for (int i = 0; i < 128; ++i) sum[i] = __uint_as_float(0x7fffffffu);
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
          if (in) {
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
        } else if (in) {
          __nv_bfloat16* d = reinterpret_cast<__nv_bfloat16*>(g.d) + (int64_t)row * g.ldd + col;
#pragma unroll
          for (int v = 0; v < 8; ++v)
            st_v4(d + 8 * v, u128{pack_bf16x2(h[8 * v], h[8 * v + 1]), pack_bf16x2(h[8 * v + 2], h[8 * v + 3]),
                                  pack_bf16x2(h[8 * v + 4], h[8 * v + 5]), pack_bf16x2(h[8 * v + 6], h[8 * v + 7])});
        }
      } else if (in) {
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

// ------------------------------------------------------- few rows: split K
// Where the 128 x 256 tiles would leave SMs idle: the weight's rows are the MMA's 128 rows and NT activations its
// columns (or 128 activations its rows and 128 weight rows its columns), and the CTAs of a cluster share a tile's blocks
// of 128 columns among them.  Each adds up its part in registers as above (a thread per MMA row; the scales of a block
// lie in shared memory, a's times b's), leaves it in shared memory, and the CTAs then add the parts of a slice of the
// activations each, in the order of their ranks, over the cluster's shared memory: no workspace, no atomics, the same
// bits from run to run.  A warp writes a row of 128 outputs.  SiLU-mul takes R = 2 blocks of weight rows, gate and up.
// What bounds it: a block of 128 columns takes a CTA 500 to 700 cycles, as long with two warpgroups that add up the
// blocks in turn or with half the waits of the issuing thread: 40 to 50 bytes a cycle come to an SM.  5 to 6 us pass
// around that (launch, first loads, the cluster's sums).  Times are with other weights each call, none of them in the L2:
// 64 x 4096 x 14336 takes 16.8 us where reading the operands takes 9.4.  With activations as columns a thread needs another scale for each of its sums, and shared
// memory brings 32 of them a cycle: 1024 cycles for 256 activations.  So 128 of them are rows, a scale a thread: 613 x
// 2048 x 4096 takes 18.2 us (256 activations as columns 26.2), 512 x 4096 x 14336 47.3 (63).
namespace g8s {
constexpr int BK = 128, Q = 128;
constexpr int SC_SLOTS = 2;
template <int NT, int R>
struct Cfg {
  // two CTAs on an SM where their stages and registers fit: one computes while the other waits
  static constexpr int PER_SM = R * NT <= 32 ? 2 : 1;
  static constexpr bool TALL = NT == Q;           // the activations are the MMA's rows
  // Blocks of columns of a stage, its waits and commits.  (512 x 4096 x 14336 52.0 us with one; with two, 64 x 4096 x
  // 14336 17.9 us, with one 17.4: fewer loads are on their way at the start.)
  static constexpr int KS = TALL ? 2 : 1;
  static constexpr int A_BYTES = R * Q * BK, B_BYTES = NT * BK, BLOCK = A_BYTES + B_BYTES, STAGE = KS * BLOCK;
  static constexpr int SC_KB = R == 1 && NT <= 64 ? 8 : 4;  // blocks of columns whose scales come together
  static constexpr int SCALES = SC_SLOTS * SC_KB * R * NT * 4;
  // In the stages, once they are empty.  (Eight lanes that store four columns of a row each: rows 16 bytes apart in the
  // banks.)
  static constexpr int PITCH = R * Q + (TALL ? 4 : 0), PARTS = NT * PITCH * 4;
  static constexpr int ROOM = (PER_SM == 2 ? 113 * 1024 : 200 * 1024) - SCALES - 1024 - 512;
  static constexpr int STAGES = ROOM / STAGE;
  static_assert(STAGES >= 2 && PARTS <= STAGES * STAGE, "stages");
  static constexpr int SMEM = 1024 + STAGES * STAGE + SCALES + 512;
  // Accumulators in TMEM, up to eight: a block's sums are read some 1000 cycles after its MMAs have begun.
  static constexpr int ACCS = (512 / PER_SM / (R * NT) < 8 ? 512 / PER_SM / (R * NT) : 8) / KS;    // groups of KS
  static constexpr int COLS = ACCS * KS * R * NT;
  static constexpr int GROUPS = R * NT >= 128 ? 2 : 1, THREADS = 128 + 128 * GROUPS;
  static constexpr int MINE = NT / GROUPS;        // sums of a thread, of each r
  static constexpr int CH = MINE >= 32 ? 32 : 16; // of them, read from TMEM at a time
  static_assert(!TALL || R == 1, "one block of weight rows");
};
}  // namespace g8s

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait_for(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

template <int NT, int R>
__global__ void __launch_bounds__(g8s::Cfg<NT, R>::THREADS, g8s::Cfg<NT, R>::PER_SM)
    gemm_fp8_split_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, GemmFp8 g,
                          int splits, int* status) {
  using namespace g8s;
  using C = Cfg<NT, R>;
  constexpr int STAGES = C::STAGES, SC_KB = C::SC_KB, KS = C::KS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* parts = reinterpret_cast<float*>(smem);                                 // [NT][R * 128]
  float* scales = reinterpret_cast<float*>(smem + STAGES * C::STAGE);            // [slot][SC_KB][R][NT]
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * C::STAGE + C::SCALES);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + C::ACCS;
  uint64_t* sfull = tempty + C::ACCS;
  uint64_t* sempty = sfull + SC_SLOTS;
  uint64_t* drain = sempty + SC_SLOTS;
  uint64_t* landed = drain + 1;
  WaitKeeper* keeper = reinterpret_cast<WaitKeeper*>(landed + 1);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(keeper + 1);
  const uint32_t* lost = &keeper->lost;

  const int warp = warp_id(), lane = lane_id();
  const int rank = blockIdx.x % splits, tile = blockIdx.x / splits, m0 = blockIdx.y * NT;
  const int nk = (g.K + BK - 1) / BK;
  const int k0 = (int)((int64_t)nk * rank / splits), k1 = (int)((int64_t)nk * (rank + 1) / splits);

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < C::ACCS; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 4 * C::GROUPS);
    }
    for (int i = 0; i < SC_SLOTS; ++i) {
      mbar_init(&sfull[i], 32);
      mbar_init(&sempty[i], 4 * C::GROUPS);
    }
    mbar_init(drain, 1);
    mbar_init(landed, 32);
    keeper->init(4 * C::GROUPS);
    fence_barrier_init();
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::COLS);
    tmem_relinquish();
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  uint32_t ok = 1;                         // as above

  if (warp == 0) {
    uint32_t stage = 0, phase = 0;
    int loads = 0;
    for (int kb = k0; kb < k1; kb += KS) {
      // (no wait for what is empty at first, nor for the accumulators below: 1 x 6144 x 4096 8.7 us, 8.95 with them)
      ok = loads < STAGES || mbar_wait_poll(&empty[stage], phase ^ 1, lost);
      if (!ok) break;
      ++loads;
      if (elect_sync()) {
        uint8_t* at = smem + stage * C::STAGE;
        mbar_arrive_expect_tx(&full[stage], min(KS, k1 - kb) * C::BLOCK);
#pragma unroll
        for (int j = 0; j < KS; ++j, at += C::BLOCK)
          if (kb + j < k1) {
            tma_load_2d(at, &tmB, &full[stage], (kb + j) * BK, tile * R * Q);    // the weight
            tma_load_2d(at + C::A_BYTES, &tmA, &full[stage], (kb + j) * BK, m0);
          }
      }
      __syncwarp();
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1;
      }
    }
    drain_loads<STAGES>(full, loads);
    mbar_arrive(landed);
  } else if (warp == 1) {
    if (cta_wait_ns(g.wait_ns) == 0) ok = 0;
    constexpr uint32_t IDESC = umma_idesc_e4m3(Q, NT);
    const uint32_t w_lo = umma_desc_sw128_lo(smem_u32(smem));
    uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
    for (int kb = k0; kb < k1 && ok; kb += KS) {
      ok = (kb - k0 < C::ACCS * KS || mbar_wait_poll(&tempty[acc], acc_phase ^ 1, lost)) &&
           mbar_wait_poll(&full[stage], phase, lost);
      if (!ok) break;
      tc_fence_after();
      if (elect_sync()) {
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          // (the two operands' tiles have the same size where they change places)
          const uint32_t at = w_lo + (stage * C::STAGE + j * C::BLOCK) / 16, other = at + C::A_BYTES / 16;
          const uint32_t wl = C::TALL ? other : at, xl = C::TALL ? at : other;
          if (kb + j < k1)
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
              for (int k = 0; k < BK / 32; ++k)
                umma_e4m3(tmem_base + ((acc * KS + j) * R + r) * NT, umma_desc_sw128_of(wl + r * (Q * BK / 16) + 2 * k),
                          umma_desc_sw128_of(xl + 2 * k), IDESC, k != 0);
        }
        umma_commit(&tfull[acc]);
        umma_commit(&empty[stage]);
        keeper->advance(kb + 1);
      }
      __syncwarp();
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1;
      }
      if (++acc == C::ACCS) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
    drain_mmas(drain);
  } else if (warp == 2) {
    if (lane == 0) keeper->keep(cta_wait_ns(g.wait_ns), status);
  } else if (warp == 3) {
    // A batch's scales are on their way while the one before is written: the loads take a microsecond and more, as
    // long as several blocks' MMAs.
    constexpr int PER = (NT + 31) / 32;
    uint32_t slot = 0, phase = 0;
    const int last = (g.N - 1) / Q;
    float v[SC_KB][PER], b[SC_KB][R];
    auto load = [&](int kb) {
#pragma unroll
      for (int k = 0; k < SC_KB; ++k) {
        const bool there = kb + k < k1;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int m = m0 + 32 * i + lane;
          v[k][i] = there && m < g.M ? __ldg(g.sa.p + m * g.sa.row + (kb + k) * g.sa.col) : 0.f;
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
          b[k][r] = there ? __ldg(g.sb.p + min(tile * R + r, last) * g.sb.row + (kb + k) * g.sb.col) : 0.f;
      }
    };
    load(k0);
    for (int kb = k0; kb < k1 && ok; kb += SC_KB) {
      float f[SC_KB][R][PER];
#pragma unroll
      for (int k = 0; k < SC_KB; ++k)
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < PER; ++i) f[k][r][i] = v[k][i] * b[k][r];
      load(kb + SC_KB);
      mbar_wait_warp(&sempty[slot], phase ^ 1, lost, ok);
      if (!ok) break;
#pragma unroll
      for (int k = 0; k < SC_KB; ++k)
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < PER; ++i)
            if (32 * i + lane < NT) scales[((slot * SC_KB + k) * R + r) * NT + 32 * i + lane] = f[k][r][i];
      mbar_arrive(&sfull[slot]);
      if (++slot == SC_SLOTS) {
        slot = 0;
        phase ^= 1;
      }
    }
  } else if (warp >= 4) {
    const int quad = warp & 3, wg = (warp - 4) >> 2;
    uint32_t acc = 0, acc_phase = 0, slot = 0, sc_phase = 0;
    float sum[R][C::MINE];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < C::MINE; ++i) sum[r][i] = 0.f;
    for (int kb = k0; kb < k1; ++kb) {
      const int k = (kb - k0) & (SC_KB - 1), j = k & (KS - 1);
      const bool last = j == KS - 1 || kb == k1 - 1;           // of its group
      if (k == 0) mbar_wait_warp(&sfull[slot], sc_phase, lost, ok);
      if (j == 0) mbar_wait_warp(&tfull[acc], acc_phase, lost, ok);
      if (lane == 0 && kb == k1 - 1) mbar_arrive(&keeper->done);     // the last wait
      tc_fence_after();
      const uint32_t tb = tmem_base + (acc * KS + j) * R * NT + wg * C::MINE + ((uint32_t)(quad * 32) << 16);
      const float* sc = scales + (slot * SC_KB + k) * R * NT + (C::TALL ? quad * 32 + lane : wg * C::MINE);
      if constexpr (C::TALL) {
        static_assert(C::MINE == 64, "two reads of 32");
        uint32_t t[2][32];
        tmem_ld32(tb, t[0]);
        tmem_ld32(tb + 32, t[1]);
        const float f = *sc;
        tmem_ld_wait_for(t[0]);
        tmem_ld_wait_for(t[1]);
        if (last) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0 && ok) mbar_arrive(&tempty[acc]);
        }
#pragma unroll
        for (int i = 0; i < 64; ++i) sum[0][i] = fmaf(__uint_as_float(t[i >> 5][i & 31]), f, sum[0][i]);
      } else {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int c = 0; c < C::MINE / C::CH; ++c) {
            uint32_t t[C::CH];
            if constexpr (C::CH == 32) tmem_ld32(tb + r * NT + c * C::CH, t);
            else tmem_ld16(tb + r * NT + c * C::CH, t);
            float4 f[C::CH / 4];
#pragma unroll
            for (int i = 0; i < C::CH / 4; ++i) f[i] = *reinterpret_cast<const float4*>(sc + r * NT + c * C::CH + 4 * i);
            tmem_ld_wait_for(t);
            if (r == R - 1 && c == C::MINE / C::CH - 1 && last) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0 && ok) mbar_arrive(&tempty[acc]);
            }
#pragma unroll
            for (int i = 0; i < C::CH; ++i)
              sum[r][c * C::CH + i] =
                  fmaf(__uint_as_float(t[i]), reinterpret_cast<const float*>(f)[i], sum[r][c * C::CH + i]);
          }
      }
      if (k == SC_KB - 1 || kb == k1 - 1) {
        __syncwarp();
        if (lane == 0 && ok) mbar_arrive(&sempty[slot]);
        if (++slot == SC_SLOTS) {
          slot = 0;
          sc_phase ^= 1;
        }
      }
      if (last && ++acc == C::ACCS) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
    // Every MMA is complete and every stage read, for the last accumulator is.  A warp that lost a wait leaves NaN,
    // whichever rank adds it up, once the loads under way have landed.
    if (!__all_sync(0xffffffffu, ok)) {
      mbar_wait(landed, 0, nullptr);
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < C::MINE; ++i) sum[r][i] = __uint_as_float(0x7fffffffu);
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < C::MINE; ++i) {
        if constexpr (C::TALL) {
          if (i % 4 == 0)
            *reinterpret_cast<float4*>(parts + (quad * 32 + lane) * C::PITCH + wg * C::MINE + i) =
                make_float4(sum[r][i], sum[r][i + 1], sum[r][i + 2], sum[r][i + 3]);
        } else {
          parts[(wg * C::MINE + i) * C::PITCH + r * Q + quad * 32 + lane] = sum[r][i];
        }
      }
  }
  __syncwarp();
  __syncthreads();
  if (splits > 1) cluster_sync();

  // ---- a warp per row of outputs: the parts of all ranks in their order
  const int rows = min(NT, g.M - m0);
  const uint32_t base = smem_u32(parts);
  for (int i = rank + splits * warp; i < rows; i += splits * (C::THREADS / 32)) {
    float4 v[R];
#pragma unroll
    for (int r = 0; r < R; ++r) v[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < splits; ++s)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const uint32_t at = base + (i * C::PITCH + r * Q + 4 * lane) * 4;
        const float4 x = splits > 1 ? ld_cluster_f32x4(cluster_addr(at, s)) : *reinterpret_cast<const float4*>(
                                                                                  parts + i * C::PITCH + r * Q + 4 * lane);
        v[r].x += x.x;
        v[r].y += x.y;
        v[r].z += x.z;
        v[r].w += x.w;
      }
    const int64_t m = m0 + i;
    const int col = tile * Q + 4 * lane;
    if constexpr (R == 2) {
      float h[4] = {silu_fast(v[0].x) * v[1].x, silu_fast(v[0].y) * v[1].y, silu_fast(v[0].z) * v[1].z,
                    silu_fast(v[0].w) * v[1].w};
      if (g.sd.p != nullptr) {
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, finite_or_zero(h[e]));
        top = fmaxf(warp_max(top), q8::TINY);
        const float mul = q8::TOP / top;
        *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(g.d) + m * g.ldd + col) =
            quant_pair(h[0], h[1], mul) | quant_pair(h[2], h[3], mul) << 16;
        if (lane == 0) g.sd.p[m * g.sd.row + tile * g.sd.col] = top / q8::TOP;
      } else {
        *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(g.d) + m * g.ldd + col) =
            make_uint2(pack_bf16x2(h[0], h[1]), pack_bf16x2(h[2], h[3]));
      }
    } else if (col < g.N) {
      if (g.epi == EPI_ADD) {
        const uint2 x = *reinterpret_cast<const uint2*>(reinterpret_cast<const __nv_bfloat16*>(g.r) + m * g.ldr + col);
        v[0].x += bf16_lo(x.x);
        v[0].y += bf16_hi(x.x);
        v[0].z += bf16_lo(x.y);
        v[0].w += bf16_hi(x.y);
      }
      *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(g.d) + m * g.ldd + col) =
          make_uint2(pack_bf16x2(v[0].x, v[0].y), pack_bf16x2(v[0].z, v[0].w));
    }
  }
  __syncwarp();
  if (splits > 1) cluster_sync();          // no CTA ends while another may still read its parts
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::COLS);
  }
}

template <int NT, int R>
static void launch_gemm_fp8_split(const GemmFp8& g, int splits, int* status, cudaStream_t stream) {
  using C = g8s::Cfg<NT, R>;
  auto kern = gemm_fp8_split_kernel<NT, R>;
  static bool attr[64] = {};
  int dev;
  cudaGetDevice(&dev);
  if (!attr[dev & 63]) {
    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
    attr[dev & 63] = true;
  }
  const CUtensorMap ta = make_tmap_u8_2d(g.a, (uint64_t)g.K, (uint64_t)g.M, (uint64_t)g.lda, g8s::BK, NT);
  const CUtensorMap tb = make_tmap_u8_2d(g.b, (uint64_t)g.K, (uint64_t)g.N, (uint64_t)g.ldb, g8s::BK, R * g8s::Q);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((g.N + R * g8s::Q - 1) / (R * g8s::Q) * splits, (g.M + NT - 1) / NT);
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = splits;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kern, ta, tb, g, splits, status);
}

// Which way a call goes: the least of the estimated times, in us.  A CTA takes `per` for a block of 128 columns and a
// fixed start and end; clusters of four and eight do not fill every SM (132 and 120 of 148 are reached); reading the
// operands takes its time whatever the CTAs.  The constants are fits to measured calls: 4096 weight rows with K = 4096
// and 14336, one CTA per tile, and for the tiles of 128 x 256.  Estimated and measured (other weights each call): 1 x 6144 x
// 4096 8.3 and 8.7 (16 activations, four CTAs; one CTA 12.6, 128 x 256 tiles 21), 64 x 4096 x 14336 15.6 and 16.8 (64,
// four; 65), 613 x 2048 x 4096 17.8 and 18.2 (128, one; 29), 64 x 28672 x 4096 with SiLU-mul 25.6 and 25.1 (128 x 256
// tiles; 64 activations by one CTA 28), 512 x 4096 x 14336 48 and 47.3 (128, one; 71).
GemmFp8Plan gemm_fp8_plan(int M, int N, int K, int epi, int sms) {
  const int r = epi == EPI_SILU_MUL ? 2 : 1, nk = (K + 127) / 128;
  const double read = ((double)M + N) * K / 5.5e6 + 4.0;
  const int64_t tiles = (int64_t)((M + 127) / 128) * ((N + 255) / 256);
  GemmFp8Plan best{0, 1};
  double cost = std::max(read, (double)((tiles + sms - 1) / sms) * (nk * 0.55 + 8.0));
  constexpr double per[2][4] = {{0.26, 0.29, 0.32, 0.375}, {0.35, 0.45, 0.70, 0}};
  for (int i = 0; i < (r == 2 ? 3 : 4); ++i) {
    const int nt = 16 << i;
    const int64_t base = (int64_t)((M + nt - 1) / nt) * ((N + 128 * r - 1) / (128 * r));
    if (base > (int64_t)1 << 24 || (M + nt - 1) / nt > 65535) continue;
    for (int s = 1; s <= 8 && s <= nk; s *= 2) {
      const int64_t room = (int64_t)((r * nt <= 32 ? 2 : 1) * sms * (s == 8 ? 0.81 : s == 4 ? 0.89 : 1.0));
      const int64_t waves = (base * s + room - 1) / room;
      // two CTAs on an SM take 1.6 times as long
      const double crowd = 0.4 + 0.6 * std::min(std::max(base * s * (r * nt <= 32 ? 2.0 : 1.0) / room, 1.0), 2.0);
      const double c = std::max(read, waves * ((nk + s - 1) / s * per[r - 1][i] * (r * nt <= 32 ? crowd : 1.0) + 4.5 + (s > 1 ? 1.5 : 0.0) + 0.01 * r * nt));
      if (c < cost) {
        cost = c;
        best = {nt, s};
      }
    }
  }
  return best;
}

void gemm_fp8(const GemmFp8& g, int sms, int* status, cudaStream_t stream) {
  if (g.M == 0 || g.N == 0) return;
  const GemmFp8Plan p = gemm_fp8_plan(g.M, g.N, g.K, g.epi, sms);
  const bool two = g.epi == EPI_SILU_MUL;
  switch (p.nt) {
    case 16: return two ? launch_gemm_fp8_split<16, 2>(g, p.splits, status, stream) : launch_gemm_fp8_split<16, 1>(g, p.splits, status, stream);
    case 32: return two ? launch_gemm_fp8_split<32, 2>(g, p.splits, status, stream) : launch_gemm_fp8_split<32, 1>(g, p.splits, status, stream);
    case 64: return two ? launch_gemm_fp8_split<64, 2>(g, p.splits, status, stream) : launch_gemm_fp8_split<64, 1>(g, p.splits, status, stream);
    case 128: return launch_gemm_fp8_split<128, 1>(g, p.splits, status, stream);
    default: break;
  }
  if (two && g.sd.p != nullptr) launch_gemm_fp8<EPI_SILU_MUL, true>(g, sms, status, stream);
  else if (two) launch_gemm_fp8<EPI_SILU_MUL, false>(g, sms, status, stream);
  else if (g.epi == EPI_ADD) launch_gemm_fp8<EPI_ADD, false>(g, sms, status, stream);
  else launch_gemm_fp8<EPI_STORE, false>(g, sms, status, stream);
}

}  // namespace cx
