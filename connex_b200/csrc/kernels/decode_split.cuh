// How decode attention over the 4-bit cache is divided among CTAs, on the
// device, from the sequences' lengths.  (The kernel over the 8-bit cache holds
// the same division itself: what is mended here has to be mended there.)
//
// A pair is a (sequence, KV head).  The blocks of all pairs, laid end to end
// with PAIR_COST blocks' worth for the fixed cost of a pair, are cut into equal
// shares, one per CTA, so that the same launch (a graph replay) is balanced for
// any lengths.  Where no pair is longer than two shares, cuts move by up to
// SLACK blocks' worth to the pair's start or end.
//
// C: struct of WARPS, THREADS, BS (tokens of a block), MIN_UNITS (a CTA's
// blocks' worth, at least), PAIR_COST, SLACK.
#pragma once

#include "common.cuh"

namespace cx {

struct DecodeShare {
  int u0, u1;        // units of this CTA
  int b;             // the sequence that u0 falls into
  int per, most;     // units of a share; by how much a cut may move
};

template <class C>
__device__ __forceinline__ int decode_slack(int units, int most) {
  return min((units - C::PAIR_COST) / 2, most);
}

// pre: [B + 1] shared words, left as the units of the pairs before sequence b.
// Every thread of the CTA calls it.
template <class C>
__device__ __forceinline__ DecodeShare decode_share(const int* __restrict__ ctx_lens, int B, int max_blocks, int Hkv,
                                                    int* pre, int* status) {
  __shared__ int wsum[C::WARPS], wtop[C::WARPS];
  __shared__ int2 share[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) pre[0] = 0;
  int run = 0, top = 0;                                         // all units; the longest sequence's
  for (int b0 = 0; b0 < B; b0 += C::THREADS) {
    const int b = b0 + tid;
    int n = 0;
    if (b < B) {
      const int given = ctx_lens[b], len = min(max(given, 0), max_blocks * C::BS);
      if (given > max_blocks * C::BS && blockIdx.x == 0) record_status(status, CX_ERR_BOUNDS);
      n = len > 0 ? ((len + C::BS - 1) / C::BS + C::PAIR_COST) * Hkv : 0;
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
    for (int w = 0; w < C::WARPS; ++w) {
      if (w < warp) add += wsum[w];
      run += wsum[w];
      top = max(top, wtop[w]);
    }
    if (b < B) pre[b + 1] = add + x;
    __syncthreads();
  }
  const int total = run;
  const int n_cta = max(1, min((int)gridDim.x, (total + C::MIN_UNITS - 1) / C::MIN_UNITS));
  DecodeShare s;
  s.per = (total + n_cta - 1) / n_cta;
  s.most = top <= 2 * s.per * Hkv ? C::SLACK : 0;
  const int x = (blockIdx.x + (tid & 1)) * s.per;        // thread 0 finds the share's start, thread 1 its end
  int lo = 0, end = total;
  if (x < total) {
    int hi = B;                                         // the sequence that holds x: the last b with pre[b] <= x
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= x) lo = mid;
      else hi = mid;
    }
    const int units = (pre[lo + 1] - pre[lo]) / Hkv, into = (x - pre[lo]) % units;
    const int slack = decode_slack<C>(units, s.most);
    end = into <= C::PAIR_COST + slack ? x - into : units - into <= slack ? x - into + units : x;
  }
  // through shared memory, not shuffles: the compiler then knows that they are the same in all lanes
  if (tid < 2) share[tid] = make_int2(end, lo);
  __syncthreads();
  s.u0 = share[0].x;
  s.u1 = share[1].x;
  s.b = share[0].y;
  return s;
}

}  // namespace cx
