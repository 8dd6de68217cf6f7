// Host entry points of the block-scaled fp8 kernels (gemm_fp8.cu).
//
// An operand is e4m3 [rows, K] with one fp32 scale per block of 128 columns and
// one row (activations) or 128 rows (weights): an element stands for value *
// scale.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace cx {

struct Fp8Scales {     // scale of (row or row block r, column block c): p[r * row + c * col]
  float* p;
  int64_t row, col;
};

// x [T, K] bf16 (ld ldx), after an RMS norm with weights w where given -> q [T, K] e4m3 (ld ldq) and its scales.
constexpr int QUANT_NORM_MAX_K = 16384;
void quantize_fp8(const void* x, int64_t ldx, const void* w, float eps, void* q, int64_t ldq, const Fp8Scales& s, int T,
                  int K, cudaStream_t stream);
// w [N, K] bf16 (ld ldw) -> q [N, K] e4m3 (ld ldq), one scale per 128 x 128 block.
void quantize_weight_fp8(const void* w, int64_t ldw, void* q, int64_t ldq, const Fp8Scales& s, int N, int K,
                         cudaStream_t stream);

struct GemmFp8 {
  const void *a, *b;          // e4m3 [M, K] (ld lda), [N, K] (ld ldb)
  int64_t lda, ldb;
  Fp8Scales sa, sb;           // [M, K / 128], [N / 128, K / 128]
  int M, N, K;
  int epi;                    // GemmEpilogue
  void* d;                    // bf16 [M, N] (SiLU-mul: [M, N / 2]), or e4m3 [M, N / 2] with sd
  int64_t ldd;
  const void* r;              // bf16 [M, N], may be d
  int64_t ldr;
  Fp8Scales sd;               // p == nullptr: bf16 output
  uint64_t wait_ns;           // limit of a wait (0: every other CTA loses its operands); outputs that lost theirs are NaN
};
constexpr uint64_t GEMM_FP8_WAIT_NS = 2000000000ull;
// How a call runs: nt = 0: tiles of 128 x 256; else tiles of 128 weight rows (SiLU-mul: 256) by nt activations,
// each shared by `splits` CTAs.
struct GemmFp8Plan {
  int nt, splits;
};
GemmFp8Plan gemm_fp8_plan(int M, int N, int K, int epi, int sms);
void gemm_fp8(const GemmFp8& g, int sms, int* status, cudaStream_t stream);

}  // namespace cx
