// Host entry points of the 4-bit paged KV cache kernels (kv_int4.cu).
//
// A cache holds [blocks, Hkv, 16 tokens, 72 bytes].  A token's 72 bytes: 64 of
// 4-bit codes (dims 2i and 2i + 1 in the low and the high half of byte i), then
// bf16 scale and minimum of dims 0..63, and of dims 64..127.  A code stands for
// minimum + code * scale.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace cx {

constexpr int KV4_ROW = 72;

struct KvInt4 {
  uint8_t* k;
  uint8_t* v;
  int num_blocks, Hkv;
};

// Rows of the fused QKV buffer [T, (Hq + 2 Hkv) * 128] (ld ldq): q rotated into out [T, Hq * 128] (ld ldo; may be the
// q columns of qkv), k rotated and v quantised into the slots (slot < 0: not cached).
void rope_cache_int4(const void* qkv, int ldq, const int* pos, const float* cos_sin, const int64_t* slots,
                     const KvInt4& c, void* out, int ldo, int T, int Hq, int max_pos, int* status, cudaStream_t s,
                     const void* q_norm, const void* k_norm, float eps);

// cached rows [rows, 72] -> bf16 [rows, 128]
void kv_values_int4(const void* cache, void* out, int64_t rows, int sms, cudaStream_t s);

// One query row per sequence over its cached tokens.  ws: fp32 [decode_int4_rows(sms, B, Hkv, G), G * DEC4_ROW], zero
// before its first use; each call leaves its counters zero, one whose waits ran out among them.  wait_ns: the limit of
// a wait (0: every copy counts as lost), below 0 the default.  Rows of which a copy was lost read as NaN.
constexpr int DEC4_ROW = 136;        // floats of one head's partial result
constexpr int DEC4_MAX_BATCH = 4096;
long decode_int4_rows(int sms, int B, int Hkv, int G);
void decode_attention_int4(const void* q, int ldq, const KvInt4& c, const int* block_tables, int max_blocks,
                           const int* ctx_lens, void* out, int ldo, int B, int Hq, float scale, float* ws, int sms,
                           int* status, int64_t wait_ns, cudaStream_t s);

}  // namespace cx
