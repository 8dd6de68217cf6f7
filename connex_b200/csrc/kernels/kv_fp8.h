// Host entry points of the 8-bit paged KV cache kernels (kv_fp8.cu).
//
// A cache holds e4m3 values [blocks, Hkv, 16, 128] and one fp32 scale per
// (block, KV head) [blocks, Hkv], a power of two, for K and for V each: a
// cached element stands for value * scale.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace cx {

struct KvFp8 {
  uint8_t* k;
  uint8_t* v;
  float* ks;
  float* vs;
  int num_blocks, Hkv;
};

// Rows of the fused QKV buffer [T, (Hq + 2 Hkv) * 128] (ld ldq): q rotated
// into out [T, Hq * 128] (ld ldo; may be the q columns of qkv), k rotated and
// v quantised into the slots' blocks (slot < 0: not cached).
void rope_cache_fp8(const void* qkv, int ldq, const int* pos, const float* cos_sin, const int64_t* slots,
                    const KvFp8& c, void* out, int ldo, int T, int Hq, int max_pos, int sms, int* status, cudaStream_t s,
                    const void* q_norm, const void* k_norm, float eps);

// Rows of one call that are handled together; longer calls run as successive launches.
constexpr int KVQ_MAX_ROWS = 8192;

// One query row per sequence over its cached tokens.  ws: fp32
// [decode_fp8_rows(sms, B, Hkv, G), G * DEC8_ROW], zero before its first use
// (each call leaves its counters zero).
constexpr int DEC8_ROW = 132;        // floats of one head's partial result
constexpr int DEC8_MAX_BATCH = 4096;
int decode_fp8_ctas(int sms);                // of a call, at most
int decode_fp8_resident(int B, int G);       // that an SM holds at a time in a call of B sequences
long decode_fp8_rows(int sms, int B, int Hkv, int G);
void decode_attention_fp8(const void* q, int ldq, const KvFp8& c, const int* block_tables, int max_blocks,
                          const int* ctx_lens, void* out, int ldo, int B, int Hq, float scale, float* ws, long ws_rows,
                          int sms, int* status, cudaStream_t s);

// Blocks pairs[i] = (source, destination) of every plane [planes, num_blocks,
// block_bytes] and, where given, of the scales [planes, num_blocks, Hkv].
void kv_copy_blocks(void* kv, float* scales, const int* pairs, int n, int planes, int num_blocks, int64_t block_bytes,
                    int Hkv, int sms, int* status, cudaStream_t s);

constexpr int KVQ_MAX_CHUNKS = 8192;

// What kv_dequant_blocks leaves for the attention over its blocks.
struct KvChunks {
  void* k;          // bf16 [blocks, Hkv, 16, 128]
  void* v;
  int blocks;       // room for this many
  int* tables;      // [B, width]
  int* tiles;       // [n_tiles << pack, 5]: the tiles that fit, in their order, in 256 >> pack tokens each
  int2* cuts;       // [n_cta / team + 1], see AttnPlan
  int* arrived;     // [2 n_cta], zero
  int64_t* before;  // [n_tiles << pack] scratch
  int n_cta, pack, team;
};
// The e4m3 blocks that the tiles (tile_info [n_tiles, 5] of the paged prefill)
// read through tables [B, width] (B <= KVQ_MAX_CHUNKS), as bf16 blocks, those
// of one sequence behind those of another.  Tiles that do not fit T rows and
// the tables are left out; more blocks than there is room for are recorded.
void kv_dequant_blocks(const KvFp8& c, const int* tables, int B, int width, const int* tile_info, int n_tiles, int T,
                       int Hq, const KvChunks& o, int* status, cudaStream_t s);

}  // namespace cx
