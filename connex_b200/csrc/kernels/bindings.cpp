// pybind11 bindings of the connex_b200._C extension (sm_100a kernels plus
// CUDA IPC plumbing for peer buffers).  Every op launches on the current
// torch stream of the tensor's device and never allocates device memory
// itself: outputs and workspaces come from the caller.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <string>
#include <vector>

#include "comm.h"
#include "gemm.h"
#include "gemm_fp8.h"
#include "kv_fp8.h"
#include "kv_int4.h"
#include "layers.h"
#include "moe.h"

namespace {

#define CHECK_CUDA(x) TORCH_CHECK((x).is_cuda(), #x " must be a CUDA tensor")
#define CHECK_BF16(x) TORCH_CHECK((x).scalar_type() == at::kBFloat16, #x " must be bf16")

cudaStream_t cur_stream(const at::Tensor& t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// A number of a message.  (Not left to the message's stream: this library may carry a C++ runtime of
// its own beside the one torch uses, and writing a number to a stream of the other ends the process.)
std::string num(int64_t x) { return std::to_string(x); }

int* status_ptr(const c10::optional<at::Tensor>& st) {
  if (!st.has_value()) return nullptr;
  TORCH_CHECK(st->scalar_type() == at::kInt && st->is_cuda(), "status must be an int32 CUDA tensor");
  return st->data_ptr<int>();
}

int row_ld(const at::Tensor& t) {
  TORCH_CHECK(t.dim() == 2, "expected a 2-D tensor");
  TORCH_CHECK(t.stride(1) == 1, "rows must be contiguous");
  return (int)t.stride(0);
}

// D = A . B^T (+ R) | SiLU-mul epilogue.  A [M,K], B [N,K], D [M,N or N/2].
void gemm(const at::Tensor& A, const at::Tensor& B, at::Tensor& D, const c10::optional<at::Tensor>& R, int64_t epi,
          int64_t bn, const c10::optional<at::Tensor>& status, int64_t max_ctas,
          const c10::optional<at::Tensor>& workspace, int64_t splits) {
  CHECK_CUDA(A);
  CHECK_CUDA(B);
  CHECK_CUDA(D);
  CHECK_BF16(A);
  CHECK_BF16(B);
  CHECK_BF16(D);
  const c10::cuda::CUDAGuard g(A.device());
  const int M = (int)A.size(0), K = (int)A.size(1), N = (int)B.size(0);
  TORCH_CHECK(B.size(1) == K, "gemm: K mismatch");
  if (epi == cx::EPI_SILU_MUL) {
    TORCH_CHECK(D.size(0) == M && D.size(1) == N / 2, "gemm: SiLU-mul output must be [M, N/2]");
  } else {
    TORCH_CHECK(D.size(0) == M && D.size(1) == N, "gemm: output shape mismatch");
  }
  const void* rp = nullptr;
  int ldr = 0;
  if (epi == cx::EPI_ADD) {
    TORCH_CHECK(R.has_value(), "gemm: residual epilogue needs R");
    CHECK_BF16((*R));
    rp = R->data_ptr();
    ldr = row_ld(*R);
  }
  if (M == 0) return;
  float* W = nullptr;
  if (splits > 1) {
    TORCH_CHECK(workspace.has_value() && workspace->is_cuda() && workspace->scalar_type() == at::kFloat &&
                    workspace->is_contiguous() && workspace->numel() >= (int64_t)M * N,
                "gemm: split-K needs a contiguous fp32 CUDA workspace of at least M*N elements (kept zero)");
    W = workspace->data_ptr<float>();
  }
  cx::gemm_bf16_tn(A.data_ptr(), B.data_ptr(), D.data_ptr(), rp, M, N, K, row_ld(A), row_ld(B), row_ld(D), ldr,
                   (int)epi, (int)bn, status_ptr(status), (int)max_ctas, cur_stream(A), W, (int)splits);
}

int64_t gemm_splits(int64_t M, int64_t N, int64_t K, int64_t epi, int64_t bn) {
  return cx::gemm_splits((int)M, (int)N, (int)K, (int)epi, (int)bn);
}

void rmsnorm(const at::Tensor& x, const c10::optional<at::Tensor>& residual, const at::Tensor& w, at::Tensor& out,
             double eps) {
  CHECK_BF16(x);
  CHECK_BF16(w);
  CHECK_BF16(out);
  const c10::cuda::CUDAGuard g(x.device());
  void* rp = nullptr;
  int ldr = 0;
  if (residual.has_value()) {
    rp = residual->data_ptr();
    ldr = row_ld(*residual);
  }
  const int H = (int)x.size(1);
  TORCH_CHECK(H % 8 == 0, "rmsnorm: hidden size must be a multiple of 8");
  cx::rmsnorm(x.data_ptr(), row_ld(x), rp, ldr, w.data_ptr(), out.data_ptr(), row_ld(out), (int)x.size(0), H,
              (float)eps, cur_stream(x));
}

void rope_cache(at::Tensor& qkv, const at::Tensor& pos, const at::Tensor& cos_sin,
                const c10::optional<at::Tensor>& slots, const c10::optional<at::Tensor>& kc,
                const c10::optional<at::Tensor>& vc, int64_t Hq, int64_t Hkv, const c10::optional<at::Tensor>& status,
                const c10::optional<at::Tensor>& q_norm, const c10::optional<at::Tensor>& k_norm, double eps) {
  CHECK_BF16(qkv);
  if (slots.has_value()) {
    TORCH_CHECK(kc.has_value() && vc.has_value(), "rope_cache: caches required with a slot mapping");
    // the kernel addresses them by these sizes and stores two bytes per element
    TORCH_CHECK(kc->scalar_type() == at::kBFloat16 && vc->scalar_type() == at::kBFloat16 && kc->dim() == 4 &&
                    kc->size(1) == Hkv && kc->size(2) > 0 && kc->size(3) == 128 && kc->is_contiguous() &&
                    vc->is_contiguous() && vc->sizes() == kc->sizes(),
                "rope_cache: caches must be contiguous bf16 [blocks, Hkv, tokens, 128]; an 8-bit cache is written by "
                "rope_cache_fp8");
    TORCH_CHECK(kc->is_cuda() && vc->is_cuda(), "rope_cache: each cache must be a CUDA tensor");
  }
  const void* qn = nullptr;
  const void* kn = nullptr;
  for (const auto* w : {&q_norm, &k_norm})
    if (w->has_value())
      TORCH_CHECK((*w)->is_cuda() && (*w)->scalar_type() == at::kBFloat16 && (*w)->numel() == 128 &&
                      (*w)->is_contiguous(),
                  "rope_cache: q/k norm weights must be contiguous bf16 CUDA [128]");
  if (q_norm.has_value()) qn = q_norm->data_ptr();
  if (k_norm.has_value()) kn = k_norm->data_ptr();
  TORCH_CHECK(pos.scalar_type() == at::kInt, "positions must be int32");
  TORCH_CHECK(cos_sin.scalar_type() == at::kFloat, "cos_sin must be fp32");
  const c10::cuda::CUDAGuard g(qkv.device());
  const int64_t* sp = nullptr;
  void *kp = nullptr, *vp = nullptr;
  int BS = 16, nb = 0;
  if (slots.has_value()) {
    TORCH_CHECK(slots->scalar_type() == at::kLong, "slot_mapping must be int64");
    sp = slots->data_ptr<int64_t>();
    kp = kc->data_ptr();
    vp = vc->data_ptr();
    nb = (int)kc->size(0);
    BS = (int)kc->size(2);
  }
  cx::rope_cache(qkv.data_ptr(), row_ld(qkv), pos.data_ptr<int>(), cos_sin.data_ptr<float>(), sp, kp, vp,
                 (int)qkv.size(0), (int)Hq, (int)Hkv, 128, BS, nb, (int)cos_sin.size(0), status_ptr(status),
                 cur_stream(qkv), qn, kn, (float)eps);
}

void embedding(const at::Tensor& ids, const at::Tensor& table, at::Tensor& out,
               const c10::optional<at::Tensor>& status) {
  TORCH_CHECK(ids.scalar_type() == at::kInt, "ids must be int32");
  const c10::cuda::CUDAGuard g(table.device());
  cx::embedding(ids.data_ptr<int>(), table.data_ptr(), out.data_ptr(), (int)ids.numel(), (int)table.size(1),
                (int)table.size(0), status_ptr(status), cur_stream(table));
}

void argmax(const at::Tensor& logits, at::Tensor& out) {
  CHECK_BF16(logits);
  TORCH_CHECK(out.scalar_type() == at::kInt, "argmax output must be int32");
  const c10::cuda::CUDAGuard g(logits.device());
  cx::argmax(logits.data_ptr(), row_ld(logits), (int)logits.size(0), (int)logits.size(1), out.data_ptr<int>(),
             cur_stream(logits));
}

void gather_rows(const at::Tensor& src, const at::Tensor& idx, at::Tensor& out) {
  const c10::cuda::CUDAGuard g(src.device());
  cx::gather_rows(src.data_ptr(), row_ld(src), idx.data_ptr<int>(), out.data_ptr(), row_ld(out), (int)idx.numel(),
                  (int)src.size(1), cur_stream(src));
}

void prefill_attention_tc(const at::Tensor& qkv, at::Tensor& out, const at::Tensor& tile_info, int64_t Hq,
                          int64_t Hkv, double scale, const c10::optional<at::Tensor>& status, int64_t tile_rows) {
  CHECK_BF16(qkv);
  CHECK_BF16(out);
  TORCH_CHECK(tile_rows == 128 || tile_rows == 256, "tile_rows must be 128 or 256");
  TORCH_CHECK(tile_info.scalar_type() == at::kInt && tile_info.dim() == 2 && tile_info.size(1) == 3,
              "tile_info must be int32 [n, 3]");
  TORCH_CHECK(qkv.size(1) == (Hq + 2 * Hkv) * 128, "qkv must hold exactly (Hq + 2 Hkv) heads of 128");
  const c10::cuda::CUDAGuard g(qkv.device());
  cx::prefill_attention_tc(qkv.data_ptr(), row_ld(qkv), (int)qkv.size(1), (int)qkv.size(0), out.data_ptr(),
                           row_ld(out), tile_info.data_ptr<int>(), (int)tile_info.size(0), (int)Hq, (int)Hkv,
                           (float)scale, status_ptr(status), cur_stream(qkv), (int)tile_rows);
}

void prefill_attention_paged(const at::Tensor& qkv, const at::Tensor& kc, const at::Tensor& vc,
                             const at::Tensor& block_tables, at::Tensor& out, const at::Tensor& tile_info, int64_t Hq,
                             int64_t Hkv, double scale, const c10::optional<at::Tensor>& status,
                             int64_t tile_rows) {
  TORCH_CHECK(tile_rows == 128 || tile_rows == 256, "tile_rows must be 128 or 256");
  CHECK_BF16(qkv);
  CHECK_BF16(kc);
  CHECK_BF16(vc);
  CHECK_BF16(out);
  TORCH_CHECK(tile_info.scalar_type() == at::kInt && tile_info.dim() == 2 && tile_info.size(1) == 5,
              "tile_info must be int32 [n, 5]");
  TORCH_CHECK(block_tables.scalar_type() == at::kInt && block_tables.dim() == 2 && block_tables.is_contiguous(),
              "block_tables must be contiguous int32 [B, max_blocks]");
  TORCH_CHECK(qkv.size(1) == (Hq + 2 * Hkv) * 128, "qkv must hold exactly (Hq + 2 Hkv) heads of 128");
  TORCH_CHECK(kc.dim() == 4 && kc.size(1) == Hkv && kc.size(2) == 16 && kc.size(3) == 128 && kc.is_contiguous() &&
                  vc.is_contiguous() && vc.sizes() == kc.sizes(),
              "caches must be contiguous [blocks, Hkv, 16, 128]");
  const c10::cuda::CUDAGuard g(qkv.device());
  cx::prefill_attention_paged_tc(qkv.data_ptr(), row_ld(qkv), (int)qkv.size(1), (int)qkv.size(0), kc.data_ptr(),
                                 vc.data_ptr(), kc.size(0) * Hkv * 16, block_tables.data_ptr<int>(),
                                 (int)block_tables.size(1), out.data_ptr(), row_ld(out), tile_info.data_ptr<int>(),
                                 (int)tile_info.size(0), (int)Hq, (int)Hkv, (float)scale, status_ptr(status),
                                 cur_stream(qkv), (int)tile_rows);
}

void decode_attention(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& block_tables,
                      const at::Tensor& ctx_lens, at::Tensor& out, int64_t Hq, int64_t max_ctx, double scale,
                      at::Tensor& workspace) {
  CHECK_BF16(q);
  CHECK_BF16(kc);
  CHECK_BF16(vc);
  TORCH_CHECK(block_tables.scalar_type() == at::kInt && ctx_lens.scalar_type() == at::kInt, "int32 tables");
  TORCH_CHECK(workspace.scalar_type() == at::kFloat, "workspace must be fp32");
  const c10::cuda::CUDAGuard g(q.device());
  const int B = (int)q.size(0);
  const int Hkv = (int)kc.size(1), BS = (int)kc.size(2);
  TORCH_CHECK(kc.dim() == 4 && kc.size(3) == 128 && kc.is_contiguous() && vc.is_contiguous() && vc.sizes() == kc.sizes(),
              "caches must be contiguous [blocks, Hkv, BS, 128]");
  const int splits = cx::decode_attention_splits((int)max_ctx);
  TORCH_CHECK(workspace.numel() >= (int64_t)B * Hq * splits * 130, "decode workspace too small");
  cx::decode_attention(q.data_ptr(), row_ld(q), kc.data_ptr(), vc.data_ptr(), block_tables.data_ptr<int>(),
                       (int)block_tables.size(1), ctx_lens.data_ptr<int>(), out.data_ptr(), row_ld(out), B, (int)Hq,
                       Hkv, BS, (int)max_ctx, (float)scale, workspace.data_ptr<float>(), cur_stream(q),
                       (long)workspace.numel(), nullptr, (long)kc.size(0));
}

int64_t decode_attention_plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t max_ctx, int64_t ws_floats) {
  return cx::decode_attention_plan((int)B, (int)Hq, (int)Hkv, (int)max_ctx, (long)ws_floats);
}

int64_t decode_workspace_floats(int64_t B, int64_t Hq, int64_t max_ctx) {
  return B * Hq * cx::decode_attention_splits((int)max_ctx) * 130;
}

// ---- 8-bit paged KV cache ----------------------------------------------------
int sms_of(const at::Tensor& t) { return at::cuda::getDeviceProperties(t.get_device())->multiProcessorCount; }

void check_same_device(const at::Tensor& a, std::initializer_list<const at::Tensor*> others, const char* what) {
  for (const auto* t : others)
    TORCH_CHECK(t->device() == a.device(), what, ": every tensor must be on ", a.device());
}

void check_status_device(const at::Tensor& a, const c10::optional<at::Tensor>& status, const char* what) {
  if (status.has_value()) check_same_device(a, {&*status}, what);
}

// rows of 16-byte vectors: [rows, cols] bf16 with contiguous rows
int row_ld16(const at::Tensor& t, const char* what) {
  TORCH_CHECK(t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1) && t.scalar_type() == at::kBFloat16, what,
              " must be bf16 [rows, columns] with contiguous rows");
  const int64_t ld = t.size(0) > 1 ? t.stride(0) : t.size(1);
  TORCH_CHECK(ld >= t.size(1) && ld % 8 == 0 && ld <= INT_MAX && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0,
              what, ": rows must start on 16-byte boundaries and not overlap");
  return (int)ld;
}

cx::KvFp8 fp8_cache(const at::Tensor& k, const at::Tensor& v, const at::Tensor& ks, const at::Tensor& vs,
                    const char* what) {
  check_same_device(k, {&v, &ks, &vs}, what);
  TORCH_CHECK(k.dim() == 4 && k.size(2) == 16 && k.size(3) == 128 && k.size(1) > 0 && k.is_contiguous() &&
                  v.is_contiguous() && v.sizes() == k.sizes() && k.scalar_type() == at::kFloat8_e4m3fn &&
                  v.scalar_type() == at::kFloat8_e4m3fn,
              what, ": caches must be contiguous float8_e4m3fn [blocks, Hkv, 16, 128]");
  for (const auto* t : {&ks, &vs})
    TORCH_CHECK(t->scalar_type() == at::kFloat && t->is_contiguous() && t->dim() == 2 && t->size(0) == k.size(0) &&
                    t->size(1) == k.size(1),
                what, ": scales must be contiguous fp32 [blocks, Hkv]");
  TORCH_CHECK(k.size(0) <= INT_MAX && ((reinterpret_cast<uintptr_t>(k.data_ptr()) |
                                        reinterpret_cast<uintptr_t>(v.data_ptr())) & 15) == 0,
              what, ": caches must start on a 16-byte boundary");
  return cx::KvFp8{static_cast<uint8_t*>(k.data_ptr()), static_cast<uint8_t*>(v.data_ptr()), ks.data_ptr<float>(),
                   vs.data_ptr<float>(), (int)k.size(0), (int)k.size(1)};
}

// What the quantising writes ask of their rows.
struct RopeRows {
  int ldq, ldo, max_pos;
  const void *qn, *kn;
};
RopeRows rope_rows(const std::string& what, const at::Tensor& qkv, const at::Tensor& pos, const at::Tensor& cos_sin,
                   const at::Tensor& slots, const at::Tensor& kc, const at::Tensor& out, int64_t Hq, int64_t Hkv,
                   const c10::optional<at::Tensor>& q_norm, const c10::optional<at::Tensor>& k_norm) {
  RopeRows r{};
  r.ldq = row_ld16(qkv, (what + ": qkv").c_str());
  r.ldo = row_ld16(out, (what + ": out").c_str());
  const int64_t T = qkv.size(0);
  TORCH_CHECK(Hq > 0 && Hkv == kc.size(1) && qkv.size(1) == (Hq + 2 * Hkv) * 128,
              what, ": qkv must hold exactly (Hq + 2 Hkv) heads of 128, Hkv as in the cache");
  TORCH_CHECK(out.size(0) == T && out.size(1) == Hq * 128, what, ": out must be [T, Hq * 128]");
  TORCH_CHECK(T <= INT_MAX, what, ": too many rows");
  TORCH_CHECK(pos.scalar_type() == at::kInt && pos.is_contiguous() && pos.numel() == T,
              what, ": positions must be contiguous int32 [T]");
  TORCH_CHECK(slots.scalar_type() == at::kLong && slots.is_contiguous() && slots.numel() == T,
              what, ": slot_mapping must be contiguous int64 [T]");
  TORCH_CHECK(cos_sin.scalar_type() == at::kFloat && cos_sin.dim() == 2 && cos_sin.size(1) == 128 &&
                  cos_sin.is_contiguous() && (reinterpret_cast<uintptr_t>(cos_sin.data_ptr()) & 15) == 0,
              what, ": cos_sin must be contiguous fp32 [positions, 128]");
  for (const auto* w : {&q_norm, &k_norm})
    if (w->has_value())
      TORCH_CHECK((*w)->device() == qkv.device() && (*w)->scalar_type() == at::kBFloat16 && (*w)->numel() == 128 &&
                      (*w)->is_contiguous() && (reinterpret_cast<uintptr_t>((*w)->data_ptr()) & 15) == 0,
                  what, ": q/k norm weights must be contiguous bf16 CUDA [128]");
  if (q_norm.has_value()) r.qn = q_norm->data_ptr();
  if (k_norm.has_value()) r.kn = k_norm->data_ptr();
  // q is rotated by the block that reads it: out may be qkv's own q columns, but no other part of it
  if (T > 0) {
    const char* a = static_cast<const char*>(qkv.data_ptr());
    const char* b = static_cast<const char*>(out.data_ptr());
    const char* a1 = a + ((T - 1) * (int64_t)r.ldq + qkv.size(1)) * 2;
    const char* b1 = b + ((T - 1) * (int64_t)r.ldo + out.size(1)) * 2;
    TORCH_CHECK(b1 <= a || a1 <= b || (a == b && (r.ldq == r.ldo || T == 1)),
                what, ": out overlaps qkv other than as its q columns");
  }
  r.max_pos = (int)std::min<int64_t>(cos_sin.size(0), INT_MAX);
  return r;
}

void rope_cache_fp8(const at::Tensor& qkv, const at::Tensor& pos, const at::Tensor& cos_sin, const at::Tensor& slots,
                    const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks, const at::Tensor& vs,
                    at::Tensor& out, int64_t Hq, int64_t Hkv, const c10::optional<at::Tensor>& status,
                    const c10::optional<at::Tensor>& q_norm, const c10::optional<at::Tensor>& k_norm, double eps) {
  const char* what = "rope_cache_fp8";
  check_same_device(qkv, {&pos, &cos_sin, &slots, &kc, &out}, what);
  check_status_device(qkv, status, what);
  const cx::KvFp8 c = fp8_cache(kc, vc, ks, vs, what);
  const RopeRows r = rope_rows(what, qkv, pos, cos_sin, slots, kc, out, Hq, Hkv, q_norm, k_norm);
  CHECK_CUDA(qkv);
  const c10::cuda::CUDAGuard g(qkv.device());
  cx::rope_cache_fp8(qkv.data_ptr(), r.ldq, pos.data_ptr<int>(), cos_sin.data_ptr<float>(), slots.data_ptr<int64_t>(), c,
                     out.data_ptr(), r.ldo, (int)qkv.size(0), (int)Hq, r.max_pos, sms_of(qkv), status_ptr(status),
                     cur_stream(qkv), r.qn, r.kn, (float)eps);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// What decode attention over a quantised cache asks of its arguments, the workspace apart.
void check_decode(const char* what, const at::Tensor& q, const at::Tensor& block_tables, const at::Tensor& ctx_lens,
                  const at::Tensor& out, int64_t Hq, int64_t Hkv, int64_t max_batch) {
  const int64_t B = q.size(0);
  TORCH_CHECK(Hq > 0 && Hq % Hkv == 0 && Hq / Hkv <= 16, what,
              ": the query heads must be a multiple of the KV heads, 16 of them per KV head at most");
  TORCH_CHECK(q.size(1) >= Hq * 128 && out.size(0) == B && out.size(1) == Hq * 128, what,
              ": q must hold Hq heads of 128 per row and out be [B, Hq * 128]");
  TORCH_CHECK(B <= max_batch, what, ": at most ", num(max_batch), " sequences per call");
  TORCH_CHECK(block_tables.scalar_type() == at::kInt && block_tables.dim() == 2 && block_tables.is_contiguous() &&
                  block_tables.size(0) == B,
              what, ": block_tables must be contiguous int32 [B, max_blocks]");
  TORCH_CHECK(ctx_lens.scalar_type() == at::kInt && ctx_lens.is_contiguous() && ctx_lens.numel() == B, what,
              ": ctx_lens must be contiguous int32 [B]");
  TORCH_CHECK(B * Hkv * (block_tables.size(1) + 16) < (int64_t)1 << 30 && block_tables.size(1) < (int64_t)1 << 26, what,
              ": block tables too large");
}

int64_t decode_fp8_rows(int64_t device, int64_t B, int64_t Hkv, int64_t G) {
  TORCH_CHECK(B >= 0 && Hkv > 0 && G > 0, "decode_workspace_fp8: bad sizes");
  return cx::decode_fp8_rows(at::cuda::getDeviceProperties(device)->multiProcessorCount, (int)B, (int)Hkv, (int)G);
}

void decode_attention_fp8(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks,
                          const at::Tensor& vs, const at::Tensor& block_tables, const at::Tensor& ctx_lens,
                          at::Tensor& out, int64_t Hq, double scale, at::Tensor& ws,
                          const c10::optional<at::Tensor>& status) {
  const char* what = "decode_attention_fp8";
  check_same_device(q, {&kc, &block_tables, &ctx_lens, &out, &ws}, what);
  check_status_device(q, status, what);
  const cx::KvFp8 c = fp8_cache(kc, vc, ks, vs, what);
  const int ldq = row_ld16(q, "decode_attention_fp8: q"), ldo = row_ld16(out, "decode_attention_fp8: out");
  check_decode(what, q, block_tables, ctx_lens, out, Hq, c.Hkv, cx::DEC8_MAX_BATCH);
  CHECK_CUDA(q);
  const int64_t B = q.size(0), G = Hq / c.Hkv;
  TORCH_CHECK(ws.scalar_type() == at::kFloat && ws.is_contiguous() && ws.dim() == 2 && ws.size(1) == G * cx::DEC8_ROW &&
                  ws.size(0) >= cx::decode_fp8_rows(sms_of(q), (int)B, c.Hkv, (int)G),
              what, ": the workspace must come from decode_workspace_fp8 for these heads and at least ", num(B),
              " sequences");
  const c10::cuda::CUDAGuard g(q.device());
  cx::decode_attention_fp8(q.data_ptr(), ldq, c, block_tables.data_ptr<int>(), (int)block_tables.size(1),
                           ctx_lens.data_ptr<int>(), out.data_ptr(), ldo, (int)B, (int)Hq, (float)scale,
                           ws.data_ptr<float>(), ws.size(0), sms_of(q), status_ptr(status), cur_stream(q));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

void kv_copy_blocks(at::Tensor& kv, const at::Tensor& pairs, const c10::optional<at::Tensor>& scales,
                    const c10::optional<at::Tensor>& status) {
  TORCH_CHECK(kv.dim() == 6 && kv.size(1) == 2 && kv.is_contiguous(),
              "kv_copy_blocks: kv must be contiguous [layers, 2, blocks, Hkv, tokens, head_dim]");
  check_same_device(kv, {&pairs}, "kv_copy_blocks");
  check_status_device(kv, status, "kv_copy_blocks");
  TORCH_CHECK(pairs.scalar_type() == at::kInt && pairs.dim() == 2 && pairs.size(1) == 2 && pairs.is_contiguous(),
              "kv_copy_blocks: pairs must be contiguous int32 [n, 2] (source, destination)");
  const int64_t n = pairs.size(0), block = kv.size(3) * kv.size(4) * kv.size(5) * kv.element_size();
  // (a block of no bytes is one of no vectors, and the kernel counts in whole ones)
  TORCH_CHECK(block > 0 && block % 16 == 0 && (reinterpret_cast<uintptr_t>(kv.data_ptr()) & 15) == 0,
              "kv_copy_blocks: blocks must be multiples of 16 bytes, not empty, on 16-byte boundaries");
  // pair i lies at the 32-bit words 2 i and 2 i + 1
  TORCH_CHECK(n <= INT_MAX / 2 && kv.size(0) * 2 <= 65535 && kv.size(2) <= INT_MAX &&
                  kv.size(0) * 2 * (block / 16) <= INT_MAX / 2,
              "kv_copy_blocks: too many blocks, or blocks too large");
  float* sp = nullptr;
  if (scales.has_value()) {
    check_same_device(kv, {&*scales}, "kv_copy_blocks");
    TORCH_CHECK(scales->scalar_type() == at::kFloat && scales->is_contiguous() && scales->dim() == 4 &&
                    scales->size(0) == kv.size(0) && scales->size(1) == 2 && scales->size(2) == kv.size(2) &&
                    scales->size(3) == kv.size(3),
                "kv_copy_blocks: scales must be contiguous fp32 [layers, 2, blocks, Hkv]");
    sp = scales->data_ptr<float>();
  } else {
    TORCH_CHECK(kv.scalar_type() != at::kFloat8_e4m3fn, "kv_copy_blocks: an 8-bit cache is copied with its scales");
  }
  CHECK_CUDA(kv);
  const c10::cuda::CUDAGuard g(kv.device());
  cx::kv_copy_blocks(kv.data_ptr(), sp, pairs.data_ptr<int>(), (int)n, (int)kv.size(0) * 2, (int)kv.size(2), block,
                     (int)kv.size(3), sms_of(kv), status_ptr(status), cur_stream(kv));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// log2 of the query heads that a prefill tile holds side by side: the power of two in the group, up to 128
int pack_log(int64_t group) {
  int p = 0;
  while (p < 7 && group > 0 && group % (2ll << p) == 0) ++p;
  return p;
}

// Workspace of prefill_attention_paged_fp8 besides the blocks: int32 words and fp32 words.
std::tuple<int64_t, int64_t> prefill_fp8_words(int64_t device, int64_t entries, int64_t n_tiles, int64_t group) {
  const int64_t ctas = at::cuda::getDeviceProperties(device)->multiProcessorCount, items = n_tiles << pack_log(group);
  return {2 * items + 2 * (ctas + 1) + 2 * ctas + entries + 5 * items, 2 * ctas * cx::AttnPlan::SLOT};
}

// Two launches: the tables' blocks as bf16 into workspaces of the caller, the
// paged prefill attention over them.  c: the quantised cache; what: the call's name.
template <class Cache>
void prefill_attention_quantised(const std::string& what, const at::Tensor& q, const Cache& c,
                                 const at::Tensor& block_tables, at::Tensor& out, const at::Tensor& tile_info, int64_t Hq,
                                 int64_t Hkv, double scale, at::Tensor& kv, const c10::optional<at::Tensor>& ints,
                                 const c10::optional<at::Tensor>& part, const c10::optional<at::Tensor>& status) {
  const int ldq = row_ld16(q, (what + ": q").c_str()), ldo = row_ld16(out, (what + ": out").c_str());
  const int64_t T = q.size(0);
  TORCH_CHECK(Hkv == c.Hkv && Hq > 0 && Hq % Hkv == 0,
              what, ": Hkv as in the cache, the query heads a multiple of it");
  // the kernel takes the row's largest score before it is scaled
  TORCH_CHECK(scale > 0 && std::isfinite(scale), what, ": the scale must be positive");
  TORCH_CHECK(q.size(1) >= Hq * 128 && out.size(0) == T && out.size(1) == Hq * 128,
              what, ": q must hold Hq heads of 128 per row and out be [T, Hq * 128]");
  TORCH_CHECK(tile_info.scalar_type() == at::kInt && tile_info.dim() == 2 && tile_info.size(1) == 5 &&
                  tile_info.is_contiguous() && (tile_info.size(0) + 1) * Hq <= INT_MAX / 5,
              what, ": tile_info must be contiguous int32 [n, 5]");
  TORCH_CHECK(block_tables.scalar_type() == at::kInt && block_tables.dim() == 2 && block_tables.is_contiguous() &&
                  block_tables.numel() <= INT_MAX && block_tables.size(1) < (int64_t)1 << 26 &&
                  block_tables.size(0) <= cx::KVQ_MAX_CHUNKS,
              what, ": block_tables must be contiguous int32 [B, max_blocks], B up to ",
              num(cx::KVQ_MAX_CHUNKS));
  TORCH_CHECK(kv.dim() == 5 && kv.size(0) == 2 && kv.size(2) == Hkv && kv.size(3) == 16 && kv.size(4) == 128 &&
                  kv.is_contiguous() && kv.scalar_type() == at::kBFloat16 && kv.size(1) * Hkv * 16 <= INT_MAX,
              what, ": the blocks' workspace must be contiguous bf16 [2, n_blocks, Hkv, 16, 128]");
  CHECK_CUDA(q);
  const int64_t entries = block_tables.numel(), n_tiles = tile_info.size(0);
  // The query heads of a KV head share a tile's rows where tokens alone would leave a quarter of them empty
  // (32/8 heads, 16 chunks at 4000: of 16 rows 141 us, 285 with tokens alone, of 128 rows 213 and 300; one
  // chunk at 30000: of 16 rows 107 and 147, of 192 137 and 158, of 256 160 and 157; one of 128 at 500 25 and 23).
  const int pack = T * 4 <= n_tiles * 256 * 3 ? pack_log(Hq / Hkv) : 0;
  const auto [n_ints, n_part] = prefill_fp8_words(q.device().index(), entries, n_tiles, Hq / Hkv);   // room for either
  TORCH_CHECK(ints.has_value() && ints->scalar_type() == at::kInt && ints->numel() == n_ints && ints->is_contiguous() &&
                  part.has_value() && part->scalar_type() == at::kFloat && part->numel() == n_part && part->is_contiguous(),
              what, ": workspaces of other sizes");
  check_same_device(q, {&*ints, &*part}, what.c_str());
  const c10::cuda::CUDAGuard g(q.device());
  TORCH_CHECK(T == 0 || n_tiles == 0 || (entries > 0 && kv.size(1) > 0),
              what, ": no block table for the tiles");
  if (T == 0 || n_tiles == 0) return;
  cx::KvChunks o;
  o.k = kv.data_ptr();
  o.v = static_cast<char*>(kv.data_ptr()) + kv.nbytes() / 2;
  o.pack = pack;
  // else they run side by side, so that the keys come from L2 for all but one (2 x 256 rows at 32256: 263 us,
  // 272 one by one); four at most, or the last team leaves SMs without work (8 query heads of one KV head,
  // 2048 rows at 6144: 71 us, 79 with eight)
  o.team = 1;
  for (int t = 2; pack == 0 && t <= 4; ++t)
    if (Hq / Hkv % t == 0) o.team = t;
  o.blocks = (int)kv.size(1);
  const int sms = sms_of(q);
  o.n_cta = std::max(1, sms / o.team) * o.team;
  o.before = reinterpret_cast<int64_t*>(ints->data_ptr<int>());      // the 8-byte words first
  o.cuts = reinterpret_cast<int2*>(o.before + (n_tiles << pack));
  o.arrived = reinterpret_cast<int*>(o.cuts + sms + 1);
  o.tables = o.arrived + 2 * sms;
  o.tiles = o.tables + entries;
  cx::kv_dequant_blocks(c, block_tables.data_ptr<int>(), (int)block_tables.size(0), (int)block_tables.size(1),
                        tile_info.data_ptr<int>(), (int)n_tiles, (int)T, (int)Hq, o, status_ptr(status), cur_stream(q));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  const cx::AttnPlan plan{o.cuts, part->data_ptr<float>(), o.arrived, o.n_cta, o.pack, o.team};
  cx::prefill_attention_paged_tc(q.data_ptr(), ldq, (int)(Hq * 128), (int)T, o.k, o.v, kv.size(1) * Hkv * 16, o.tables,
                                 (int)block_tables.size(1), out.data_ptr(), ldo, o.tiles, (int)n_tiles, (int)Hq,
                                 (int)Hkv, (float)scale, status_ptr(status), cur_stream(q), 256, &plan);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

void prefill_attention_paged_fp8(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks,
                                 const at::Tensor& vs, const at::Tensor& block_tables, at::Tensor& out,
                                 const at::Tensor& tile_info, int64_t Hq, int64_t Hkv, double scale, at::Tensor& kv,
                                 const c10::optional<at::Tensor>& ints, const c10::optional<at::Tensor>& part,
                                 const c10::optional<at::Tensor>& status) {
  const char* what = "prefill_attention_paged_fp8";
  check_same_device(q, {&kc, &block_tables, &out, &tile_info, &kv}, what);
  check_status_device(q, status, what);
  prefill_attention_quantised(what, q, fp8_cache(kc, vc, ks, vs, what), block_tables, out, tile_info, Hq, Hkv, scale, kv,
                              ints, part, status);
}

// ---- 4-bit paged KV cache ----------------------------------------------------
cx::KvInt4 int4_cache(const at::Tensor& k, const at::Tensor& v, const char* what) {
  check_same_device(k, {&v}, what);
  TORCH_CHECK(k.dim() == 4 && k.size(2) == 16 && k.size(3) == cx::KV4_ROW && k.size(1) > 0 && k.is_contiguous() &&
                  v.is_contiguous() && v.sizes() == k.sizes() && k.scalar_type() == at::kByte && v.scalar_type() == at::kByte,
              what, ": caches must be contiguous uint8 [blocks, Hkv, 16, 72]");
  TORCH_CHECK(k.size(0) <= INT_MAX && k.size(1) <= INT_MAX && ((reinterpret_cast<uintptr_t>(k.data_ptr()) |
                                        reinterpret_cast<uintptr_t>(v.data_ptr())) & 15) == 0,
              what, ": caches must start on a 16-byte boundary");
  return cx::KvInt4{static_cast<uint8_t*>(k.data_ptr()), static_cast<uint8_t*>(v.data_ptr()), (int)k.size(0),
                    (int)k.size(1)};
}

void rope_cache_int4(const at::Tensor& qkv, const at::Tensor& pos, const at::Tensor& cos_sin, const at::Tensor& slots,
                     const at::Tensor& kc, const at::Tensor& vc, at::Tensor& out, int64_t Hq,
                     int64_t Hkv, const c10::optional<at::Tensor>& status, const c10::optional<at::Tensor>& q_norm,
                     const c10::optional<at::Tensor>& k_norm, double eps) {
  const char* what = "rope_cache_int4";
  check_same_device(qkv, {&pos, &cos_sin, &slots, &kc, &out}, what);
  check_status_device(qkv, status, what);
  const cx::KvInt4 c = int4_cache(kc, vc, what);
  const RopeRows r = rope_rows(what, qkv, pos, cos_sin, slots, kc, out, Hq, Hkv, q_norm, k_norm);
  CHECK_CUDA(qkv);
  const c10::cuda::CUDAGuard g(qkv.device());
  cx::rope_cache_int4(qkv.data_ptr(), r.ldq, pos.data_ptr<int>(), cos_sin.data_ptr<float>(), slots.data_ptr<int64_t>(), c,
                      out.data_ptr(), r.ldo, (int)qkv.size(0), (int)Hq, r.max_pos, status_ptr(status), cur_stream(qkv),
                      r.qn, r.kn, (float)eps);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

void kv_values_int4(const at::Tensor& cache, at::Tensor& out) {
  check_same_device(cache, {&out}, "kv_values_int4");
  TORCH_CHECK(cache.scalar_type() == at::kByte && cache.dim() >= 1 && cache.size(-1) == cx::KV4_ROW &&
                  cache.is_contiguous() && (reinterpret_cast<uintptr_t>(cache.data_ptr()) & 3) == 0,
              "kv_values_int4: the cache must be contiguous uint8 [..., 72]");
  auto shape = cache.sizes().vec();
  shape.back() = 128;
  TORCH_CHECK(out.scalar_type() == at::kBFloat16 && out.is_contiguous() && out.sizes() == at::IntArrayRef(shape) &&
                  (reinterpret_cast<uintptr_t>(out.data_ptr()) & 15) == 0,
              "kv_values_int4: out must be contiguous bf16 [..., 128]");
  CHECK_CUDA(cache);
  const c10::cuda::CUDAGuard g(cache.device());
  cx::kv_values_int4(cache.data_ptr(), out.data_ptr(), cache.numel() / cx::KV4_ROW, sms_of(cache), cur_stream(cache));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

int64_t decode_int4_rows(int64_t device, int64_t B, int64_t Hkv, int64_t G) {
  TORCH_CHECK(B >= 0 && Hkv > 0 && G > 0, "decode_workspace_int4: bad sizes");
  return cx::decode_int4_rows(at::cuda::getDeviceProperties(device)->multiProcessorCount, (int)B, (int)Hkv, (int)G);
}

void decode_attention_int4(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& vc,
                           const at::Tensor& block_tables, const at::Tensor& ctx_lens, at::Tensor& out, int64_t Hq,
                           double scale, at::Tensor& ws, const c10::optional<at::Tensor>& status, int64_t wait_ns) {
  const char* what = "decode_attention_int4";
  check_same_device(q, {&kc, &block_tables, &ctx_lens, &out, &ws}, what);
  check_status_device(q, status, what);
  const cx::KvInt4 c = int4_cache(kc, vc, what);
  const int ldq = row_ld16(q, "decode_attention_int4: q"), ldo = row_ld16(out, "decode_attention_int4: out");
  check_decode(what, q, block_tables, ctx_lens, out, Hq, c.Hkv, cx::DEC4_MAX_BATCH);
  CHECK_CUDA(q);
  const int64_t B = q.size(0), G = Hq / c.Hkv;
  TORCH_CHECK(ws.scalar_type() == at::kFloat && ws.is_contiguous() && ws.dim() == 2 && ws.size(1) == G * cx::DEC4_ROW &&
                  ws.size(0) >= cx::decode_int4_rows(sms_of(q), (int)B, c.Hkv, (int)G),
              what, ": the workspace must come from decode_workspace_int4 for these heads and at least ", num(B),
              " sequences");
  const c10::cuda::CUDAGuard g(q.device());
  cx::decode_attention_int4(q.data_ptr(), ldq, c, block_tables.data_ptr<int>(), (int)block_tables.size(1),
                            ctx_lens.data_ptr<int>(), out.data_ptr(), ldo, (int)B, (int)Hq, (float)scale,
                            ws.data_ptr<float>(), sms_of(q), status_ptr(status), wait_ns, cur_stream(q));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

void prefill_attention_paged_int4(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& vc,
                                  const at::Tensor& block_tables, at::Tensor& out, const at::Tensor& tile_info, int64_t Hq,
                                  int64_t Hkv, double scale, at::Tensor& kv, const c10::optional<at::Tensor>& ints,
                                  const c10::optional<at::Tensor>& part, const c10::optional<at::Tensor>& status) {
  const char* what = "prefill_attention_paged_int4";
  check_same_device(q, {&kc, &block_tables, &out, &tile_info, &kv}, what);
  check_status_device(q, status, what);
  prefill_attention_quantised(what, q, int4_cache(kc, vc, what), block_tables, out, tile_info, Hq, Hkv, scale, kv, ints,
                              part, status);
}

// ---- block-scaled fp8 ----------------------------------------------------------
// What a call writes shares no memory with what its other CTAs read.  (Views with gaps may lie between one another's
// rows, as two ranges of columns do: those are the caller's to keep apart.)
void check_apart(const at::Tensor& out, std::initializer_list<const at::Tensor*> others, const char* what) {
  auto bytes = [](const at::Tensor& t) { return t.numel() * (int64_t)t.element_size(); };
  if (out.numel() == 0 || !out.is_non_overlapping_and_dense()) return;
  const char* a = static_cast<const char*>(out.data_ptr());
  for (const auto* t : others) {
    if (t->numel() == 0 || !t->is_non_overlapping_and_dense()) continue;
    const char* b = static_cast<const char*>(t->data_ptr());
    TORCH_CHECK(a + bytes(out) <= b || b + bytes(*t) <= a, what, " overlaps another tensor of the call");
  }
}
// e4m3 rows that a TMA can read: [rows, cols], contiguous rows on 16-byte boundaries
int64_t fp8_ld(const at::Tensor& t, const char* what) {
  TORCH_CHECK(t.dim() == 2 && t.scalar_type() == at::kFloat8_e4m3fn && (t.size(1) <= 1 || t.stride(1) == 1), what,
              " must be float8_e4m3fn [rows, columns] with contiguous rows");
  const int64_t ld = t.size(0) > 1 ? t.stride(0) : t.size(1);
  TORCH_CHECK(t.size(1) % 16 == 0 && ld >= t.size(1) && ld % 16 == 0 &&
                  (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0 && t.size(0) <= INT_MAX / 2 &&
                  t.size(1) <= INT_MAX / 2 && ld < (int64_t)1 << 39,
              what, ": columns must be a multiple of 16 and rows start on 16-byte boundaries without overlap");
  return ld;
}
// fp32 scales of `rows` rows (or blocks of them) and ceil(cols / 128) column blocks, any strides
cx::Fp8Scales fp8_scales(const at::Tensor& s, int64_t rows, int64_t cols, const char* what) {
  TORCH_CHECK(s.scalar_type() == at::kFloat && s.dim() == 2 && s.size(0) == rows && s.size(1) == (cols + 127) / 128, what,
              " must be fp32 [", num(rows), ", ", num((cols + 127) / 128), "]");
  return cx::Fp8Scales{s.data_ptr<float>(), s.stride(0), s.stride(1)};
}
// scales that a call writes: no two of them in one place
cx::Fp8Scales fp8_scales_out(const at::Tensor& s, int64_t rows, int64_t cols, const char* what) {
  const cx::Fp8Scales r = fp8_scales(s, rows, cols, what);
  const int64_t kb = s.size(1);
  TORCH_CHECK((rows <= 1 || r.row > 0) && (kb <= 1 || r.col > 0) &&
                  (rows <= 1 || kb <= 1 || r.row >= kb * r.col || r.col >= rows * r.row),
              what, " must not overlap itself");
  return r;
}

void quantize_fp8(const at::Tensor& x, const c10::optional<at::Tensor>& norm, double eps, at::Tensor& q,
                  at::Tensor& scale) {
  check_same_device(x, {&q, &scale}, "quantize_fp8");
  const int ldx = row_ld16(x, "quantize_fp8: x");
  const int64_t T = x.size(0), K = x.size(1), ldq = fp8_ld(q, "quantize_fp8: out");
  TORCH_CHECK(q.size(0) == T && q.size(1) == K, "quantize_fp8: out must have x's shape");
  const cx::Fp8Scales s = fp8_scales_out(scale, T, K, "quantize_fp8: scale");
  check_apart(q, {&x, &scale}, "quantize_fp8: out");
  check_apart(scale, {&x}, "quantize_fp8: scale");
  const void* w = nullptr;
  if (norm.has_value()) {
    check_same_device(x, {&*norm}, "quantize_fp8");
    TORCH_CHECK(norm->scalar_type() == at::kBFloat16 && norm->dim() == 1 && norm->numel() == K && norm->is_contiguous() &&
                    (reinterpret_cast<uintptr_t>(norm->data_ptr()) & 15) == 0,
                "quantize_fp8: norm must be contiguous bf16 [columns of x]");
    TORCH_CHECK(K <= cx::QUANT_NORM_MAX_K, "quantize_fp8: at most ", num(cx::QUANT_NORM_MAX_K), " columns with a norm");
    w = norm->data_ptr();
  }
  CHECK_CUDA(x);
  const c10::cuda::CUDAGuard g(x.device());
  cx::quantize_fp8(x.data_ptr(), ldx, w, (float)eps, q.data_ptr(), ldq, s, (int)T, (int)K, cur_stream(x));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

void quantize_weight_fp8(const at::Tensor& w, at::Tensor& q, at::Tensor& scale) {
  check_same_device(w, {&q, &scale}, "quantize_weight_fp8");
  const int ldw = row_ld16(w, "quantize_weight_fp8: w");
  const int64_t N = w.size(0), K = w.size(1), ldq = fp8_ld(q, "quantize_weight_fp8: out");
  TORCH_CHECK(q.size(0) == N && q.size(1) == K, "quantize_weight_fp8: out must have w's shape");
  const cx::Fp8Scales s = fp8_scales_out(scale, (N + 127) / 128, K, "quantize_weight_fp8: scale");
  check_apart(q, {&w, &scale}, "quantize_weight_fp8: out");
  check_apart(scale, {&w}, "quantize_weight_fp8: scale");
  TORCH_CHECK((N + 127) / 128 <= 65535, "quantize_weight_fp8: too many rows");
  CHECK_CUDA(w);
  const c10::cuda::CUDAGuard g(w.device());
  cx::quantize_weight_fp8(w.data_ptr(), ldw, q.data_ptr(), ldq, s, (int)N, (int)K, cur_stream(w));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// out: bf16, or e4m3 with out_scale (SiLU-mul alone)
void gemm_fp8(const at::Tensor& a, const at::Tensor& sa, const at::Tensor& b, const at::Tensor& sb, at::Tensor& out,
              const c10::optional<at::Tensor>& out_scale, const c10::optional<at::Tensor>& residual, int64_t epi,
              const c10::optional<at::Tensor>& status, int64_t wait_ns) {
  check_same_device(a, {&sa, &b, &sb, &out}, "gemm_fp8");
  check_status_device(a, status, "gemm_fp8");
  cx::GemmFp8 g{};
  g.lda = fp8_ld(a, "gemm_fp8: a");
  g.ldb = fp8_ld(b, "gemm_fp8: b");
  const int64_t M = a.size(0), K = a.size(1), N = b.size(0);
  TORCH_CHECK(b.size(1) == K && K > 0, "gemm_fp8: a and b must have the same columns, not none");
  TORCH_CHECK(N % 8 == 0, "gemm_fp8: the rows of b must be a multiple of 8");
  g.sa = fp8_scales(sa, M, K, "gemm_fp8: a's scales");
  g.sb = fp8_scales(sb, (N + 127) / 128, K, "gemm_fp8: b's scales");
  const bool silu = epi == cx::EPI_SILU_MUL;
  TORCH_CHECK(epi == cx::EPI_STORE || epi == cx::EPI_ADD || silu, "gemm_fp8: unknown epilogue");
  TORCH_CHECK(!silu || N % 256 == 0, "gemm_fp8: SiLU-mul needs the rows of b to be a multiple of 256");
  const int64_t n_out = silu ? N / 2 : N;
  TORCH_CHECK(out.dim() == 2 && out.size(0) == M && out.size(1) == n_out, "gemm_fp8: out must be [", num(M), ", ",
              num(n_out), "]");
  if (out.numel() == 0) return;
  check_apart(out, {&a, &sa, &b, &sb}, "gemm_fp8: out");
  if (out_scale.has_value()) {
    check_apart(*out_scale, {&out, &a, &sa, &b, &sb}, "gemm_fp8: out's scales");
    TORCH_CHECK(silu, "gemm_fp8: only the SiLU-mul output is quantised");
    check_same_device(a, {&*out_scale}, "gemm_fp8");
    g.ldd = fp8_ld(out, "gemm_fp8: out");
    g.sd = fp8_scales_out(*out_scale, M, n_out, "gemm_fp8: out's scales");
  } else {
    g.ldd = row_ld16(out, "gemm_fp8: out");
  }
  TORCH_CHECK((epi == cx::EPI_ADD) == residual.has_value(), "gemm_fp8: the residual goes with its epilogue");
  if (residual.has_value()) {
    check_same_device(a, {&*residual}, "gemm_fp8");
    g.ldr = row_ld16(*residual, "gemm_fp8: residual");
    TORCH_CHECK(residual->sizes() == out.sizes(), "gemm_fp8: residual must have out's shape");
    // read and written element by element by one thread each: the same place or another, but not shifted
    const char *x0 = static_cast<const char*>(residual->data_ptr()), *y0 = static_cast<const char*>(out.data_ptr());
    const char *x1 = x0 + (M > 0 ? ((M - 1) * g.ldr + N) * 2 : 0), *y1 = y0 + (M > 0 ? ((M - 1) * g.ldd + N) * 2 : 0);
    TORCH_CHECK(x1 <= y0 || y1 <= x0 || (x0 == y0 && (g.ldr == g.ldd || M == 1)),
                "gemm_fp8: out overlaps the residual other than as itself");
    g.r = residual->data_ptr();
  }
  CHECK_CUDA(a);
  const c10::cuda::CUDAGuard guard(a.device());
  g.a = a.data_ptr();
  g.b = b.data_ptr();
  g.d = out.data_ptr();
  g.M = (int)M;
  g.N = (int)N;
  g.K = (int)K;
  g.epi = (int)epi;
  g.wait_ns = wait_ns < 0 ? cx::GEMM_FP8_WAIT_NS : (uint64_t)wait_ns;
  cx::gemm_fp8(g, sms_of(a), status_ptr(status), cur_stream(a));
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// ---- peer-memory movement (addresses may be local or peer-mapped) ----------
int64_t kv_push_layer(int64_t src_k, int64_t src_v, int64_t dst_k, int64_t dst_v, const at::Tensor& pairs,
                      int64_t src_heads, int64_t dst_heads, int64_t src_h0, int64_t dst_h0, int64_t n_heads,
                      int64_t chunk_bytes, int64_t src_blocks, int64_t dst_blocks, int64_t ready, int64_t max_ctas,
                      const c10::optional<at::Tensor>& status, int64_t span, int64_t threads) {
  TORCH_CHECK(pairs.scalar_type() == at::kInt && pairs.is_cuda(), "pairs must be int32 CUDA [n, 2]");
  const c10::cuda::CUDAGuard g(pairs.device());
  return cx::kv_push_layer(reinterpret_cast<const void*>(src_k), reinterpret_cast<const void*>(src_v),
                           reinterpret_cast<void*>(dst_k), reinterpret_cast<void*>(dst_v), pairs.data_ptr<int>(),
                           (int)pairs.size(0), (int)src_heads, (int)dst_heads, (int)src_h0, (int)dst_h0, (int)n_heads,
                           (int)chunk_bytes, (int)src_blocks, (int)dst_blocks, reinterpret_cast<uint32_t*>(ready),
                           (int)max_ctas, status_ptr(status), cur_stream(pairs), reinterpret_cast<uint64_t*>(span),
                           (int)threads);
}

int64_t copy_segments(const at::Tensor& segs, int64_t total_bytes, int64_t ready, int64_t max_ctas,
                      const c10::optional<at::Tensor>& status) {
  TORCH_CHECK(segs.scalar_type() == at::kLong && segs.is_cuda() && segs.dim() == 2 && segs.size(1) == 3,
              "segs must be int64 CUDA [n, 3]");
  const c10::cuda::CUDAGuard g(segs.device());
  return cx::copy_segments(segs.data_ptr<int64_t>(), (int)segs.size(0), total_bytes,
                           reinterpret_cast<uint32_t*>(ready), (int)max_ctas, status_ptr(status), cur_stream(segs));
}

// Weight sync: jobs int64 [n, WS_JOB_COLS] on the device and its host copy
// (validated here); destinations are a multicast address or up to
// WS_MAX_DST plain bases (with optional flag words).
int64_t wsync(const at::Tensor& jobs_dev, const at::Tensor& jobs_cpu, int64_t dst_bytes, std::vector<int64_t> bases,
              std::vector<int64_t> flags, int64_t mc_base, int64_t mc_flag, int64_t max_ctas, int64_t scatter_bytes) {
  TORCH_CHECK(jobs_dev.is_cuda() && jobs_dev.scalar_type() == at::kLong && jobs_dev.is_contiguous() &&
                  jobs_dev.dim() == 2 && jobs_dev.size(1) == cx::WS_JOB_COLS,
              "jobs_dev must be contiguous int64 CUDA [n, ", num(cx::WS_JOB_COLS), "]");
  TORCH_CHECK(!jobs_cpu.is_cuda() && jobs_cpu.scalar_type() == at::kLong && jobs_cpu.is_contiguous() &&
                  jobs_cpu.sizes() == jobs_dev.sizes(),
              "jobs_cpu must be the contiguous host copy of jobs_dev");
  TORCH_CHECK(flags.empty() || flags.size() == bases.size(), "one flag per destination (or none)");
  const c10::cuda::CUDAGuard g(jobs_dev.device());
  return cx::wsync(jobs_dev.data_ptr<int64_t>(), jobs_cpu.data_ptr<int64_t>(), (int)jobs_dev.size(0), dst_bytes,
                   reinterpret_cast<const uint64_t*>(bases.data()),
                   flags.empty() ? nullptr : reinterpret_cast<const uint64_t*>(flags.data()), (int)bases.size(),
                   (uint64_t)mc_base, (uint64_t)mc_flag, (int)max_ctas, scatter_bytes, cur_stream(jobs_dev));
}

void chan_copy(std::vector<int64_t> src, std::vector<int64_t> dst, std::vector<int64_t> bytes, int64_t wait_on,
               int64_t wait_target, int64_t timeout_ns, int64_t signal, int64_t value, int64_t mode, int64_t done_ctr,
               int64_t ctas, const at::Tensor& status, int64_t abort) {
  TORCH_CHECK(src.size() == dst.size() && dst.size() == bytes.size(), "chan_copy: segment lists differ in length");
  TORCH_CHECK(status.is_cuda() && status.scalar_type() == at::kInt, "chan_copy: status must be an int32 CUDA word");
  const c10::cuda::CUDAGuard g(status.device());
  cx::chan_copy(reinterpret_cast<const uint64_t*>(src.data()), reinterpret_cast<const uint64_t*>(dst.data()),
                reinterpret_cast<const uint64_t*>(bytes.data()), (int)src.size(),
                reinterpret_cast<const uint32_t*>(wait_on), (uint32_t)wait_target, (uint64_t)timeout_ns,
                reinterpret_cast<const uint32_t*>(abort), reinterpret_cast<uint32_t*>(signal), (uint32_t)value,
                (int)mode, reinterpret_cast<uint32_t*>(done_ctr), (int)ctas, status.data_ptr<int>(), cur_stream(status));
}

void wait_flag(int64_t flag, int64_t target, int64_t timeout_ns, const at::Tensor& status) {
  const c10::cuda::CUDAGuard g(status.device());
  cx::wait_flag(reinterpret_cast<const uint32_t*>(flag), (uint32_t)target, (uint64_t)timeout_ns,
                status.data_ptr<int>(), cur_stream(status));
}

void write_flag(int64_t flag, int64_t value, bool add, const at::Tensor& like) {
  const c10::cuda::CUDAGuard g(like.device());
  cx::write_flag(reinterpret_cast<uint32_t*>(flag), (uint32_t)value, add, cur_stream(like));
}

// ---- expert parallelism -------------------------------------------------------
// peers: int64 CUDA tensor [7, N] of addresses (counts, count_flag, recv,
// recv_meta, data_flag, comb, comb_flag) on every rank.
cx::EpPeers ep_peers(const at::Tensor& peers) {
  TORCH_CHECK(peers.scalar_type() == at::kLong && peers.is_cuda() && peers.dim() == 2 && peers.size(0) == 7,
              "peers must be int64 CUDA [7, N]");
  const uint64_t* p = reinterpret_cast<const uint64_t*>(peers.data_ptr<int64_t>());
  const int64_t N = peers.size(1);
  return cx::EpPeers{p, p + N, p + 2 * N, p + 3 * N, p + 4 * N, p + 5 * N, p + 6 * N};
}

void ep_count(const at::Tensor& topk_idx, const at::Tensor& l2p, const at::Tensor& l2p_cnt, int64_t S, int64_t me,
              at::Tensor& pos, at::Tensor& slot_of, const at::Tensor& peers, at::Tensor& comb_expect,
              int64_t arrivals_per_row, const c10::optional<at::Tensor>& status) {
  const c10::cuda::CUDAGuard g(topk_idx.device());
  TORCH_CHECK(topk_idx.scalar_type() == at::kInt && topk_idx.is_contiguous() && topk_idx.dim() == 2,
              "topk_idx must be contiguous int32 [T, K]");
  TORCH_CHECK(pos.numel() >= topk_idx.numel() && slot_of.numel() >= topk_idx.numel(),
              "ep_count: pos / slot_of hold fewer than T*K entries (more tokens than the layer's capacity)");
  TORCH_CHECK(l2p.scalar_type() == at::kInt && l2p.dim() == 2 && l2p_cnt.numel() == l2p.size(0),
              "l2p must be int32 [E, R] with l2p_cnt [E]");
  cx::ep_count(topk_idx.data_ptr<int>(), l2p.data_ptr<int>(), l2p_cnt.data_ptr<int>(), (int)l2p.size(1),
               (int)topk_idx.size(0), (int)topk_idx.size(1), (int)peers.size(1), (int)S, (int)me, pos.data_ptr<int>(),
               slot_of.data_ptr<int>(), ep_peers(peers), reinterpret_cast<uint32_t*>(comb_expect.data_ptr<int>()),
               (int)arrivals_per_row, status_ptr(status), cur_stream(topk_idx));
}

void ep_dispatch(const at::Tensor& x, const at::Tensor& topk_w, const at::Tensor& pos, const at::Tensor& slot_of,
                 const at::Tensor& counts_local, int64_t K, int64_t S, int64_t me, int64_t R_max, int64_t count_target,
                 const at::Tensor& peers, const c10::optional<at::Tensor>& status) {
  CHECK_BF16(x);
  const c10::cuda::CUDAGuard g(x.device());
  TORCH_CHECK(x.is_contiguous() && topk_w.is_contiguous() && topk_w.numel() == x.size(0) * K,
              "ep_dispatch: x [T, H] and topk_w [T, K] must be contiguous and agree");
  TORCH_CHECK(pos.numel() >= x.size(0) * K, "ep_dispatch: more tokens than the layer's capacity");
  cx::ep_dispatch(x.data_ptr(), topk_w.data_ptr<float>(), pos.data_ptr<int>(), slot_of.data_ptr<int>(),
                  counts_local.data_ptr<int>(), (int)x.size(0), (int)K, (int)x.size(1), (int)peers.size(1), (int)S,
                  (int)me, (int)R_max, (uint32_t)count_target, ep_peers(peers), status_ptr(status), cur_stream(x));
}

void ep_grouped_gemm(const at::Tensor& A, const at::Tensor& B, int64_t n_per_expert, at::Tensor& D,
                     const at::Tensor& counts_local, int64_t S, int64_t me, int64_t mode, const at::Tensor& recv_meta,
                     const at::Tensor& peers, int64_t H, int64_t wait_flag, int64_t wait_target,
                     const c10::optional<at::Tensor>& status) {
  CHECK_BF16(A);
  CHECK_BF16(B);
  const c10::cuda::CUDAGuard g(A.device());
  cx::ep_grouped_gemm(A.data_ptr(), row_ld(A), B.data_ptr(), (int)n_per_expert, (int)A.size(1), D.data_ptr(),
                      (int)D.stride(0), counts_local.data_ptr<int>(), (int)peers.size(1), (int)S, (int)me,
                      (int)A.size(0), (int)mode, recv_meta.data_ptr<int>(), ep_peers(peers), (int)H,
                      reinterpret_cast<const uint32_t*>(wait_flag), (uint32_t)wait_target, status_ptr(status),
                      cur_stream(A));
}

void ep_combine(const at::Tensor& comb, const at::Tensor& slot_of, int64_t T, int64_t K, at::Tensor& y,
                int64_t comb_flag, const at::Tensor& expect, const c10::optional<at::Tensor>& status) {
  const c10::cuda::CUDAGuard g(comb.device());
  TORCH_CHECK(comb.size(0) >= T * K && slot_of.numel() >= T * K && y.size(0) >= T && y.size(1) == comb.size(1),
              "ep_combine: buffers smaller than T*K rows");
  cx::ep_combine(comb.data_ptr(), slot_of.data_ptr<int>(), (int)T, (int)K, (int)y.size(1), y.data_ptr(),
                 reinterpret_cast<const uint32_t*>(comb_flag), reinterpret_cast<const uint32_t*>(expect.data_ptr<int>()),
                 status_ptr(status), cur_stream(comb));
}

// The whole EP layer in one call: count, dispatch, the two grouped GEMMs and
// combine, launched back to back on the current stream (one crossing from
// Python instead of five; the kernels' own waits order the phases across
// ranks).  Targets are the cumulative u32 counter values this forward waits for.
void ep_forward(const at::Tensor& x, const at::Tensor& topk_idx, const at::Tensor& topk_w, const at::Tensor& l2p,
                const at::Tensor& l2p_cnt, at::Tensor& out, const at::Tensor& w13, const at::Tensor& w2,
                at::Tensor& pos, at::Tensor& slot_of, const at::Tensor& counts, const at::Tensor& recv,
                const at::Tensor& recv_meta, at::Tensor& mid, const at::Tensor& comb, at::Tensor& comb_expect,
                const at::Tensor& peers, int64_t S, int64_t me, int64_t ffn, int64_t R_max, int64_t count_target,
                int64_t data_flag, int64_t data_target, int64_t comb_flag, const c10::optional<at::Tensor>& status,
                const std::vector<int64_t>& events) {
  const int64_t T = x.size(0), H = x.size(1), K = topk_idx.size(1);
  TORCH_CHECK(H % 256 == 0, "ep_forward: hidden size must be a multiple of 256");
  TORCH_CHECK(events.empty() || events.size() == 6, "ep_forward: events are 6 CUDA event handles or none");
  // optional per-phase timing: events[i] recorded before phase i (and after the last)
  const cudaStream_t st = cur_stream(x);
  auto mark = [&](int i) {
    if (!events.empty()) C10_CUDA_CHECK(cudaEventRecord(reinterpret_cast<cudaEvent_t>(events[i]), st));
  };
  mark(0);
  ep_count(topk_idx, l2p, l2p_cnt, S, me, pos, slot_of, peers, comb_expect, H / 256, status);
  mark(1);
  ep_dispatch(x, topk_w, pos, slot_of, counts, K, S, me, R_max, count_target, peers, status);
  mark(2);
  ep_grouped_gemm(recv, w13, 2 * ffn, mid, counts, S, me, 0, recv_meta, peers, H, data_flag, data_target, status);
  mark(3);
  ep_grouped_gemm(mid, w2, H, mid, counts, S, me, 1, recv_meta, peers, H, data_flag, data_target, status);
  mark(4);
  ep_combine(comb, slot_of, T, K, out, comb_flag, comb_expect, status);
  mark(5);
}

// ---- CUDA IPC ---------------------------------------------------------------
// Export the allocation that contains `ptr`: returns (handle bytes, offset of
// ptr inside the allocation).
std::pair<py::bytes, int64_t> ipc_export(int64_t ptr, int64_t device) {
  const c10::cuda::CUDAGuard g((c10::DeviceIndex)device);
  CUdeviceptr base = 0;
  size_t size = 0;
  using RangeFn = CUresult (*)(CUdeviceptr*, size_t*, CUdeviceptr);
  static RangeFn range = nullptr;
  if (range == nullptr) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    C10_CUDA_CHECK(cudaGetDriverEntryPoint("cuMemGetAddressRange", &p, cudaEnableDefault, &q));
    TORCH_CHECK(q == cudaDriverEntryPointSuccess && p, "cuMemGetAddressRange unavailable");
    range = reinterpret_cast<RangeFn>(p);
  }
  TORCH_CHECK(range(&base, &size, (CUdeviceptr)ptr) == CUDA_SUCCESS, "cuMemGetAddressRange failed");
  cudaIpcMemHandle_t h;
  C10_CUDA_CHECK(cudaIpcGetMemHandle(&h, reinterpret_cast<void*>(base)));
  return {py::bytes(reinterpret_cast<const char*>(&h), sizeof(h)), (int64_t)(ptr - (int64_t)base)};
}

int64_t ipc_open(const std::string& handle, int64_t device) {
  TORCH_CHECK(handle.size() == sizeof(cudaIpcMemHandle_t), "bad IPC handle size");
  const c10::cuda::CUDAGuard g((c10::DeviceIndex)device);
  cudaIpcMemHandle_t h;
  memcpy(&h, handle.data(), sizeof(h));
  void* p = nullptr;
  C10_CUDA_CHECK(cudaIpcOpenMemHandle(&p, h, cudaIpcMemLazyEnablePeerAccess));
  return reinterpret_cast<int64_t>(p);
}

void ipc_close(int64_t ptr, int64_t device) {
  const c10::cuda::CUDAGuard g((c10::DeviceIndex)device);
  C10_CUDA_CHECK(cudaIpcCloseMemHandle(reinterpret_cast<void*>(ptr)));
}

bool enable_peer_access(int64_t device, int64_t peer) {
  const c10::cuda::CUDAGuard g((c10::DeviceIndex)device);
  int can = 0;
  C10_CUDA_CHECK(cudaDeviceCanAccessPeer(&can, (int)device, (int)peer));
  if (!can) return false;
  cudaError_t e = cudaDeviceEnablePeerAccess((int)peer, 0);
  if (e == cudaErrorPeerAccessAlreadyEnabled) {
    (void)cudaGetLastError();
    return true;
  }
  C10_CUDA_CHECK(e);
  return true;
}

// Wrap a raw device address as a tensor view (no ownership).
at::Tensor from_ptr(int64_t ptr, std::vector<int64_t> shape, at::ScalarType dtype, int64_t device) {
  auto opts = at::TensorOptions().dtype(dtype).device(at::kCUDA, (c10::DeviceIndex)device);
  return torch::from_blob(reinterpret_cast<void*>(ptr), shape, opts);
}

}  // namespace


PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "connex_b200 sm_100a kernels";
  m.def("gemm", &gemm, py::arg("A"), py::arg("B"), py::arg("D"), py::arg("R") = py::none(), py::arg("epi") = 0,
        py::arg("bn") = 0, py::arg("status") = py::none(), py::arg("max_ctas") = 0,
        py::arg("workspace") = py::none(), py::arg("splits") = 1);
  m.def("rmsnorm", &rmsnorm);
  m.def("rope_cache", &rope_cache, py::arg("qkv"), py::arg("pos"), py::arg("cos_sin"), py::arg("slots"),
        py::arg("kc"), py::arg("vc"), py::arg("Hq"), py::arg("Hkv"), py::arg("status") = py::none(),
        py::arg("q_norm") = py::none(), py::arg("k_norm") = py::none(), py::arg("eps") = 1e-6);
  m.def("embedding", &embedding);
  m.def("argmax", &argmax);
  m.def("gather_rows", &gather_rows);
  m.def("prefill_attention", &prefill_attention_tc);
  m.def("prefill_attention_paged", &prefill_attention_paged);
  m.def("attention_exp_split", &cx::attention_exp_split);
  m.def("attention_profile", &cx::attention_profile);
  m.def("decode_attention", &decode_attention);
  m.def("decode_attention_plan", &decode_attention_plan);
  m.def("decode_workspace_floats", &decode_workspace_floats);
  m.def("rope_cache_fp8", &rope_cache_fp8);
  m.def("decode_fp8_rows", &decode_fp8_rows);
  m.attr("DECODE_FP8_ROW") = cx::DEC8_ROW;
  m.def("decode_fp8_resident", &cx::decode_fp8_resident);
  m.def("decode_attention_fp8", &decode_attention_fp8);
  m.def("kv_copy_blocks", &kv_copy_blocks);
  m.def("prefill_fp8_words", &prefill_fp8_words);
  m.def("prefill_attention_paged_fp8", &prefill_attention_paged_fp8);
  m.def("rope_cache_int4", &rope_cache_int4);
  m.def("kv_values_int4", &kv_values_int4);
  m.def("decode_int4_rows", &decode_int4_rows);
  m.attr("DECODE_INT4_ROW") = cx::DEC4_ROW;
  m.attr("KV_INT4_ROW") = cx::KV4_ROW;
  m.def("decode_attention_int4", &decode_attention_int4, py::arg("q"), py::arg("k_cache"), py::arg("v_cache"),
        py::arg("block_tables"), py::arg("ctx_lens"), py::arg("out"), py::arg("n_q_heads"), py::arg("scale"),
        py::arg("workspace"), py::arg("status"), py::arg("wait_ns") = -1);
  m.def("prefill_attention_paged_int4", &prefill_attention_paged_int4);
  m.def("quantize_fp8", &quantize_fp8);
  m.def("quantize_weight_fp8", &quantize_weight_fp8);
  m.def("gemm_fp8", &gemm_fp8, py::arg("a"), py::arg("a_scale"), py::arg("b"), py::arg("b_scale"), py::arg("out"),
        py::arg("out_scale"), py::arg("residual"), py::arg("epi"), py::arg("status"), py::arg("wait_ns") = -1);
  // (activations per tile or 0, CTAs per tile) of a call
  m.def("gemm_fp8_plan", [](int64_t M, int64_t N, int64_t K, int64_t epi, int64_t sms) {
    const cx::GemmFp8Plan p = cx::gemm_fp8_plan((int)M, (int)N, (int)K, (int)epi, (int)sms);
    return std::make_tuple(p.nt, p.splits);
  });
  m.def("kv_push_layer", &kv_push_layer);
  m.def("gemm_splits", &gemm_splits);
  m.def("gemm_raster_group", &cx::gemm_raster_group);
  m.def("copy_segments", &copy_segments);
  m.def("wsync", &wsync, py::arg("jobs_dev"), py::arg("jobs_cpu"), py::arg("dst_bytes"), py::arg("bases"),
        py::arg("flags"), py::arg("mc_base"), py::arg("mc_flag"), py::arg("max_ctas"), py::arg("scatter_bytes") = 0);
  m.attr("WS_JOB_COLS") = cx::WS_JOB_COLS;
  m.attr("WS_MAX_DST") = cx::WS_MAX_DST;
  m.def("chan_copy", &chan_copy, py::arg("src"), py::arg("dst"), py::arg("bytes"), py::arg("wait_on"),
        py::arg("wait_target"), py::arg("timeout_ns"), py::arg("signal"), py::arg("value"), py::arg("mode"),
        py::arg("done_ctr"), py::arg("ctas"), py::arg("status"), py::arg("abort") = 0);
  m.attr("CH_MAX_SEGS") = cx::CH_MAX_SEGS;
  m.def("wait_flag", &wait_flag);
  m.def("write_flag", &write_flag);
  m.def("ep_count", &ep_count);
  m.def("ep_dispatch", &ep_dispatch);
  m.def("ep_grouped_gemm", &ep_grouped_gemm);
  m.def("ep_combine", &ep_combine);
  m.def("ep_forward", &ep_forward);
  m.attr("EP_DISPATCH_CTAS") = cx::EP_DISPATCH_CTAS;
  m.def("ipc_export", &ipc_export);
  m.def("ipc_open", &ipc_open);
  m.def("ipc_close", &ipc_close);
  m.def("enable_peer_access", &enable_peer_access);
  m.def("from_ptr", &from_ptr);
  m.attr("EPI_STORE") = (int)cx::EPI_STORE;
  m.attr("EPI_ADD") = (int)cx::EPI_ADD;
  m.attr("EPI_SILU_MUL") = (int)cx::EPI_SILU_MUL;
}
