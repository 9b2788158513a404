// launch.hpp — host entry points of the kernel translation units.
//
// Each function validates nothing (plan.cpp already did) and enqueues on
// `s`.  Shapes: A[M,K] row-major, W[N,K] as 32-element blocks along K,
// C[M,N] row-major.
#pragma once

#include <hip/hip_runtime.h>

#include "plan.hpp"

namespace nfhip {

// Device workspace owned by the provider (allocated at init): fp32 partial
// tiles of split-K launches and one counter per output tile.  Counters start
// at zero and every split-K launch leaves them at zero again (the last
// workgroup of a tile resets its counter), so no per-launch clearing is
// needed.  Launches on the provider's single stream never overlap, so they
// share it.
struct Workspace {
  float* part = nullptr;
  uint32_t* cnt = nullptr;
  size_t part_floats = 0;
  uint32_t cnt_len = 0;
};

// Every block format; `in_bytes` (the input buffer size) bounds every read of `w`.
hipError_t launch_dequant(QFmt q, EType out_t, const void* w, uint64_t in_bytes, void* out, uint64_t count,
                          hipStream_t s);

hipError_t launch_gemv(QFmt q, EType t, const void* A, const void* W, void* C, uint32_t M,
                       uint32_t N, uint32_t K, hipStream_t s);

// Launch-floor calibration: stream `bytes` from `src` (read only, nothing
// stored), or an empty kernel when bytes < 16.
hipError_t launch_diag_read(const void* src, uint64_t bytes, hipStream_t s);

// Several decode GEMVs over the same activations A (same format, dtype, M
// and K; each with its own weights, output and N) in one launch, each job
// computed exactly as launch_gemv would.  hipErrorNotSupported when the
// jobs do not suit one launch (the caller then launches them one by one).
constexpr int kGemvGroupMax = 4;
struct GemvJob {
  const void* W;
  void* C;
  uint32_t N;
};
hipError_t launch_gemv_group(QFmt q, EType t, const void* A, const GemvJob* jobs, uint32_t n, uint32_t M,
                             uint32_t K, hipStream_t s);
hipError_t launch_skinny_group(QFmt q, EType t, const void* A, const GemvJob* jobs, uint32_t n, uint32_t M,
                               uint32_t K, const Workspace& ws, hipStream_t s);

// Small-batch MFMA kernels (f32 up to 64 rows a launch, f16 up to 128);
// skinny_fits() says whether a shape and operand alignment suit them,
// ring_serves() which shapes launch_skinny hands to the ring kernel.
bool ring_serves(QFmt q, EType t, uint32_t M, uint32_t N, uint32_t K);
hipError_t launch_skinny_ring(QFmt q, const void* A, const GemvJob* jobs, uint32_t n, uint32_t M, uint32_t K,
                              const Workspace& ws, hipStream_t s);
bool skinny_fits(uint32_t M, uint32_t N, uint32_t K, const void* A, const void* W);
uint32_t skinny_max_rows(EType t);  // activation rows per launch
hipError_t launch_skinny(QFmt q, EType t, const void* A, const void* W, void* C, uint32_t M, uint32_t N,
                         uint32_t K, const Workspace& ws, hipStream_t s);
// Several small-batch linears over the same activations (same
// format, dtype and K) in one launch, each computed exactly as launch_skinny
// would; hipErrorNotSupported when they would not get the same kernel
// variant and K split on their own (the caller launches them one by one).

// tile: Tuning::gemm_tile (-1 = register-dequantizing kernel, 0..6 = an
// LDS-staged tile shape).
hipError_t launch_gemm_mfma(QFmt q, EType t, const void* A, const void* W, void* C, uint32_t M,
                            uint32_t N, uint32_t K, int tile, const Workspace& ws, hipStream_t s);

hipError_t launch_generic(QFmt q, EType t, const void* A, const void* W, void* C, uint32_t M,
                          uint32_t N, uint32_t K, hipStream_t s);

// Dense fp16 x fp16 linear on the tiled MFMA kernel, fp16 or fp32 output;
// hipErrorInvalidValue when the shape/alignment does not fit it (K % 64,
// 16-B aligned operands).
hipError_t launch_dense_mfma_f16(const void* A, const void* B, void* C, uint32_t M, uint32_t N, uint32_t K,
                                 bool out_f32, hipStream_t s);

// Dense linear with at least one fp32 operand (fp16 operands widened
// exactly) on the fp32 MFMA; hipErrorNotSupported when K % 32 != 0 or an
// operand is not 16-B aligned.
hipError_t launch_dense_mfma_f32(EType a, EType b, EType c, const void* A, const void* B, void* C, uint32_t M,
                                 uint32_t N, uint32_t K, const Workspace& ws, hipStream_t s);

hipError_t launch_dense(EType a, EType b, EType c, const void* A, const void* B, void* C,
                        uint32_t M, uint32_t N, uint32_t K, const Workspace& ws, hipStream_t s);

// ---- layer ops (kernels/layer.hip) -------------------------------------------
hipError_t launch_binary(EwFn fn, EType t, const void* a, const void* b, void* out, uint64_t n, hipStream_t s);
hipError_t launch_unary(EwFn fn, EType t, const void* in, void* out, uint64_t n, hipStream_t s);
hipError_t launch_mock_prefill(const void* in, void* k, void* v, uint64_t nk, uint64_t nv, hipStream_t s);
hipError_t launch_rms_norm(EType t, const void* in, const void* w, void* out, uint32_t rows, uint32_t dim, float eps,
                           hipStream_t s);
// The residual addition and the norm after it: sum = a + b, out = rms_norm of
// sum; and silu with the product after it: act = silu(gate), out = act * up
// (up_first: up * act, which differs in the payload where both are NaN).
// The bits of the separate launches; hipErrorNotSupported for operands (odd
// alignment, row lengths) that need them.
hipError_t launch_add_rms_norm(EType t, const void* a, const void* b, void* sum, const void* w, void* out,
                               uint32_t rows, uint32_t dim, float eps, hipStream_t s);
hipError_t launch_silu_mul(EType t, const void* gate, const void* up, void* act, void* out, uint64_t n, bool up_first,
                           hipStream_t s);
// batch: rope_batch ([seq, n_heads, head_dim], pos = token + step); else rope
// (pos = step).  One or two jobs of n elements each in a launch.
struct RopeArgs {
  const void* in;
  void* out;
  uint64_t n;
  uint32_t n_heads;
};
hipError_t launch_rope(EType t, bool batch, const RopeArgs* jobs, uint32_t n_jobs, uint32_t head_dim, uint32_t step,
                       float theta, hipStream_t s);
// ws: the provider workspace (partials of rows split into chunks), may be null
hipError_t launch_softmax(const void* in, void* out, uint32_t rows, uint32_t dim, float* ws, size_t ws_floats,
                          hipStream_t s);
hipError_t launch_argmax(const void* in, void* out, uint32_t rows, uint32_t dim, float* ws, size_t ws_floats,
                         hipStream_t s);
// MoE (metal_provider.mm:1907-1997): per token, softmax over the first
// min(n_experts, 64) gate logits, the top_k (<= 8) largest in index order of
// ties, renormalized; and the weighted sum of the selected experts' rows.
hipError_t launch_moe_gate(const void* logits, void* ids, void* weights, uint32_t batch, uint32_t n_experts,
                           uint32_t top_k, hipStream_t s);
hipError_t launch_moe_scatter(const void* experts, uint32_t expert_rows, const void* ids, const void* weights,
                              void* out, uint32_t batch, uint32_t top_k, uint32_t dim, hipStream_t s);
hipError_t launch_embedding(EType t, const void* w, uint32_t vocab, const void* ids, void* out, uint64_t n,
                            uint32_t dim, uint32_t seq_len, hipStream_t s);

// ---- attention (kernels/attention.hip) ---------------------------------------
struct AttnArgs {
  const void* q = nullptr;
  const void* k_new = nullptr;  // Cached / Gqa: rows appended to the cache first
  const void* v_new = nullptr;
  void* k = nullptr;  // Plain: K; Cached / Gqa: cache_k; Paged: K pool
  void* v = nullptr;
  const uint32_t* block_table = nullptr;  // Paged
  void* out = nullptr;
  LayerParams lp;
  uint64_t pool_blocks = 0;  // Paged: whole blocks the pools hold
  float* ws = nullptr;       // decode partials (the provider's split-K workspace)
  size_t ws_floats = 0;
};
hipError_t launch_attention(EType t, const AttnArgs& a, hipStream_t s);

// ---- serving: a batch of sequences over a paged cache (kernels/paged*.hip) ----
struct PagedBatch {
  const uint32_t* table = nullptr;  // [n_seqs, width] physical blocks
  const int32_t* starts = nullptr;  // [n_seqs + 1] first row of each sequence
  const int32_t* lens = nullptr;    // [n_seqs] positions of each, its rows included
  uint32_t n_seqs = 0, width = 0, rows = 0, n_kv = 0, dim = 0, block_size = 0;
  uint32_t limit = 0;   // positions a sequence may hold
  uint32_t blocks = 0;  // whole blocks in the pools
};
hipError_t launch_paged_append(EType t, PoolType pool, const PagedBatch& b, const void* k, const void* v, void* k_pool,
                               void* v_pool, hipStream_t s);
hipError_t launch_paged_gather(EType t, PoolType pool, const PagedBatch& b, const void* k_pool, const void* v_pool,
                               void* k, void* v, hipStream_t s);
// Attention of the batch's rows; `ws` holds the partials of keys split over workgroups.
// lse: [rows, n_heads], or null.
hipError_t launch_paged_chunk(EType t, PoolType pool, const PagedBatch& b, uint32_t n_heads, const void* q,
                              const void* k_pool, const void* v_pool, void* out, float* lse, const Workspace& ws,
                              hipStream_t s);
// The same where the sequences first[g] .. first[g + 1] - 1 share their first len[g]
// positions, which lie where the table of the first of them says.
struct PagedShared {
  const int32_t* first = nullptr;  // [n_groups + 1]
  const int32_t* len = nullptr;    // [n_groups]
  uint32_t n_groups = 0;
};
hipError_t launch_paged_prefix(EType t, PoolType pool, const PagedBatch& b, const PagedShared& sh, uint32_t n_heads,
                               const void* q, const void* k_pool, const void* v_pool, void* out, float* lse,
                               const Workspace& ws, hipStream_t s);
// weights[s][kv head][position] (rows of `width`) = theta held + the sum of the rows'
// attention weights; theta 0 does not read `held`.
hipError_t launch_paged_weights(EType t, PoolType pool, const PagedBatch& b, uint32_t n_heads, const void* q,
                                const void* k_pool, const float* lse, const float* held, float* weights, uint32_t width,
                                float theta, const Workspace& ws, hipStream_t s);
// Eviction: of each sequence and KV head the budget[s][1] last positions and those of the
// largest weights, budget[s][0] together and at most `top`, in order of position; `kept`
// [n_seqs, n_kv, top] says which, and their rows go to the blocks of `to` [n_seqs, ceil(top
// / block_size)] in the second pools, of to_blocks blocks.  b.starts and b.rows are not used.
struct PagedEvict {
  const void* k = nullptr;
  const void* v = nullptr;
  const float* weights = nullptr;  // [n_seqs, n_kv, width]
  const int32_t* budget = nullptr; // [n_seqs, 2]
  const uint32_t* to = nullptr;
  void* k_to = nullptr;
  void* v_to = nullptr;
  float* weights_to = nullptr;
  int32_t* lens_to = nullptr;
  int32_t* kept = nullptr;
  uint32_t width = 0, top = 0, to_blocks = 0;
};
hipError_t launch_paged_evict(PoolType pool, const PagedBatch& b, const PagedEvict& e, const Workspace& ws, hipStream_t s);

// ---- sampling (kernels/sample.hip) ---------------------------------------------
hipError_t launch_sample(EType t, const void* logits, const float* u, const float* params, const int32_t* top_k,
                         int32_t* token, float* prob, uint32_t rows, uint32_t n, const Workspace& ws, hipStream_t s);

}  // namespace nfhip
