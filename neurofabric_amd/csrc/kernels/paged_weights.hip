// paged_weights.hip — the attention weights that a sequence's rows give its cached
// positions (paged_kv_weights): for position j of sequence s and KV head g
//   W[s][g][j] = theta held[s][g][j] + sum over rows r >= j, heads h of g:
//                exp(q_rh . k_j / sqrt(dim) - lse[r][h]),
// with lse the log-sum-exp that the attention left.  The positions of the rows
// themselves start from 0.  Positions past the length, and sequences without rows,
// are left as they are.  An 8-bit cache is read as f16 for f16 rows, as the
// attention reads it.
#include <type_traits>

#include "paged.hpp"

namespace nfk {
namespace paged {

struct Weigh {
  PagedBatch b;
  const void* q;
  const uint8_t* k;
  const float* lse;
  const float* held;
  float* out;
  uint32_t n_heads, width;
  float theta, scale;
};

// The sequence's first row, rows and positions; false without rows or positions.
struct Span {
  uint32_t start, rows;
  int64_t pos0;  // position of the first row
  int len;       // positions, at most `limit`
};
__device__ __forceinline__ bool find_span(const PagedBatch& b, uint32_t seq, Span& t) {
  const int64_t a = b.starts[seq], e = b.starts[seq + 1];
  const int32_t len = b.lens[seq];
  if (a < 0 || e <= a || e > (int64_t)b.rows || len <= 0) return false;
  t.start = (uint32_t)a;
  t.rows = (uint32_t)(e - a);
  t.pos0 = (int64_t)len - (e - a);
  t.len = len < (int64_t)b.limit ? len : (int)b.limit;
  return true;
}

// Any head_dim, head ratio and alignment: 64 keys a workgroup, as f32 in LDS; a lane
// scores one key, the four waves take query rows in turn and add up at the end.
constexpr int kAnyDim = 256;
template <typename T, PoolType PT>
__global__ __launch_bounds__(256) void weights_any_kernel(Weigh w) {
  __shared__ float ks[64][kAnyDim + 1];
  __shared__ float part[4][64];
  const PagedBatch& b = w.b;
  const uint32_t g = blockIdx.y, seq = blockIdx.z, D = b.dim;
  Span t;
  if (!find_span(b, seq, t)) return;
  const uint32_t h0 = (uint32_t)(((uint64_t)g * w.n_heads + b.n_kv - 1) / b.n_kv);  // heads h with h n_kv / n_heads == g
  const uint32_t h1 = (uint32_t)(((uint64_t)(g + 1) * w.n_heads + b.n_kv - 1) / b.n_kv), G = h1 - h0;
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t row0 = ((uint64_t)seq * b.n_kv + g) * w.width;
  for (int64_t t0 = (int64_t)blockIdx.x * 64; t0 < t.len; t0 += (int64_t)gridDim.x * 64) {
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < 64 * D; i += 256) {
      const uint32_t j = i / D, d = i % D;
      const uint32_t phys = t0 + j < t.len ? find_block(b, seq, t0 + j) : ~0u;
      float x = 0.f;
      if (phys != ~0u)
        x = row_value<T, PT>(b, w.k + page_offset<PT>(b, phys, g), (uint32_t)(t0 + j) % b.block_size, d);
      ks[j][d] = x;
    }
    __syncthreads();
    const int64_t p = t0 + lane;
    const bool have = p < t.len && find_block(b, seq, p) != ~0u;
    float sum = 0.f;
    const uint64_t n = (uint64_t)t.rows * G;
    for (uint64_t r = wave; r < n; r += 4) {
      const uint32_t tok = (uint32_t)(r / G), h = h0 + (uint32_t)(r % G);
      const int64_t pos = t.pos0 + tok;
      if (pos < t0) continue;  // uniform
      const uint64_t at = (uint64_t)(t.start + tok) * w.n_heads + h;
      const T* q = static_cast<const T*>(w.q) + at * D;
      const float lse = w.lse[at];
      float dot = 0.f;
      for (uint32_t d = 0; d < D; ++d) dot += (float)q[d] * ks[lane][d];
      const float x = dot * w.scale;
      if (have && p <= pos && x != -INFINITY && lse != -INFINITY) sum += expf(x - lse);
    }
    part[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && p < t.len) {
      sum = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
      const float held = w.theta != 0.f && p < t.pos0 ? w.theta * w.held[row0 + p] : 0.f;
      w.out[row0 + p] = held + sum;
    }
  }
}

template <typename T, PoolType PT>
hipError_t weights(Weigh& w, hipStream_t s) {
  const PagedBatch& b = w.b;
  const uint64_t tiles = ((uint64_t)b.limit + 63) / 64, most = (65536 + (uint64_t)b.n_kv * b.n_seqs - 1) / ((uint64_t)b.n_kv * b.n_seqs);
  const dim3 grid((unsigned)(tiles < most ? tiles : most), b.n_kv, b.n_seqs);
  weights_any_kernel<T, PT><<<grid, 256, 0, s>>>(w);
  return hipGetLastError();
}

}  // namespace paged
}  // namespace nfk

namespace nfhip {

hipError_t launch_paged_weights(EType t, PoolType pool, const PagedBatch& b, uint32_t n_heads, const void* q,
                                const void* k_pool, const float* lse, const float* held, float* weights, uint32_t width,
                                float theta, hipStream_t s) {
  using namespace nfk;
  if (b.rows == 0 || b.n_seqs == 0 || b.limit == 0) return hipSuccess;
  paged::Weigh w{b, q, static_cast<const uint8_t*>(k_pool), lse, held, weights, n_heads, width, theta, 1.0f / sqrtf((float)b.dim)};
  if (t == EType::F16)
    return pool == PoolType::I8 ? paged::weights<half_t, PoolType::I8>(w, s) : paged::weights<half_t, PoolType::F16>(w, s);
  return pool == PoolType::I8 ? paged::weights<float, PoolType::I8>(w, s) : paged::weights<float, PoolType::F32>(w, s);
}

}  // namespace nfhip
