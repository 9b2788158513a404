// paged_attention.hip — attention of chunks of new tokens over a paged cache
// (flash_attention_paged_chunk): row r of sequence s, at position pos, attends
// to positions 0 .. pos of its sequence,
//   o = sum_p exp(x_p - m) v_p / sum_p exp(x_p - m),  x_p = q . k_p / sqrt(dim),
// with m the running maximum of an online softmax.  Query head h reads KV head
// h * n_kv / n_heads.  A position without storage counts as no key; a row
// without any key gives zeros; rows of no sequence are left as they are.
#include <type_traits>

#include "paged.hpp"

namespace nfk {
namespace paged {

constexpr int kMaxDim = 256;
constexpr int kTile = 64;

// Any head_dim, head ratio and alignment.  A workgroup takes one (row, head);
// its four waves take 64-key tiles in turn: a lane scores one key, then the
// lanes lie over head_dim for the tile's 64 value rows, and the waves' (m, l,
// acc) are merged at the end.
template <typename T, PoolType PT>
__global__ __launch_bounds__(256) void chunk_any_kernel(PagedBatch b, uint32_t n_heads, float scale,
                                                        const T* __restrict__ q, const uint8_t* __restrict__ kp,
                                                        const uint8_t* __restrict__ vp, T* __restrict__ out) {
  constexpr int NW = 4, R = kMaxDim / 64;
  __shared__ float qs[kMaxDim];
  __shared__ float ps[NW][kTile];
  __shared__ uint32_t pb[NW][kTile];
  __shared__ float part_acc[NW][kMaxDim];
  __shared__ float part_m[NW], part_l[NW];
  const uint32_t row = blockIdx.x, h = blockIdx.y;
  uint32_t seq;
  int64_t pos;
  if (!find_row(b, row, seq, pos)) return;  // uniform
  const uint32_t kvh = (uint32_t)((uint64_t)h * b.n_kv / n_heads);
  const uint32_t D = b.dim;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t qrow = ((uint64_t)row * n_heads + h) * D;
  for (uint32_t d = threadIdx.x; d < D; d += 256) qs[d] = (float)q[qrow + d];
  __syncthreads();
  const int64_t last = pos < (int64_t)b.limit ? pos : (int64_t)b.limit - 1;
  float acc[R], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int r = 0; r < R; ++r) acc[r] = 0.0f;
  for (int64_t t0 = (int64_t)wave * kTile; t0 <= last; t0 += NW * kTile) {
    const int64_t p = t0 + lane;
    const uint32_t phys = p <= last ? find_block(b, seq, p) : ~0u;
    float s = -INFINITY;
    if (phys != ~0u) {
      const uint8_t* page = kp + page_offset<PT>(b, phys, kvh);
      const uint32_t slot = (uint32_t)p % b.block_size;
      float dot = 0.0f;
      for (uint32_t d = 0; d < D; ++d) dot += qs[d] * page_value<PT>(b, page, slot, d);
      s = dot * scale;
    }
    float tmax = s;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) tmax = fmaxf(tmax, __shfl_xor(tmax, o));
    if (tmax == -INFINITY) {
      if (__ballot(phys != ~0u && s != s) == 0) continue;  // no key of this tile counts
    }
    const float m_new = fmaxf(m, tmax);
    const float corr = m == m_new ? 1.0f : expf(m - m_new);
    const float pw = s == -INFINITY ? 0.0f : expf(s - m_new);
    l = l * corr + wave_sum(pw);
    m = m_new;
#pragma unroll
    for (int r = 0; r < R; ++r) acc[r] *= corr;
    ps[wave][lane] = pw;  // read back by this wave only
    pb[wave][lane] = s == -INFINITY ? ~0u : phys;
    __builtin_amdgcn_wave_barrier();
    const int nk = (int)(last - t0 + 1 < kTile ? last - t0 + 1 : kTile);
    for (int j = 0; j < nk; ++j) {
      const uint32_t pj = pb[wave][j];
      if (pj == ~0u) continue;  // uniform
      const uint8_t* page = vp + page_offset<PT>(b, pj, kvh);
      const uint32_t slot = (uint32_t)(t0 + j) % b.block_size;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const uint32_t d = lane + 64 * r;
        if (d < D) acc[r] += ps[wave][j] * page_value<PT>(b, page, slot, d);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
#pragma unroll
  for (int r = 0; r < R; ++r) part_acc[wave][lane + 64 * r] = acc[r];
  if (lane == 0) {
    part_m[wave] = m;
    part_l[wave] = l;
  }
  __syncthreads();
  float M = -INFINITY, L = 0.0f, wt[NW];
#pragma unroll
  for (int w = 0; w < NW; ++w) M = fmaxf(M, part_m[w]);
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    wt[w] = part_m[w] == M ? 1.0f : part_m[w] == -INFINITY ? 0.0f : expf(part_m[w] - M);
    L += part_l[w] * wt[w];
  }
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  for (uint32_t d = threadIdx.x; d < D; d += 256) {
    float o = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) o += part_acc[w][d] * wt[w];
    out[qrow + d] = (T)(o * inv);
  }
}

template <typename T, PoolType PT>
hipError_t chunk(const PagedBatch& b, uint32_t n_heads, const void* q, const void* kp, const void* vp, void* out,
                 const nfhip::Workspace&, hipStream_t s) {
  const float scale = 1.0f / sqrtf((float)b.dim);
  chunk_any_kernel<T, PT><<<dim3(b.rows, n_heads), 256, 0, s>>>(b, n_heads, scale, (const T*)q, (const uint8_t*)kp,
                                                                (const uint8_t*)vp, (T*)out);
  return hipGetLastError();
}

}  // namespace paged
}  // namespace nfk

namespace nfhip {

hipError_t launch_paged_chunk(EType t, PoolType pool, const PagedBatch& b, uint32_t n_heads, const void* q,
                              const void* k_pool, const void* v_pool, void* out, const Workspace& ws, hipStream_t s) {
  using namespace nfk;
  if (b.rows == 0 || b.n_seqs == 0) return hipSuccess;
  if (t == EType::F16)
    return pool == PoolType::I8 ? paged::chunk<half_t, PoolType::I8>(b, n_heads, q, k_pool, v_pool, out, ws, s)
                                : paged::chunk<half_t, PoolType::F16>(b, n_heads, q, k_pool, v_pool, out, ws, s);
  return pool == PoolType::I8 ? paged::chunk<float, PoolType::I8>(b, n_heads, q, k_pool, v_pool, out, ws, s)
                              : paged::chunk<float, PoolType::F32>(b, n_heads, q, k_pool, v_pool, out, ws, s);
}

}  // namespace nfhip
