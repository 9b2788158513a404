// paged_evict.hip — eviction from a paged cache by accumulated weight
// (paged_kv_evict).  Of the L positions of a sequence each KV head keeps the last r
// and, of the first L - r, the k - r of the largest weights (equal ones: the lower
// position first; NaN and positions without storage below all others).  In order of
// position they become the positions 0 .. k - 1 of the sequence in its new blocks.
#include "paged.hpp"

namespace nfk {
namespace paged {

using nfhip::PagedEvict;

// A weight as an integer of the same order: NaN 0, then -inf, .. -0 = 0 .. +inf.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0;
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);  // -0 becomes 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct Budget {
  int len, keep, recent;
};
__device__ __forceinline__ Budget find_budget(const PagedBatch& b, const PagedEvict& e, uint32_t seq) {
  const int32_t n = b.lens[seq], k = e.budget[2 * seq], r = e.budget[2 * seq + 1];
  Budget t;
  t.len = n < 0 ? 0 : n < (int64_t)b.limit ? n : (int)b.limit;
  t.keep = k < 0 ? 0 : k < t.len ? k : t.len;
  if ((int64_t)t.keep > (int64_t)e.top) t.keep = (int)e.top;
  t.recent = r < 0 ? 0 : r < t.keep ? r : t.keep;
  return t;
}

// A workgroup per sequence and KV head.  The least order that stays is found bit by bit,
// counting the row's weights at each; then the row is gone over once more in order of
// position, 256 at a time.
constexpr int kSelect = 256;
__global__ __launch_bounds__(kSelect) void select_kernel(PagedBatch b, PagedEvict e) {
  constexpr int NW = kSelect / 64;
  __shared__ uint32_t count[2][NW];
  const uint32_t g = blockIdx.x, seq = blockIdx.y;
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Budget t = find_budget(b, e, seq);
  if (g == 0 && tid == 0) e.lens_to[seq] = t.keep;
  const uint64_t row = (uint64_t)seq * b.n_kv + g;
  const float* w = e.weights + row * e.width;
  const int old = t.len - t.recent;  // positions that are chosen among
  const uint32_t want = (uint32_t)(t.keep - t.recent);
  auto key = [&](int p) { return find_block(b, seq, p) == ~0u ? 0u : order_of(w[p]); };
  auto total = [&](uint32_t mine, int buf) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mine += __shfl_xor(mine, o);
    if (lane == 0) count[buf][wave] = mine;
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) all += count[buf][i];
    return all;
  };
  uint32_t least = 0;  // the largest value that at least `want` positions reach
  int buf = 0;
  if (want > 0)
    for (int bit = 31; bit >= 0; --bit, buf ^= 1) {
      const uint32_t at = least | 1u << bit;
      uint32_t mine = 0;
      for (int p = tid; p < old; p += kSelect) mine += key(p) >= at;
      if (total(mine, buf) >= want) least = at;
    }
  uint32_t above = 0;
  if (want > 0)
    for (int p = tid; p < old; p += kSelect) above += key(p) > least;
  above = total(above, buf);
  const uint32_t ties = want - above;  // of the equal ones, the first so many stay
  uint32_t kept = 0, equal = 0;
  for (int p0 = 0; p0 < t.len && kept < (uint32_t)t.keep; p0 += kSelect) {
    const int p = p0 + (int)tid;
    const uint32_t x = p < old ? key(p) : 0;
    const bool tie = want > 0 && p < old && x == least;
    const uint64_t tied = __ballot(tie);
    __syncthreads();
    if (lane == 0) count[0][wave] = __popcll(tied);
    __syncthreads();
    uint32_t before = equal;
    for (uint32_t i = 0; i < NW; ++i) {
      if (i < wave) before += count[0][i];
      equal += count[0][i];
    }
    before += __popcll(tied & ((1ull << lane) - 1));
    const bool stays = p < t.len && (p >= old || (want > 0 && (x > least || (tie && before < ties))));
    const uint64_t all = __ballot(stays);
    if (lane == 0) count[1][wave] = __popcll(all);
    __syncthreads();
    uint32_t to = kept;
    for (uint32_t i = 0; i < NW; ++i) {
      if (i < wave) to += count[1][i];
      kept += count[1][i];
    }
    to += __popcll(all & ((1ull << lane) - 1));
    if (stays) {
      e.kept[row * e.top + to] = p;
      e.weights_to[row * e.width + to] = w[p];
    }
  }
}

// A wave per kept row of a KV head, element by element (I8: and its scales).  A row
// without storage becomes zeros.
template <PoolType PT>
__global__ __launch_bounds__(256) void move_any_kernel(PagedBatch b, PagedEvict e) {
  const uint32_t g = blockIdx.y, seq = blockIdx.z, lane = threadIdx.x & 63;
  const uint32_t keep = (uint32_t)find_budget(b, e, seq).keep, pages = (e.top + b.block_size - 1) / b.block_size;
  const uint64_t row = (uint64_t)seq * b.n_kv + g;
  for (uint32_t i = blockIdx.x * 4 + (threadIdx.x >> 6); i < keep; i += gridDim.x * 4) {
    const int64_t p = e.kept[row * e.top + i];
    const uint32_t from = find_block(b, seq, p), to = e.to[(uint64_t)seq * pages + i / b.block_size];
    if (to >= e.to_blocks) continue;
    const uint32_t fs = (uint32_t)p % b.block_size, ts = i % b.block_size;
    const uint64_t src = from == ~0u ? 0 : page_offset<PT>(b, from, g), dst = page_offset<PT>(b, to, g);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint8_t* s = static_cast<const uint8_t*>(j ? e.v : e.k) + src;
      uint8_t* d = static_cast<uint8_t*>(j ? e.v_to : e.k_to) + dst;
      for (uint32_t x = lane; x < b.dim; x += 64) {
        if constexpr (PT == PoolType::F32)
          reinterpret_cast<float*>(d)[ts * b.dim + x] = from == ~0u ? 0.f : reinterpret_cast<const float*>(s)[fs * b.dim + x];
        else if constexpr (PT == PoolType::F16)
          reinterpret_cast<uint16_t*>(d)[ts * b.dim + x] = from == ~0u ? 0 : reinterpret_cast<const uint16_t*>(s)[fs * b.dim + x];
        else
          d[ts * b.dim + x] = from == ~0u ? 0 : s[fs * b.dim + x];
      }
      if constexpr (PT == PoolType::I8) {
        const uint32_t n = b.dim / 32, codes = b.block_size * b.dim;
        if (lane < n)
          reinterpret_cast<uint16_t*>(d + codes)[ts * n + lane] =
              from == ~0u ? 0 : reinterpret_cast<const uint16_t*>(s + codes)[fs * n + lane];
      }
    }
  }
}

template <PoolType PT>
hipError_t evict(const PagedBatch& b, const PagedEvict& e, hipStream_t s) {
  select_kernel<<<dim3(b.n_kv, b.n_seqs), kSelect, 0, s>>>(b, e);
  if (e.top == 0) return hipGetLastError();
  const uint64_t rows = ((uint64_t)e.top + 3) / 4, most = (65536 + (uint64_t)b.n_kv * b.n_seqs - 1) / ((uint64_t)b.n_kv * b.n_seqs);
  move_any_kernel<PT><<<dim3((unsigned)(rows < most ? rows : most), b.n_kv, b.n_seqs), 256, 0, s>>>(b, e);
  return hipGetLastError();
}

}  // namespace paged
}  // namespace nfk

namespace nfhip {

hipError_t launch_paged_evict(PoolType pool, const PagedBatch& b, const PagedEvict& e, hipStream_t s) {
  using namespace nfk;
  if (b.n_seqs == 0) return hipSuccess;
  return pool == PoolType::I8    ? paged::evict<PoolType::I8>(b, e, s)
         : pool == PoolType::F16 ? paged::evict<PoolType::F16>(b, e, s)
                                 : paged::evict<PoolType::F32>(b, e, s);
}

}  // namespace nfhip
