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

// A workgroup per sequence and KV head, in three parts.
// 1. The least order that stays, 11, 11 and 10 bits at a time: a histogram of the row's
//    orders that agree in the bits known so far, and the bin in which the rank wanted lies.
// 2. Each wave takes a run of the positions and counts what stays of it, and its ties.
// 3. With the sums of the runs before it, each wave writes its own.
// The row is read five times, from the caches after the first.
constexpr int kSelect = 1024, kSelectWaves = kSelect / 64, kBins = 2048;
struct SelectLds {
  uint32_t bins[kBins];
  uint32_t wave[2][kSelectWaves];
  uint32_t pick[2];  // the bin, and how many orders lie above it
};
__global__ __launch_bounds__(kSelect) void select_kernel(PagedBatch b, PagedEvict e) {
  constexpr int U = 8;  // loads in flight
  __shared__ SelectLds lds;
  const uint32_t g = blockIdx.x, seq = blockIdx.y;
  const uint32_t tid = threadIdx.x, lane = tid & 63;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
  const Budget t = find_budget(b, e, seq);
  if (g == 0 && tid == 0) e.lens_to[seq] = t.keep;
  if (t.keep == 0) return;  // uniform
  const uint64_t row = (uint64_t)seq * b.n_kv + g;
  const float* w = e.weights + row * e.width;
  const int old = t.len - t.recent;  // positions that are chosen among
  const uint32_t want = (uint32_t)(t.keep - t.recent);
  // Where all blocks are in the pools no position is looked up.
  const uint32_t blocks = ((uint32_t)t.len + b.block_size - 1) / b.block_size;
  bool holes = false;
  for (uint32_t i = tid; i < blocks; i += kSelect) holes = holes || b.table[(uint64_t)seq * b.width + i] >= b.blocks;
  holes = __syncthreads_or(holes) != 0;
  auto key_of = [&](float x, int p) { return holes && find_block(b, seq, p) == ~0u ? 0u : order_of(x); };

  uint32_t least = 0, left = want;  // the bits of it known, and the rank wanted among what agrees with them
  if (want > 0 && want < (uint32_t)old) {
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const uint32_t mask = pass == 2 ? 1023u : 2047u, known = pass == 0 ? 0u : ~0u << (pass == 1 ? 21 : 10);
      for (int i = tid; i < kBins; i += kSelect) lds.bins[i] = 0;
      __syncthreads();
      for (int p0 = tid; p0 < old; p0 += kSelect * U) {
        float x[U];
#pragma unroll
        for (int i = 0; i < U; ++i) x[i] = w[min(p0 + kSelect * i, old - 1)];
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const int p = p0 + kSelect * i;
          if (p >= old) break;
          const uint32_t k = key_of(x[i], p);
          if ((k & known) == least) atomicAdd(&lds.bins[(k >> shift) & mask], 1u);
        }
      }
      __syncthreads();
      // Bins from the top: thread t has 2047 - 2t and the one below, and the sum of those above.
      const uint32_t hi = lds.bins[kBins - 1 - 2 * tid], lo = lds.bins[kBins - 2 - 2 * tid];
      uint32_t up = hi + lo;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t v = __shfl_up(up, o);
        if ((int)lane >= o) up += v;
      }
      if (lane == 63) lds.wave[0][wave] = up;
      __syncthreads();
      uint32_t above = up - hi - lo;
      for (uint32_t i = 0; i < wave; ++i) above += lds.wave[0][i];
      if (above < left && above + hi >= left) {
        lds.pick[0] = kBins - 1 - 2 * tid;
        lds.pick[1] = above;
      } else if (above + hi < left && above + hi + lo >= left) {
        lds.pick[0] = kBins - 2 - 2 * tid;
        lds.pick[1] = above + hi;
      }
      __syncthreads();
      least |= lds.pick[0] << shift;
      left -= lds.pick[1];
    }
  }
  // All of the first `old` stay where want == old: each is above `least` or a tie.
  const uint32_t ties = want == (uint32_t)old ? 0xFFFFFFFFu : left;
  const bool any = want > 0;
  const int run = (int)(((uint32_t)t.len + 64 * kSelectWaves - 1) / (64 * kSelectWaves)) * 64;
  const int from = (int)wave * run, to = min(from + run, t.len);
  uint32_t n_above = 0, n_tied = 0;
  auto each = [&](auto f) {
    for (int p0 = from; p0 < to; p0 += 64 * 4) {
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = w[min(p0 + 64 * i + (int)lane, t.len - 1)];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int p = p0 + 64 * i + (int)lane;
        if (p0 + 64 * i >= to) break;  // uniform
        const uint32_t k = p < old ? key_of(x[i], p) : 0u;
        const uint64_t above = __ballot(p < t.len && (p >= old || (any && k > least)));
        const uint64_t tied = __ballot(any && p < old && k == least);
        f(p, x[i], above, tied);
      }
    }
  };
  each([&](int, float, uint64_t above, uint64_t tied) {
    n_above += __popcll(above);
    n_tied += __popcll(tied);
  });
  if (lane == 0) {
    lds.wave[0][wave] = n_above;
    lds.wave[1][wave] = n_tied;
  }
  __syncthreads();
  uint32_t at = 0, tie = 0;  // kept ones and ties before
  for (uint32_t i = 0; i < wave; ++i) {
    at += lds.wave[0][i];
    tie += lds.wave[1][i];
  }
  at += min(tie, ties);
  const uint64_t below = (1ull << lane) - 1;
  each([&](int p, float x, uint64_t above, uint64_t tied) {
    const bool stays = ((above >> lane) & 1) || (((tied >> lane) & 1) && tie + __popcll(tied & below) < ties);
    const uint64_t all = __ballot(stays);
    if (stays) {
      const uint32_t i = at + __popcll(all & below);
      e.kept[row * e.top + i] = p;
      e.weights_to[row * e.width + i] = x;
    }
    at += __popcll(all);
    tie += __popcll(tied);
  });
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

// Rows of whole 16-byte pieces: a lane per piece, as many rows a wave as fit, kRows of them
// in flight, K and V.  Bound by HBM.
constexpr int kRows = 4;
template <PoolType PT>
__global__ __launch_bounds__(256) void move_kernel(PagedBatch b, PagedEvict e) {
  const uint32_t g = blockIdx.y, seq = blockIdx.z, lane = threadIdx.x & 63;
  const uint32_t keep = (uint32_t)find_budget(b, e, seq).keep, pages = (e.top + b.block_size - 1) / b.block_size;
  const uint64_t row = (uint64_t)seq * b.n_kv + g;
  const uint32_t bytes = PT == PoolType::I8 ? b.dim : b.dim * (PT == PoolType::F16 ? 2 : 4), pieces = bytes / 16;
  const uint32_t per = 64 / pieces, sub = lane / pieces, piece = lane % pieces;
  const uint32_t codes = b.block_size * b.dim, scales = b.dim / 32;  // I8
  const uint32_t step = 4 * per;
  for (uint32_t i0 = (blockIdx.x * kRows * 4 + (threadIdx.x >> 6)) * per; i0 < keep; i0 += gridDim.x * kRows * step) {
    uint64_t src[kRows], dst[kRows];
    uint32_t fs[kRows], ts[kRows];
    bool live[kRows], have[kRows];
    int32_t p[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const uint32_t i = i0 + r * step + sub;
      live[r] = sub < per && i < keep;
      p[r] = e.kept[row * e.top + (live[r] ? i : 0)];
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const uint32_t i = live[r] ? i0 + r * step + sub : 0;
      const uint32_t from = find_block(b, seq, p[r]), to = e.to[(uint64_t)seq * pages + i / b.block_size];
      live[r] = live[r] && to < e.to_blocks;
      have[r] = from != ~0u;
      fs[r] = have[r] ? (uint32_t)p[r] % b.block_size : 0;
      ts[r] = i % b.block_size;
      src[r] = have[r] ? page_offset<PT>(b, from, g) : 0;
      dst[r] = live[r] ? page_offset<PT>(b, to, g) : 0;
    }
    u32x4 x[2][kRows];
    uint16_t sc[2][kRows];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const uint8_t* s = static_cast<const uint8_t*>(j ? e.v : e.k) + src[r];
        x[j][r] = u32x4{0, 0, 0, 0};
        sc[j][r] = 0;
        if (live[r] && have[r]) {
          x[j][r] = *reinterpret_cast<const u32x4*>(s + (uint64_t)fs[r] * bytes + 16 * piece);
          if (PT == PoolType::I8 && piece < scales) sc[j][r] = reinterpret_cast<const uint16_t*>(s + codes)[fs[r] * scales + piece];
        }
      }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        if (!live[r]) continue;
        uint8_t* d = static_cast<uint8_t*>(j ? e.v_to : e.k_to) + dst[r];
        *reinterpret_cast<u32x4*>(d + (uint64_t)ts[r] * bytes + 16 * piece) = x[j][r];
        if (PT == PoolType::I8 && piece < scales) reinterpret_cast<uint16_t*>(d + codes)[ts[r] * scales + piece] = sc[j][r];
      }
  }
}

template <PoolType PT>
hipError_t evict(const PagedBatch& b, const PagedEvict& e, hipStream_t s) {
  select_kernel<<<dim3(b.n_kv, b.n_seqs), kSelect, 0, s>>>(b, e);
  if (e.top == 0) return hipGetLastError();
  const uintptr_t all = reinterpret_cast<uintptr_t>(e.k) | reinterpret_cast<uintptr_t>(e.v) |
                        reinterpret_cast<uintptr_t>(e.k_to) | reinterpret_cast<uintptr_t>(e.v_to);
  const uint64_t page = nfhip::page_bytes(PT, (uint64_t)b.block_size * b.dim), bytes = nfhip::page_bytes(PT, 16ull * b.dim) / 16;
  if (all % 16 == 0 && page % 16 == 0 && (PT == PoolType::I8 ? b.dim : bytes) % 16 == 0) {
    const uint32_t pieces = (PT == PoolType::I8 ? b.dim : (uint32_t)bytes) / 16, rows = 4 * kRows * (64 / pieces);
    const uint64_t n = ((uint64_t)e.top + rows - 1) / rows;
    move_kernel<PT><<<dim3((unsigned)(n < 65536 ? n : 65536), b.n_kv, b.n_seqs), 256, 0, s>>>(b, e);
    return hipGetLastError();
  }
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
