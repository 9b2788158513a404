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

// The choice, for a sequence and KV head ("row"), in three parts.
// 1. The least order that stays, 11, 11 and 10 bits at a time: a histogram of the orders
//    that agree in the bits known so far, and the bin in which the rank wanted lies.
// 2. Runs of the positions, of a wave each, are counted: what stays, and ties.
// 3. With the sums of the runs before it, each wave writes its own.
// A row of up to some thousand positions is one workgroup's, all in one launch; its
// steps, one after the other, bound it (600 positions 10 us; 32 sequences of up to 4096, 8 KV
// heads, 14.6; 131072 positions 158).  Longer ones are cut into chunks, and what the chunks
// have to know of each other is left between launches (two sequences of 131072, 8 KV heads:
// clearing 5 us, the histograms 7 each, counts 8, writing 10).
constexpr int kBins = 2048, kPasses = 3;
__device__ __forceinline__ int shift_of(int pass) { return pass == 0 ? 21 : pass == 1 ? 10 : 0; }
__device__ __forceinline__ uint32_t known_of(int pass) { return pass == 0 ? 0u : ~0u << (pass == 1 ? 21 : 10); }

// The last `left` known bits of the least order, and the rank wanted among what agrees with it.
struct Least {
  uint32_t order, left;
};

template <int THREADS>
struct SelectLds {
  uint32_t bins[kBins];
  uint32_t wave[2][THREADS / 64];
  uint32_t pick[3];  // the bin, how many orders lie above it and how many in it
};

// V weights of a row, at positions V v - off .. V v - off + V - 1 of the `n` that it has.
// V = 4: `off` elements before the row lies a multiple of 16 bytes.
template <int V>
struct RowV {
  typedef float vec __attribute__((ext_vector_type(4)));
  const float* w;
  int off, n;
  __device__ __forceinline__ RowV(const float* row, int count)
      : w(row), off(V == 4 ? (int)((reinterpret_cast<uintptr_t>(row) >> 2) & 3) : 0), n(count) {}
  __device__ __forceinline__ int vectors() const { return (n + off + V - 1) / V; }
  __device__ __forceinline__ vec get(int v) const {
    const int p = V * v - off;
    if constexpr (V == 1) return vec{w[p], 0.f, 0.f, 0.f};
    if (p >= 0 && p + V <= n) return *reinterpret_cast<const vec*>(w + p);
    vec x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (p + i >= 0 && p + i < n) x[i] = w[p + i];
    return x;
  }
};

template <int THREADS, int V>
struct Select {
  static constexpr int U = V == 1 ? 8 : 4, WAVES = THREADS / 64, PER = kBins / THREADS;  // vectors in flight; bins a thread
  typedef typename RowV<V>::vec vec;
  const PagedBatch& b;
  const PagedEvict& e;
  SelectLds<THREADS>& lds;
  uint32_t seq, tid, lane, wave;
  Budget t;
  uint64_t row;
  int old;        // positions that are chosen among
  uint32_t want;  // how many of them stay
  RowV<V> w;
  bool holes;     // a block of the row is not in the pools: positions are looked up

  __device__ __forceinline__ Select(const PagedBatch& b_, const PagedEvict& e_, uint32_t g, uint32_t s, SelectLds<THREADS>& l)
      : b(b_), e(e_), lds(l), seq(s), tid(threadIdx.x), lane(threadIdx.x & 63),
        wave((uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6))), t(find_budget(b_, e_, s)),
        row((uint64_t)s * b_.n_kv + g), old(t.len - t.recent), want((uint32_t)(t.keep - t.recent)),
        w(e_.weights + row * e_.width, t.len), holes(false) {}
  // Whether a block of the positions of the vectors v0 .. v1 - 1 is missing.
  __device__ __forceinline__ void look(int v0, int v1) {
    const int p0 = max(V * v0 - w.off, 0), p1 = min(V * v1 - w.off, t.len);
    bool h = false;
    if (p0 < p1)
      for (uint32_t i = (uint32_t)p0 / b.block_size + tid; i <= (uint32_t)(p1 - 1) / b.block_size; i += THREADS)
        h = h || b.table[(uint64_t)seq * b.width + i] >= b.blocks;
    holes = __syncthreads_or(h) != 0;
  }
  __device__ __forceinline__ uint32_t key_of(float x, int p) const { return holes && find_block(b, seq, p) == ~0u ? 0u : order_of(x); }
  // Whether there is anything to choose: else all or none of the first `old` stay.
  __device__ __forceinline__ bool chooses() const { return want > 0 && want < (uint32_t)old; }

  // The workgroup's bins of one pass.
  __device__ __forceinline__ void count(int pass, uint32_t least, int v0, int v1) {
    const int shift = shift_of(pass);
    const uint32_t mask = pass == 2 ? 1023u : 2047u, known = known_of(pass);
    for (int i = tid; i < kBins; i += THREADS) lds.bins[i] = 0;
    __syncthreads();
    for (int a = v0 + (int)tid; a < v1; a += THREADS * U) {
      vec x[U];
#pragma unroll
      for (int i = 0; i < U; ++i) x[i] = w.get(min(a + THREADS * i, v1 - 1));
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int v = a + THREADS * i;
        if (v >= v1) break;
#pragma unroll
        for (int c = 0; c < V; ++c) {
          const int p = V * v - w.off + c;
          if (p < 0 || p >= old) continue;
          const uint32_t k = key_of(x[i][c], p);
          if ((k & known) == least) atomicAdd(&lds.bins[(k >> shift) & mask], 1u);
        }
      }
    }
    __syncthreads();
  }
  // The bin of the rank wanted among `bins`, PER from the top a thread.
  __device__ __forceinline__ Least pick(const uint32_t* bins, int pass, Least l) {
    uint32_t n[PER], mine = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      n[i] = bins[kBins - 1 - PER * (int)tid - i];
      mine += n[i];
    }
    uint32_t up = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t v = __shfl_up(up, o);
      if ((int)lane >= o) up += v;
    }
    if (lane == 63) lds.wave[0][wave] = up;
    __syncthreads();
    uint32_t above = up - mine;
    for (uint32_t i = 0; i < wave; ++i) above += lds.wave[0][i];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (above < l.left && above + n[i] >= l.left) {
        lds.pick[0] = kBins - 1 - PER * tid - i;
        lds.pick[1] = above;
        lds.pick[2] = n[i];
      }
      above += n[i];
    }
    __syncthreads();
    return {l.order | lds.pick[0] << shift_of(pass), l.left - lds.pick[1]};
  }

  // f(first position, weights, bits of those that stay for sure, bits of the ties) for
  // the vectors from .. to - 1 of a wave.
  template <typename F>
  __device__ __forceinline__ void each(uint32_t least, int from, int to, F f) {
    const bool any = want > 0;
    for (int v0 = from; v0 < to; v0 += 64 * U) {
      vec x[U];
#pragma unroll
      for (int i = 0; i < U; ++i) x[i] = w.get(min(v0 + 64 * i + (int)lane, to - 1));
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int v = v0 + 64 * i + (int)lane, p0 = V * v - w.off;
        if (v0 + 64 * i >= to) break;  // uniform
        uint32_t above = 0, tied = 0;
#pragma unroll
        for (int c = 0; c < V; ++c) {
          const int p = p0 + c;
          if (v >= to || p < 0 || p >= t.len) continue;
          const uint32_t k = p < old && any ? key_of(x[i][c], p) : 0u;
          if (p >= old || (any && k > least)) above |= 1u << c;
          else if (any && k == least) tied |= 1u << c;
        }
        f(p0, x[i], above, tied);
      }
    }
  }
  // The runs of the waves in v0 .. v1 - 1.
  __device__ __forceinline__ int run(int v0, int v1) const { return (v1 - v0 + 64 * WAVES - 1) / (64 * WAVES) * 64; }
  // What stays for sure, and ties, of a wave's run.
  __device__ __forceinline__ uint2 tally(uint32_t least, int from, int to) {
    uint32_t n_above = 0, n_tied = 0;
    each(least, from, to, [&](int, const vec&, uint32_t above, uint32_t tied) {
      n_above += __popc(above);
      n_tied += __popc(tied);
    });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      n_above += __shfl_xor(n_above, o);
      n_tied += __shfl_xor(n_tied, o);
    }
    return {n_above, n_tied};
  }
  // Writes a wave's run; `before` stay for sure or are ties before it, the first `ties` of which stay.
  __device__ __forceinline__ void write(uint32_t least, uint32_t ties, int from, int to, uint2 before) {
    uint32_t tie = before.y, at = before.x + min(tie, ties);
    auto lower = [&](uint32_t mine, uint32_t& sum) {  // in the lanes below, and in all
      if constexpr (V == 1) {
        const uint64_t all = __ballot(mine != 0);
        sum = (uint32_t)__popcll(all);
        return (uint32_t)__popcll(all & ((1ull << lane) - 1));
      }
      uint32_t up = mine;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t v = __shfl_up(up, o);
        if ((int)lane >= o) up += v;
      }
      sum = (uint32_t)__builtin_amdgcn_readlane((int)up, 63);
      return up - mine;
    };
    each(least, from, to, [&](int p0, const vec& x, uint32_t above, uint32_t tied) {
      if (__ballot(tied != 0) != 0) {  // uniform
        uint32_t sum, mine = tie + lower(__popc(tied), sum);
        tie += sum;
#pragma unroll
        for (int c = 0; c < V; ++c)
          if ((tied >> c) & 1) above |= mine++ < ties ? 1u << c : 0u;
      }
      uint32_t sum, i = at + lower(__popc(above), sum);
      at += sum;
#pragma unroll
      for (int c = 0; c < V; ++c)
        if ((above >> c) & 1) {
          e.kept[row * e.top + i] = p0 + c;
          e.weights_to[row * e.width + i] = x[c];
          ++i;
        }
    });
  }
};
// Ties that stay: all of the first `old` do where want == old, being above order 0 or ties.
__device__ __forceinline__ uint32_t ties_of(bool chooses, const Least& l) { return chooses ? l.left : 0xFFFFFFFFu; }

constexpr int kSelect = 1024;
__global__ __launch_bounds__(kSelect) void select_kernel(PagedBatch b, PagedEvict e) {
  __shared__ SelectLds<kSelect> lds;
  Select<kSelect, 1> s(b, e, blockIdx.x, blockIdx.y, lds);
  if (blockIdx.x == 0 && s.tid == 0) e.lens_to[s.seq] = s.t.keep;
  if (s.t.keep == 0) return;  // uniform
  const int vectors = s.w.vectors();
  s.look(0, vectors);
  Least l{0, s.want};
  if (s.chooses())
#pragma unroll 1
    for (int pass = 0; pass < kPasses; ++pass) {
      s.count(pass, l.order, 0, vectors);
      l = s.pick(lds.bins, pass, l);
      if (lds.pick[2] == l.left) {  // uniform: the whole bin stays (and something below it goes)
        l = {l.order - 1, 0};
        break;
      }
    }
  const int run = s.run(0, vectors), from = (int)s.wave * run, to = min(from + run, vectors);
  const uint2 n = s.tally(l.order, from, to);
  __syncthreads();
  if (s.lane == 0) {
    lds.wave[0][s.wave] = n.x;
    lds.wave[1][s.wave] = n.y;
  }
  __syncthreads();
  uint2 before{0, 0};
  for (uint32_t i = 0; i < s.wave; ++i) {
    before.x += lds.wave[0][i];
    before.y += lds.wave[1][i];
  }
  s.write(l.order, ties_of(s.chooses(), l), from, to, before);
}

// Long rows.  Workgroup x takes 4096 positions; for each row the workspace has the bins of
// three passes, what is known after each, and the chunks' counts.
constexpr int kChunkVectors = 1024, kChunkThreads = 256;
struct LongRows {
  uint32_t* bins;   // [pass][row][kBins]
  Least* least;     // [pass][row]
  uint2* counts;    // [row][wave of a chunk]
  uint32_t rows, chunks;
};
__global__ __launch_bounds__(256) void clear_kernel(uint4* p, uint32_t n) {
  for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) p[i] = uint4{0, 0, 0, 0};
}
// Pass `pass` of the histogram (0 .. 2), the counts (3), or the writing (4).
template <int PASS>
__global__ __launch_bounds__(kChunkThreads) void long_kernel(PagedBatch b, PagedEvict e, LongRows r) {
  __shared__ SelectLds<kChunkThreads> lds;
  Select<kChunkThreads, 4> s(b, e, blockIdx.y, blockIdx.z, lds);
  if (PASS == 0 && blockIdx.x == 0 && blockIdx.y == 0 && s.tid == 0) e.lens_to[s.seq] = s.t.keep;
  const int v0 = (int)blockIdx.x * kChunkVectors, v1 = min(v0 + kChunkVectors, s.w.vectors());
  if (s.t.keep == 0 || v0 >= v1) return;  // uniform
  if (PASS < kPasses && !s.chooses()) return;
  Least l{0, s.want};
  if (PASS > 0 && s.chooses()) {
    if (PASS == 4) l = r.least[2 * r.rows + s.row];
    else {
      if (PASS > 1) l = r.least[(PASS - 2) * r.rows + s.row];
      l = s.pick(r.bins + ((uint64_t)(PASS - 1) * r.rows + s.row) * kBins, PASS - 1, l);
      if (blockIdx.x == 0 && s.tid == 0) r.least[(PASS - 1) * r.rows + s.row] = l;
      __syncthreads();
    }
  }
  s.look(v0, v1);
  if constexpr (PASS < kPasses) {
    s.count(PASS, l.order, v0, v1);
    uint32_t* const bins = r.bins + ((uint64_t)PASS * r.rows + s.row) * kBins;
    for (int i = s.tid; i < kBins; i += kChunkThreads)
      if (lds.bins[i]) atomicAdd(bins + i, lds.bins[i]);  // whole numbers: in any order
  } else {
    constexpr int W = kChunkThreads / 64;
    const int run = kChunkVectors / W, from = v0 + (int)s.wave * run, to = min(from + run, v1);
    uint2* const counts = r.counts + (uint64_t)s.row * r.chunks * W;
    const uint32_t mine = blockIdx.x * W + s.wave;
    if constexpr (PASS == kPasses) {
      const uint2 n = from < to ? s.tally(l.order, from, to) : uint2{0, 0};
      if (s.lane == 0) counts[mine] = n;
    } else {
      uint2 n{0, 0};
      for (uint32_t i = s.lane; i < mine; i += 64) {
        n.x += counts[i].x;
        n.y += counts[i].y;
      }
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) {
        n.x += __shfl_xor(n.x, o);
        n.y += __shfl_xor(n.y, o);
      }
      if (from < to) s.write(l.order, ties_of(s.chooses(), l), from, to, n);
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

// Rows of whole 16-byte pieces: a lane per piece, as many rows a wave as fit, kRows of them
// in flight, K and V.  Bound by HBM: 1024 rows of 32 sequences, 8 KV heads of 128, f16, 0.27
// GB in 60 us, 4.5 TB/s; 32768 of two, I8, 0.28 GB in 57 to 70 us, 4 to 4.9 TB/s.
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

// One workgroup takes 9 us and 1.1 us for each 1024 positions (and as long again for each
// 256 rows), the six launches of the chunks 25 us.
constexpr uint64_t kLongRow = 16384;
inline hipError_t select(const PagedBatch& b, const PagedEvict& e, const nfhip::Workspace& ws, hipStream_t s) {
  const uint64_t rows = (uint64_t)b.n_kv * b.n_seqs;
  const uint64_t chunks = ((uint64_t)b.limit + 3 + 4 * kChunkVectors - 1) / (4 * kChunkVectors);
  const uint64_t bins = kPasses * rows * kBins, words = bins + kPasses * rows * 2 + rows * chunks * (kChunkThreads / 64) * 2;
  if (b.limit * ((rows + 255) / 256) <= kLongRow || !ws.part || words > ws.part_floats) {
    select_kernel<<<dim3(b.n_kv, b.n_seqs), kSelect, 0, s>>>(b, e);
    return hipGetLastError();
  }
  LongRows r;
  r.bins = reinterpret_cast<uint32_t*>(ws.part);
  r.least = reinterpret_cast<Least*>(r.bins + bins);
  r.counts = reinterpret_cast<uint2*>(r.least + kPasses * rows);
  r.rows = (uint32_t)rows;
  r.chunks = (uint32_t)chunks;
  const uint32_t n = (uint32_t)(bins / 4);
  clear_kernel<<<dim3((n + 1023) / 1024 < 1024 ? (n + 1023) / 1024 : 1024), 256, 0, s>>>(reinterpret_cast<uint4*>(r.bins), n);
  const dim3 grid(r.chunks, b.n_kv, b.n_seqs);
  long_kernel<0><<<grid, kChunkThreads, 0, s>>>(b, e, r);
  long_kernel<1><<<grid, kChunkThreads, 0, s>>>(b, e, r);
  long_kernel<2><<<grid, kChunkThreads, 0, s>>>(b, e, r);
  long_kernel<3><<<grid, kChunkThreads, 0, s>>>(b, e, r);
  long_kernel<4><<<grid, kChunkThreads, 0, s>>>(b, e, r);
  return hipGetLastError();
}

template <PoolType PT>
hipError_t evict(const PagedBatch& b, const PagedEvict& e, const nfhip::Workspace& ws, hipStream_t s) {
  hipError_t err = select(b, e, ws, s);
  if (err != hipSuccess) return err;
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

hipError_t launch_paged_evict(PoolType pool, const PagedBatch& b, const PagedEvict& e, const Workspace& ws, hipStream_t s) {
  using namespace nfk;
  if (b.n_seqs == 0) return hipSuccess;
  return pool == PoolType::I8    ? paged::evict<PoolType::I8>(b, e, ws, s)
         : pool == PoolType::F16 ? paged::evict<PoolType::F16>(b, e, ws, s)
                                 : paged::evict<PoolType::F32>(b, e, ws, s);
}

}  // namespace nfhip
