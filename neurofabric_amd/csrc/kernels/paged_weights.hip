// paged_weights.hip — the attention weights that a sequence's rows give its cached
// positions (paged_kv_weights): for position j of sequence s and KV head g
//   W[s][g][j] = theta held[s][g][j] + sum over rows r >= j, heads h of g:
//                exp(q_rh . k_j / sqrt(dim) - lse[r][h]),
// with lse the log-sum-exp that the attention left.  The positions of the rows
// themselves start from 0.  Positions past the length, and sequences without rows,
// are left as they are.  An 8-bit cache is read as f16 for f16 rows, as the
// attention reads it.
#include "paged_attention.hpp"

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
  uint32_t keys;    // of a workgroup
  uint64_t lo, hi;  // query rows of a KV head of the sequences that a launch takes
  // Many rows: cuts of a sequence's rows, and where each leaves its sums, [cut][sequence
  // among those][KV head][limit], if there is more than one.
  uint32_t cuts, many;
  float* part;
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
// scores one key, the four waves take query rows in turn and add up at the end.  Bound by
// LDS and the vector ALU (8 single tokens over 4096 positions, 32 heads over 8 KV heads of
// 80, f16: 171 us, 0.3 TB/s).
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
    float some = 0.f;  // of up to 32 rows
    uint32_t rows = 0;
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
      if (have && p <= pos && x != -INFINITY && lse != -INFINITY) some += expf(x - lse);
      if (++rows % 32 == 0) {  // uniform
        sum += some;
        some = 0.f;
      }
    }
    sum += some;
    part[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && p < t.len) {
      sum = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
      const float held = w.theta != 0.f && p < t.pos0 ? w.theta * w.held[row0 + p] : 0.f;
      w.out[row0 + p] = held + sum;
    }
  }
}

// ---- on MFMA ---------------------------------------------------------------------------
//
// S[row][key] = Q . K^T with the keys as the columns: a lane has one key (of a tile) and
// some of the rows, so a position's weights are added up in its registers, and over the 4
// (or 2) lanes of a column at the end.  Keys are the B operand as the cache holds them, a
// lane's 16 bytes; exp(x - lse) is one v_exp_f32 of base 2.  Where a sequence has many rows
// and few keys, its rows are cut as well, and the cuts' sums joined by another kernel.  The
// order of every sum is fixed.  Two tiles' weights are added up by themselves, and then to the
// position's, so that a sum of thousands of like weights is not rounded once for each row (4096
// rows of 8 heads that weigh 0.03 each: off by 39 half steps, by 3073 as one sum; 2048 rows of
// two prompts of 8192: 1.8e-7 and 7.1e-7 from 64 bits, 319 us both).

// What is taken off a row's score in base 2.
__device__ __forceinline__ float base_of(float lse) { return lse * 1.4426950408889634f; }
// The position up to which a row's weights count: a row that counts for nothing sees no
// position, as its scores may be infinite or NaN.
constexpr int kNowhere = -1;
__device__ __forceinline__ int sees_up_to(bool live, float lse, int64_t pos) {
  return live && lse != -INFINITY ? (int)pos : kNowhere;
}

// The sequence of a workgroup, its keys and query rows; false for none.
struct Task {
  Span t;
  RowTile tile;
  uint32_t group, live;
  int begin, end;
};
__device__ __forceinline__ bool find_task(const Weigh& w, uint32_t chunk, uint32_t seq, Task& k) {
  if (!find_span(w.b, seq, k.t)) return false;
  k.group = w.n_heads / w.b.n_kv;
  const uint64_t rows = (uint64_t)k.t.rows * k.group;
  const int64_t begin = (int64_t)chunk * w.keys;
  if (rows <= w.lo || rows > w.hi || begin >= (int64_t)k.t.len) return false;
  k.live = (uint32_t)rows;
  k.begin = (int)begin;
  k.end = begin + (int64_t)w.keys < (int64_t)k.t.len ? (int)(begin + w.keys) : k.t.len;
  k.tile.seq = seq;
  return true;
}
// Sequence number `at` among those with more than `lo` query rows; n_seqs for none.
__device__ __forceinline__ uint32_t find_many(const Weigh& w, uint32_t at) {
  const PagedBatch& b = w.b;
  const uint32_t group = w.n_heads / b.n_kv;
  for (uint32_t s0 = 0; s0 < b.n_seqs; s0 += 64) {
    const uint32_t s = s0 + (threadIdx.x & 63);
    Span t;
    const uint64_t mine = __ballot(s < b.n_seqs && find_span(b, s, t) && (uint64_t)t.rows * group > w.lo);
    const uint32_t n = (uint32_t)__popcll(mine);
    if (at < n) {
      uint64_t left = mine;
      for (; at > 0; --at) left &= left - 1;
      return s0 + (uint32_t)__builtin_ctzll(left);
    }
    at -= n;
  }
  return b.n_seqs;
}
__device__ __forceinline__ uint64_t q_row(const Weigh& w, const Task& k, uint32_t r, uint32_t kvh) {
  return (uint64_t)(k.t.start + r / k.group) * w.n_heads + kvh * k.group + r % k.group;
}
// A position's element: its old weight, faded, and the sum of the new ones.
__device__ __forceinline__ float held_of(const Weigh& w, uint64_t row0, const Task& k, int p) {
  return w.theta != 0.f && p < k.end && (int64_t)p < k.t.pos0 ? w.theta * w.held[row0 + p] : 0.f;
}

// Keys of one 16-key group as B operands, f16 (16x16x32) or f32 (16x16x4, whose order of
// dims is free: step s of lane group g is dim DD/4 g + s).
template <typename T, PoolType PT, int DD>
struct Keys16;
template <PoolType PT, int DD>
struct Keys16<half_t, PT, DD> {
  static constexpr bool I8 = PT == PoolType::I8;
  static constexpr int KS = DD / 32, NP = KS / 2;
  // I8: 16 codes are a lane's operands of two steps, the order of dims being free
  u32x4 raw[I8 ? (NP > 0 ? NP : 1) : KS];
  uint2 odd;  // I8, odd KS: the last 32 dims
  half_t scale[I8 ? KS : 1];
  // The dim of a lane's first element in step s.
  static __device__ __forceinline__ int dim(int s, int g) {
    return !I8 || s >= 2 * NP ? 32 * s + 8 * g : 64 * (s / 2) + 16 * g + 8 * (s % 2);
  }
  template <typename R>
  __device__ __forceinline__ void fetch(const R& rows, const uint8_t* pool, int j, int n, int g) {
    const uint8_t* kr = rows.row(pool, j, n);
    if constexpr (I8) {
      const half_t* sc = rows.scale(pool, j, n);
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        raw[p] = *reinterpret_cast<const u32x4*>(kr + 64 * p + 16 * g);
        scale[2 * p] = sc[2 * p + (g >> 1)];
      }
      if constexpr (KS % 2) {
        odd = *reinterpret_cast<const uint2*>(kr + 64 * NP + 8 * g);
        scale[KS - 1] = sc[KS - 1];
      }
    } else {
#pragma unroll
      for (int s = 0; s < KS; ++s) raw[s] = *reinterpret_cast<const u32x4*>(kr + 64 * s + 16 * g);
    }
  }
  __device__ __forceinline__ half8 get(int s) const {
    if constexpr (!I8) return __builtin_bit_cast(half8, raw[s]);
    else if (s >= 2 * NP) return dequant8(odd, scale[KS - 1]);
    else return dequant8(s % 2 ? uint2{raw[s / 2][2], raw[s / 2][3]} : uint2{raw[s / 2][0], raw[s / 2][1]}, scale[s / 2 * 2]);
  }
};
template <PoolType PT, int DD>
struct Keys16<float, PT, DD> {
  static constexpr bool I8 = PT == PoolType::I8;
  static constexpr int DG = DD / 4;
  float4v raw[I8 ? 1 : DG / 4];
  uint2 codes[I8 ? DG / 8 : 1];
  half_t scale[I8 ? DG / 8 : 1];
  template <typename R>
  __device__ __forceinline__ void fetch(const R& rows, const uint8_t* pool, int j, int n, int g) {
    const uint8_t* kr = rows.row(pool, j, n);
    if constexpr (I8) {
      const half_t* sc = rows.scale(pool, j, n);
#pragma unroll
      for (int p = 0; p < DG / 8; ++p) {
        codes[p] = *reinterpret_cast<const uint2*>(kr + DG * g + 8 * p);
        scale[p] = sc[(DG * g + 8 * p) / 32];
      }
    } else {
#pragma unroll
      for (int p = 0; p < DG / 4; ++p) raw[p] = *reinterpret_cast<const float4v*>(kr + 4 * (DG * g + 4 * p));
    }
  }
  __device__ __forceinline__ void all(float* x) const {
    if constexpr (I8) {
#pragma unroll
      for (int p = 0; p < DG / 8; ++p) codes8_f32(codes[p], (float)scale[p], x + 8 * p);
    } else {
#pragma unroll
      for (int p = 0; p < DG; ++p) x[p] = raw[p / 4][p % 4];
    }
  }
};
// 16 query rows as the A operand.
template <typename T, PoolType PT, int DD>
struct Query16;
template <PoolType PT, int DD>
struct Query16<half_t, PT, DD> {
  half8 x[DD / 32];
  __device__ __forceinline__ void fetch(const void* q, uint64_t row, int g) {
#pragma unroll
    for (int s = 0; s < DD / 32; ++s)
      x[s] = *reinterpret_cast<const half8*>(static_cast<const half_t*>(q) + row * DD + Keys16<half_t, PT, DD>::dim(s, g));
  }
  __device__ __forceinline__ float4v dot(const Keys16<half_t, PT, DD>& k) const {
    float4v c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < DD / 32; ++s) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[s], k.get(s), c, 0, 0, 0);
    return c;
  }
};
template <PoolType PT, int DD>
struct Query16<float, PT, DD> {
  float4v x[DD / 16];
  __device__ __forceinline__ void fetch(const void* q, uint64_t row, int g) {
#pragma unroll
    for (int s = 0; s < DD / 16; ++s)
      x[s] = *reinterpret_cast<const float4v*>(static_cast<const float*>(q) + row * DD + DD / 4 * g + 4 * s);
  }
  __device__ __forceinline__ float4v dot(const Keys16<float, PT, DD>& k) const {
    float b[DD / 4];
    k.all(b);
    float4v c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < DD / 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[s / 4][s % 4], b[s], c, 0, 0, 0);
    return c;
  }
};

// Single tokens and short chunks, up to 16 NT query rows, which stay in registers while
// the waves take 32-key tiles in turn, the next one's loads in flight.  Bound by HBM: 64
// single tokens over up to 8192 positions, 32 heads over 8 KV heads of 128, f16, 0.70 GB in
// 157 us, 4.4 TB/s; 16 over up to 32768, I8, 0.38 GB in 92 us, 4.1 TB/s, the codes'
// conversion beside it; one of 100 positions, f32, 4.9 us, by its latency.
template <typename T, PoolType PT, int DD, int NT, bool UNI>
__global__ __launch_bounds__(256) void weights_few_kernel(Weigh w) {
  Task k;
  const uint32_t kvh = blockIdx.y;
  if (!find_task(w, blockIdx.x, blockIdx.z, k)) return;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const float scale_log2 = w.scale * 1.4426950408889634f;
  const uint64_t row0 = ((uint64_t)k.tile.seq * w.b.n_kv + kvh) * w.width;
  Rows<PT, DD, 2, UNI, false> rows(w.b, k.tile, kvh, k.end, Border{});
  int t0 = k.begin + 32 * wave;
  if (t0 >= k.end) return;
  rows.look(t0);
  Query16<T, PT, DD> qa[NT];
  float base[NT][4];
  int pos[NT][4];
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    qa[u].fetch(w.q, q_row(w, k, min(16u * u + n, k.live - 1), kvh), g);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t r = 16 * u + 4 * g + i, at = min(r, k.live - 1);
      const float lse = w.lse[q_row(w, k, at, kvh)];
      pos[u][i] = sees_up_to(r < k.live, lse, k.t.pos0 + at / k.group);
      base[u][i] = base_of(lse);
    }
  }
  Keys16<T, PT, DD> keys[2];
  auto fetch = [&]() {
#pragma unroll
    for (int j = 0; j < 2; ++j) keys[j].fetch(rows, w.k, j, n, g);
  };
  rows.take(t0);
  fetch();
  if (t0 + 128 < k.end) rows.look(t0 + 128);
  for (;;) {
    const uint32_t seen = (uint32_t)rows.have();
    const int p = t0 + 16 * (g & 1) + n;
    const float held = held_of(w, row0, k, p);
    float4v sc[NT][2];
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int j = 0; j < 2; ++j) sc[u][j] = qa[u].dot(keys[j]);
    const int next = t0 + 128;
    if (next < k.end) {  // uniform
      rows.take(next);
      fetch();
      if (next + 128 < k.end) rows.look(next + 128);
    }
    float x[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      x[j] = 0.f;
#pragma unroll
      for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[u][j][i], scale_log2, -base[u][i]));
          x[j] += t0 + 16 * j + n <= pos[u][i] ? e : 0.f;
        }
      x[j] = sum4((seen >> (16 * j + n)) & 1 ? x[j] : 0.f);
    }
    if (g < 2 && p < k.end) w.out[row0 + p] = held + (g ? x[1] : x[0]);
    if (next >= k.end) break;
    t0 = next;
  }
}

// Tiles of `per` rows from the row `r0` on: those of cut `cut`.
struct Rows2 {
  uint32_t from, to;
};
__device__ __forceinline__ Rows2 cut_rows(const Weigh& w, const Task& k, uint32_t r0, uint32_t per, uint32_t cut) {
  if (r0 >= k.live) return {0, 0};
  const uint64_t n = (k.live - r0 + per - 1) / per;
  const uint64_t end = r0 + n * (cut + 1) / w.cuts * per;
  return {r0 + (uint32_t)(n * cut / w.cuts) * per, end < k.live ? (uint32_t)end : k.live};
}
// A position's sum: the element, or a cut's part of it.
__device__ __forceinline__ void put_sum(const Weigh& w, uint32_t cut, uint32_t kvh, uint64_t row0, int p, float held, float x) {
  if (w.cuts == 1) w.out[row0 + p] = held + x;
  else w.part[(((uint64_t)cut * w.many + blockIdx.z) * w.b.n_kv + kvh) * w.b.limit + p] = x;
}
// The cuts' sums, in order, and what was held.
__global__ __launch_bounds__(256) void weights_join_kernel(Weigh w) {
  Task k;
  const uint32_t kvh = blockIdx.y, seq = find_many(w, blockIdx.z);
  if (seq >= w.b.n_seqs || !find_task(w, blockIdx.x, seq, k)) return;
  const int p = k.begin + (int)threadIdx.x;
  if (p >= k.end) return;
  const uint64_t row0 = ((uint64_t)seq * w.b.n_kv + kvh) * w.width;
  const float held = held_of(w, row0, k, p);
  const float* part = w.part + ((uint64_t)blockIdx.z * w.b.n_kv + kvh) * w.b.limit + p;
  float x = 0.f;
  for (uint32_t c = 0; c < w.cuts; ++c) x += part[(uint64_t)c * w.many * w.b.n_kv * w.b.limit];
  w.out[row0 + p] = held + x;
}

// Many query rows, f16: 64 keys a wave stay in registers as B operands, 32-row tiles of the
// queries go through LDS for all four waves on v_mfma_f32_32x32x16_f16.  Per tile and wave
// there are DD / 8 MFMAs and 32 exponentials a lane, about as long: those of the tile before
// are issued between the MFMAs of the next one.  2048 rows of two sequences with 8192
// positions, 32 heads of 128: 241 GFLOP in 313 to 319 us a pass on several cards, 755 to 769 TFLOP/s, where a product of
// 8192 in each size reaches 1187; the MFMA pipes are 37 % busy, as the exponentials, the
// subtractions before them and the sums take as many issue slots.
template <PoolType PT, int DD, bool UNI>
__global__ __launch_bounds__(256, 2) void weights_many_kernel(Weigh w) {
  constexpr int KS = DD / 16, QP = DD + 8, CPR = DD / 8, NU = (32 * CPR + 255) / 256;
  __shared__ __attribute__((aligned(16))) half_t qs[3][32 * QP];
  __shared__ __attribute__((aligned(16))) float base[3][32];
  __shared__ __attribute__((aligned(16))) int place[3][32];
  Task k;
  const uint32_t kvh = blockIdx.y, seq = find_many(w, blockIdx.z), cut = blockIdx.x % w.cuts;
  if (seq >= w.b.n_seqs || !find_task(w, blockIdx.x / w.cuts, seq, k)) return;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, hf = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const float scale_log2 = w.scale * 1.4426950408889634f;
  const uint64_t row0 = ((uint64_t)k.tile.seq * w.b.n_kv + kvh) * w.width;
  const int t0 = k.begin + 64 * wave;  // (a workgroup's keys: 256)
  // the wave's keys
  Rows<PT, DD, 4, UNI, false> rows(w.b, k.tile, kvh, k.end, Border{});
  half8 kb[2][KS];
  uint64_t seen = 0;
  if (t0 < k.end) {  // uniform
    rows.look(t0);
    rows.take(t0);
    seen = rows.have();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      // lanes exchange for the rows' places, so both groups of 16 are asked for by all
      const uint8_t* r0 = rows.row(w.k, 2 * j, n & 15);
      const uint8_t* r1 = rows.row(w.k, 2 * j + 1, n & 15);
      const uint8_t* kr = n < 16 ? r0 : r1;
      if constexpr (PT == PoolType::I8) {
        const half_t* s0 = rows.scale(w.k, 2 * j, n & 15);
        const half_t* s1 = rows.scale(w.k, 2 * j + 1, n & 15);
        const half_t* sc = n < 16 ? s0 : s1;
#pragma unroll
        for (int s = 0; s < KS; ++s) kb[j][s] = dequant8(*reinterpret_cast<const uint2*>(kr + 16 * s + 8 * hf), sc[s / 2]);
      } else {
#pragma unroll
        for (int s = 0; s < KS; ++s) kb[j][s] = *reinterpret_cast<const half8*>(kr + 32 * s + 16 * hf);
      }
    }
  }
  const float held0 = held_of(w, row0, k, t0 + lane);

  // The first tile with a row that sees a key of the workgroup.
  const int64_t skip = (int64_t)k.begin - k.t.pos0;
  const Rows2 mine_rows = cut_rows(w, k, skip <= 0 ? 0 : (uint32_t)skip * k.group / 32 * 32, 32, cut);
  const uint32_t r0 = mine_rows.from, r_end = mine_rows.to;
  u32x4 raw[NU];
  float b0 = 0.f;
  int p0 = 0;
  // Token and head of a row, 32 rows further with each tile.
  struct Row {
    uint32_t token, head;
  };
  const uint32_t tokens = 32 / k.group, heads = 32 % k.group;
  auto row_at = [&](uint32_t r) { return Row{r / k.group, r % k.group}; };
  auto go_on = [&](Row& r) {
    r.token += tokens;
    r.head += heads;
    if (r.head >= k.group) {
      r.head -= k.group;
      ++r.token;
    }
  };
  auto place_of = [&](const Row& r) {  // past the last token: the last row
    const bool in = r.token < k.t.rows;
    return (uint64_t)(k.t.start + (in ? r.token : k.t.rows - 1)) * w.n_heads + kvh * k.group + (in ? r.head : k.group - 1);
  };
  Row at[NU], mine, first;
  auto begin = [&]() {
    uint32_t from = r0;
    asm volatile("" : "+s"(from));  // found anew in each pass, and not kept in registers for the next
    mine = row_at(from + (tid & 31));
    first = row_at(from);
#pragma unroll
    for (int u = 0; u < NU; ++u) at[u] = row_at(from + (tid + 256 * u < 32 * CPR ? tid + 256 * u : 32 * CPR - 1) / CPR);
  };
  auto fetch = [&]() {  // the next tile
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int ch = tid + 256 * u < 32 * CPR ? tid + 256 * u : 32 * CPR - 1;
      raw[u] = *reinterpret_cast<const u32x4*>(static_cast<const half_t*>(w.q) + place_of(at[u]) * DD + 8 * (ch % CPR));
      go_on(at[u]);
    }
    if (tid < 32) {
      b0 = w.lse[place_of(mine)];
      p0 = sees_up_to(mine.token < k.t.rows, b0, k.t.pos0 + mine.token);
      go_on(mine);
    }
  };
  auto stage = [&](int buf) {
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int ch = tid + 256 * u;
      if (32 * CPR % 256 == 0 || ch < 32 * CPR) *reinterpret_cast<u32x4*>(&qs[buf][ch / CPR * QP + 8 * (ch % CPR)]) = raw[u];
    }
    if (tid < 32) {
      base[buf][tid] = b0 == -INFINITY ? INFINITY : base_of(b0);
      place[buf][tid] = p0;
    }
  };
  float x[2] = {0.f, 0.f}, t[2] = {0.f, 0.f};  // the sums, and those of the last tiles
  // The scores of the tile in buffer `buf` into `next`, and the weights of those of `last`,
  // whose tile (bases in buffer `old`) has no row that does not see all keys (OPEN).
  auto step = [&](int buf, f32x16* next, int old, const f32x16* last, auto open_c) {
    constexpr bool OPEN = decltype(open_c)::value;
    half8 a[3];
#pragma unroll
    for (int s = 0; s < 2; ++s) a[s] = *reinterpret_cast<const half8*>(&qs[buf][n * QP + 16 * s + 8 * hf]);
    float4v bs[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) bs[q] = *reinterpret_cast<const float4v*>(&base[old][8 * q + 4 * hf]);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) next[j][i] = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      if (s + 2 < KS) a[(s + 2) % 3] = *reinterpret_cast<const half8*>(&qs[buf][n * QP + 16 * (s + 2) + 8 * hf]);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        next[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[s % 3], kb[j][s], next[j], 0, 0, 0);
        constexpr int EACH = 16 / KS;  // KS = 8, 6, 4: 2, 2 (and 4 more at the end), 4
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
          const int i = EACH * s + e;
          float v = __builtin_amdgcn_exp2f(__builtin_fmaf(last[j][i], scale_log2, -bs[i / 4][i % 4]));
          if constexpr (!OPEN) v = t0 + 32 * j + n <= place[old][8 * (i / 4) + 4 * hf + i % 4] ? v : 0.f;
          t[j] += v;
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 16 / KS * KS; i < 16; ++i) {
        float v = __builtin_amdgcn_exp2f(__builtin_fmaf(last[j][i], scale_log2, -bs[i / 4][i % 4]));
        if constexpr (!OPEN) v = t0 + 32 * j + n <= place[old][8 * (i / 4) + 4 * hf + i % 4] ? v : 0.f;
        t[j] += v;
      }
  };
  auto flush = [&]() {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      x[j] += t[j];
      t[j] = 0.f;
    }
  };
  // A row that counts for nothing weighs exp2(-inf) as well, unless its score is infinite or
  // NaN: where a sum is, all tiles are gone through again with a test of each row's place
  // (a look at each tile's rows took 331 us where this takes 319).
  for (bool strict = false;; strict = true) {
    if (r0 < r_end) {  // uniform
      // A first tile whose rows weigh exp2(-inf) stands before the first.
      begin();
      fetch();
      stage(0);
      if (tid < 32) {
        base[2][tid] = INFINITY;
        place[2][tid] = 0x7FFFFFFF;
      }
      if (r0 + 32 < r_end) fetch();
      __syncthreads();
      f32x16 sc[2][2];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[1][j][i] = 0.f;
      int buf = 0, old = 2;
      uint32_t r = r0;  // the tile in buf
      bool open = true; // the one in old: all rows see all keys
      // Two tiles a round, so that the scores' registers are known.
      for (;;) {
        bool done = false;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (done) break;
          const int nb = 3 - buf - old;
          const bool more = r + 32 < r_end;
          if (more) {
            stage(nb);  // its readers passed the last barrier
            if (r + 64 < r_end) fetch();
          }
          if (t0 < k.end) {  // uniform
            if (open) step(buf, sc[h], old, sc[h ^ 1], std::true_type{});
            else step(buf, sc[h], old, sc[h ^ 1], std::false_type{});
          }
          open = !strict && (int64_t)k.t.pos0 + first.token >= (int64_t)t0 + 63;
          go_on(first);
          old = buf;
          buf = nb;
          r += 32;
          __syncthreads();
          if (!more) {
            // the last tile's weights
            if (t0 < k.end) {
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const int at = 8 * (i / 4) + 4 * hf + i % 4;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                  const float v = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[h][j][i], scale_log2, -base[old][at]));
                  t[j] += t0 + 32 * j + n <= place[old][at] ? v : 0.f;
                }
              }
            }
            done = true;
          }
        }
        flush();
        if (done) break;
      }
    }
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 2; ++j) bad = bad || ((seen >> (32 * j + n)) & 1 && !(__builtin_fabsf(x[j]) < INFINITY));
    if (strict || !__syncthreads_or(bad)) break;  // uniform
    x[0] = x[1] = 0.f;
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) x[j] = sum2((seen >> (32 * j + n)) & 1 ? x[j] : 0.f);
  if (t0 + lane < k.end) put_sum(w, cut, kvh, row0, t0 + lane, held0, hf ? x[1] : x[0]);
}

// Many query rows, f32: 32 keys a wave stay in registers, 16-row tiles of the queries come
// straight from the caches, the next one in flight; the f32 MFMA's time hides them.  512
// rows of two sequences with 2048 positions, 32 heads of 128: 15 GFLOP, 183 us, 82 TFLOP/s
// of 153 (with one buffer of queries 261 where this took 213); the waits between a tile's few
// sums.
template <PoolType PT, int DD, bool UNI>
__global__ NF_TWO_PER_CU void weights_many_f32_kernel(Weigh w) {
  constexpr int DG = DD / 4;
  Task k;
  const uint32_t kvh = blockIdx.y, seq = find_many(w, blockIdx.z), cut = blockIdx.x % w.cuts;
  if (seq >= w.b.n_seqs || !find_task(w, blockIdx.x / w.cuts, seq, k)) return;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const float scale_log2 = w.scale * 1.4426950408889634f;
  const uint64_t row0 = ((uint64_t)k.tile.seq * w.b.n_kv + kvh) * w.width;
  const int t0 = k.begin + 32 * wave;  // (a workgroup's keys: 128)
  if (t0 >= k.end) return;
  Rows<PT, DD, 2, UNI, false> rows(w.b, k.tile, kvh, k.end, Border{});
  rows.look(t0);
  rows.take(t0);
  const uint32_t seen = (uint32_t)rows.have();
  float kb[2][DG];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    Keys16<float, PT, DD> keys;
    keys.fetch(rows, w.k, j, n, g);
    keys.all(kb[j]);
  }
  const int p = t0 + 16 * (g & 1) + n;
  const float held = held_of(w, row0, k, p);
  const int64_t skip = (int64_t)t0 - k.t.pos0;
  const Rows2 mine_rows = cut_rows(w, k, skip <= 0 ? 0 : (uint32_t)skip * k.group / 16 * 16, 16, cut);
  uint32_t r0 = mine_rows.from;
  const uint32_t r_end = mine_rows.to;
  Query16<float, PT, DD> qa[2];
  float lse[2][4];  // nothing is computed from a load before its turn, which would wait for it
  auto fetch = [&](int buf, uint32_t r) {
    qa[buf].fetch(w.q, q_row(w, k, min(r + n, k.live - 1), kvh), g);
#pragma unroll
    for (int i = 0; i < 4; ++i) lse[buf][i] = w.lse[q_row(w, k, min(r + 4 * g + i, k.live - 1), kvh)];
  };
  float x[2] = {0.f, 0.f};
  if (r0 < r_end) fetch(0, r0);
  while (r0 < r_end) {
    float t[2] = {0.f, 0.f};  // of two tiles
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (r0 >= r_end) continue;  // uniform
      // whether or not there is a next tile: behind a branch, the wait for this one's rows
      // would be one for the next one's too
      fetch(h ^ 1, r0 + 16);
      __builtin_amdgcn_sched_barrier(0);
      float4v sc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int s = 0; s < DG; ++s)
#pragma unroll
        for (int j = 0; j < 2; ++j) sc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(qa[h].x[s / 4][s % 4], kb[j][s], sc[j], 0, 0, 0);
      float base[4];
      bool count[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        base[i] = base_of(lse[h][i]);
        count[i] = sees_up_to(r0 + 4 * g + i < k.live, lse[h][i], 0) == 0;
      }
      const int64_t first = k.t.pos0 + r0 / k.group;
      if (first >= (int64_t)t0 + 31 && __ballot(!(count[0] && count[1] && count[2] && count[3])) == 0) {  // uniform: all rows see all keys
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) t[j] += __builtin_amdgcn_exp2f(__builtin_fmaf(sc[j][i], scale_log2, -base[i]));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t pos = k.t.pos0 + (r0 + 4 * g + i) / k.group;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[j][i], scale_log2, -base[i]));
            t[j] += count[i] && (int64_t)t0 + 16 * j + n <= pos ? e : 0.f;
          }
        }
      }
      r0 += 16;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) x[j] += t[j];
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) x[j] = sum4((seen >> (16 * j + n)) & 1 ? x[j] : 0.f);
  if (g < 2 && p < k.end) put_sum(w, cut, kvh, row0, p, held, g ? x[1] : x[0]);
}

// ---- launch ------------------------------------------------------------------------------

template <typename T, PoolType PT, int DD, bool UNI>
hipError_t weights_mfma(Weigh& w, const nfhip::Workspace& ws, hipStream_t s) {
  constexpr bool F16 = std::is_same<T, half_t>::value;
  constexpr uint32_t kManyKeys = F16 ? 256 : 128;
  const PagedBatch& b = w.b;
  const uint64_t rows = (uint64_t)b.rows * (w.n_heads / b.n_kv), pairs = (uint64_t)b.n_kv * b.n_seqs;
  // Rows of a sequence are known on the device only: each kernel leaves the sequences that
  // are the other's.  A lone sequence's are the kernel's for many, though it may have few of
  // the batch's rows, the others padding.
  const uint32_t few_rows = rows > 16ull * b.n_seqs ? 32 : 16;
  const bool many = rows > few_rows, few = b.n_seqs > 1 || !many;
  if (many) {
    w.lo = few ? few_rows : 0;
    w.hi = ~0ull;
    w.keys = kManyKeys;
    const uint64_t most = rows / (few_rows + 1);  // such sequences
    w.many = (uint32_t)(most < b.n_seqs ? most : b.n_seqs);
    const uint64_t chunks = (b.limit + (uint64_t)kManyKeys - 1) / kManyKeys, wgs = chunks * b.n_kv * w.many;
    // Cuts of the rows for two workgroups a CU, of four tiles at least, as far as their sums
    // fit the workspace (494 tokens of 4 heads over 4833 positions, one KV head, f32: 296 us
    // without).
    const uint64_t tile_rows = F16 ? 128 : 64, mean = rows / w.many, floats = (uint64_t)w.many * b.n_kv * b.limit;
    uint64_t cuts = wgs < 512 ? 512 / wgs : 1;
    if (cuts > mean / tile_rows) cuts = mean / tile_rows;
    if (!ws.part || cuts * floats > ws.part_floats) cuts = ws.part ? ws.part_floats / floats : 1;
    w.cuts = (uint32_t)(cuts < 1 ? 1 : cuts);
    w.part = ws.part;
    const dim3 grid((unsigned)(chunks * w.cuts), b.n_kv, w.many);
    if constexpr (F16) weights_many_kernel<PT, DD, UNI><<<grid, 256, 0, s>>>(w);
    else weights_many_f32_kernel<PT, DD, UNI><<<grid, 256, 0, s>>>(w);
    if (w.cuts > 1) {
      w.keys = 256;
      weights_join_kernel<<<dim3((unsigned)((b.limit + 255ull) / 256), b.n_kv, w.many), 256, 0, s>>>(w);
    }
  }
  if (few) {
    // Keys of a workgroup, some 8192 workgroups where no sequence is shorter than the bound:
    // 64 sequences of up to 8192 positions, f16, by 256, 512 and 1024 keys 170, 160, 165 us;
    // 16 of up to 32768, I8, 107, 103, 113.
    uint64_t keys = ((uint64_t)b.limit * pairs / 8192 + 127) / 128 * 128;
    keys = keys < 128 ? 128 : keys > 2048 ? 2048 : keys;
    w.lo = 0;
    w.hi = few_rows;
    w.keys = (uint32_t)keys;
    const dim3 grid((unsigned)((b.limit + keys - 1) / keys), b.n_kv, b.n_seqs);
    if (few_rows == 32) weights_few_kernel<T, PT, DD, 2, UNI><<<grid, 256, 0, s>>>(w);
    else weights_few_kernel<T, PT, DD, 1, UNI><<<grid, 256, 0, s>>>(w);
  }
  return hipGetLastError();
}

template <typename T, PoolType PT>
hipError_t weights(Weigh& w, const nfhip::Workspace& ws, hipStream_t s) {
  const PagedBatch& b = w.b;
  if (pieces_fit<PT>(b, w.n_heads, Operands{w.q, w.k, nullptr, nullptr, nullptr})) {
    const bool uni = uniform_blocks(b);
    if (b.dim == 128) return (uni ? weights_mfma<T, PT, 128, true> : weights_mfma<T, PT, 128, false>)(w, ws, s);
    if (b.dim == 96) return (uni ? weights_mfma<T, PT, 96, true> : weights_mfma<T, PT, 96, false>)(w, ws, s);
    return (uni ? weights_mfma<T, PT, 64, true> : weights_mfma<T, PT, 64, false>)(w, ws, s);
  }
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
                                float theta, const Workspace& ws, hipStream_t s) {
  using namespace nfk;
  if (b.rows == 0 || b.n_seqs == 0 || b.limit == 0) return hipSuccess;
  paged::Weigh w{b, q, static_cast<const uint8_t*>(k_pool), lse, held, weights, n_heads, width, theta, 1.0f / sqrtf((float)b.dim), 0, 0, 0, 1, 0, nullptr};
  if (t == EType::F16)
    return pool == PoolType::I8 ? paged::weights<half_t, PoolType::I8>(w, ws, s) : paged::weights<half_t, PoolType::F16>(w, ws, s);
  return pool == PoolType::I8 ? paged::weights<float, PoolType::I8>(w, ws, s) : paged::weights<float, PoolType::F32>(w, ws, s);
}

}  // namespace nfhip
