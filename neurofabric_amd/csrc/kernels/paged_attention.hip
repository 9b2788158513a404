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
// acc) are merged at the end.  Element loads, which every query head of a KV head
// makes again, and the vector ALU bound it: single tokens of 8 sequences of 4096
// positions with 32 query and 8 KV heads of 80 take 650 us in f16, where heads of 128
// on the MFMA kernel take 31.
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

// ---- shared by the MFMA kernels --------------------------------------------------

// Row tiles of the batch.  A sequence of n rows (tokens) has n G query rows per
// KV head (G query heads read it), row r being token r / G, head kvh G + r % G:
// all of them share the KV head's keys.  Sequences with `lo` < n G <= `hi` query
// rows are cut into tiles of `per`; tile `idx` of KV head and batch is found by a
// scan over the sequences, 64 at a time.
struct RowTile {
  uint32_t seq, first, rows;  // sequence, first query row, query rows of the sequence
  uint32_t start;             // the sequence's first token
  int pos0;                   // position of that token
  int len;                    // positions of the sequence, at most `limit`
};

__device__ __forceinline__ bool find_tile(const PagedBatch& b, uint32_t idx, uint32_t G, uint32_t per, uint64_t lo,
                                          uint64_t hi, RowTile& t) {
  const int lane = threadIdx.x & 63;
  for (uint32_t s0 = 0; s0 < b.n_seqs; s0 += 64) {
    const uint32_t s = s0 + lane;
    uint32_t n = 0, start = 0;
    int32_t len = 0;
    if (s < b.n_seqs) {
      const int64_t a = b.starts[s], e = b.starts[s + 1];
      len = b.lens[s];
      if (a >= 0 && e > a && e <= (int64_t)b.rows) {
        n = (uint32_t)(e - a);
        start = (uint32_t)a;
      }
    }
    const uint64_t rows = (uint64_t)n * G;
    const uint32_t tiles = rows > lo && rows <= hi ? (uint32_t)((rows + per - 1) / per) : 0;
    uint32_t up = tiles;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t v = __shfl_up(up, o);
      if (lane >= o) up += v;
    }
    const uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)up, 63);
    if (idx < total) {
      const int at = __builtin_ctzll(__ballot(up > idx));
      auto of = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, at); };
      t.seq = s0 + at;
      t.first = (idx - of(up - tiles)) * per;
      t.rows = of((uint32_t)rows);
      t.start = of(start);
      const int l = (int)of((uint32_t)len);
      t.pos0 = l - (int)of(n);
      t.len = l < (int)b.limit ? l : (int)b.limit;
      return true;
    }
    idx -= total;
  }
  return false;
}

// What every kernel of an attention launch is given.
struct Chunk {
  PagedBatch b;
  const void* q;
  const uint8_t* k;
  const uint8_t* v;
  void* out;
  float* ml;   // partials: (maximum, sum) of split sp of query row (token, head) at 2 ((token H + head) splits + sp)
  float* acc;  // and its unscaled output row
  uint32_t n_heads, group, splits, keys_per_split;
  uint32_t tiles;  // grid size: row tiles per KV head
  uint64_t lo, hi; // query rows of the sequences that this launch takes
  float scale_log2;  // scale * log2(e): softmax in base 2
};

// Splits that a sequence of `len` positions takes.
__device__ __forceinline__ uint32_t splits_of(const Chunk& c, int len) {
  return len <= 0 ? 1u : ((uint32_t)len + c.keys_per_split - 1) / c.keys_per_split;
}

__device__ __forceinline__ uint64_t shfl64(uint64_t v, int src) {
  return (uint64_t)(uint32_t)__shfl((int)(uint32_t)v, src) | (uint64_t)(uint32_t)__shfl((int)(uint32_t)(v >> 32), src) << 32;
}

// Where the rows of a tile of 16 N keys lie.  UNI (block_size a power of two of at least
// 16): each 16 keys lie in one block, whose address is the same for the wave and stays
// in scalar registers, so a lane's address is that and an offset that never changes.
// Otherwise lane j looks up key j's row, and the others ask it: 18 exchanges between
// lanes and the 64-bit additions for each 32-key tile of an I8 cache, where the time is
// that of instructions (decode of four long sequences 214 us, with UNI 164).
// look() reads the table entries of the tile that take() then makes the current one, so
// that they arrive while the one before is computed; by vector loads, as scalar ones
// and LDS reads share a counter that can only be waited for as a whole.  Keys without
// a row have that of the pool's first key, and no bit in have().
template <PoolType PT, int DD, int N, bool UNI>
struct Rows {
  static constexpr uint32_t kRow = PT == PoolType::I8 ? DD : PT == PoolType::F16 ? 2 * DD : 4 * DD;
  const PagedBatch& b;
  const uint32_t* table;  // of the sequence
  uint32_t page;          // bytes of a page (at most 65536 * 256 * 4)
  uint64_t block, head;   // bytes of a block, and from its start to the KV head's page
  int end;                // keys below it
  int shift;              // UNI: log2 of block_size
  uint32_t entry;         // UNI: lane h has the block of the next tile's group h
  int cur;                // UNI: the current tile's first key
  uint64_t base[N];
  uint32_t scales[N];
  uint64_t off, next_off;  // else: the lane's key
  uint32_t sc, next_sc;
  uint64_t valid, next_valid;

  __device__ __forceinline__ Rows(const PagedBatch& b_, uint32_t seq, uint32_t kvh, int end_)
      : b(b_), table(b_.table + (uint64_t)seq * b_.width),
        page((uint32_t)nfhip::page_bytes(PT, (uint64_t)b_.block_size * DD)), block((uint64_t)b_.n_kv * page),
        head((uint64_t)kvh * page), end(end_), shift(__builtin_ctz(b_.block_size)) {}
  // From a key's row to its scales.
  __device__ __forceinline__ uint32_t to_scales(uint32_t at) const {
    return PT == PoolType::I8 ? (b.block_size - at) * DD + at * (DD / 16) : 0;
  }
  __device__ __forceinline__ void look(int t0) {
    if constexpr (UNI) {
      const int p = t0 + 16 * (int)(threadIdx.x & (N - 1));
      entry = table[(uint32_t)min(p, end - 1) >> shift];  // past the end: the last key's block, whose bits are cleared
    } else {
      const int p = t0 + (int)(threadIdx.x & (16 * N - 1));
      next_off = 0;
      next_sc = 0;
      bool ok = false;
      if (p < end) {
        const uint32_t k = (uint32_t)p / b.block_size, at = (uint32_t)p - k * b.block_size, phys = table[k];
        ok = phys < b.blocks;
        if (ok) {
          next_off = phys * block + head + at * kRow;
          next_sc = to_scales(at);
        }
      }
      next_valid = __ballot(ok);
      if constexpr (N < 4) next_valid &= (1ull << (16 * N)) - 1;
    }
  }
  __device__ __forceinline__ void take(int t0) {
    if constexpr (UNI) {
      cur = t0;
      valid = 0;
#pragma unroll
      for (int h = 0; h < N; ++h) {
        const uint32_t phys = (uint32_t)__builtin_amdgcn_readlane((int)entry, h);
        const uint32_t at = (uint32_t)(t0 + 16 * h) & (b.block_size - 1);
        const bool ok = phys < b.blocks;
        base[h] = ok ? phys * block + head + at * kRow : 0;
        scales[h] = ok ? to_scales(at) : 0;
        valid |= (uint64_t)(ok ? 0xFFFFu : 0u) << (16 * h);
      }
      const int left = end - t0;
      if (left < 16 * N) valid &= (1ull << left) - 1;
    } else {
      off = next_off;
      sc = next_sc;
      valid = next_valid;
    }
  }
  // base[h], and scales[h] in `to`, for an h that is known when the kernel runs and the same
  // for the wave; between take() and the next look().
  __device__ __forceinline__ uint64_t place(int h, uint32_t& to) const {
    const uint32_t phys = (uint32_t)__builtin_amdgcn_readlane((int)entry, h);
    const uint32_t at = (uint32_t)(cur + 16 * h) & (b.block_size - 1);
    const bool ok = phys < b.blocks;
    to = ok ? to_scales(at) : 0;
    return ok ? phys * block + head + at * kRow : 0;
  }
  __device__ __forceinline__ uint64_t have() const { return valid; }
  // The row of a key of the first two groups that differs between lanes, and its scales.
  // (Lanes exchange here: no branch around the exchange may leave one out.)
  __device__ __forceinline__ const uint8_t* row_of(const uint8_t* pool, uint32_t r) const {
    if constexpr (UNI) return pool + (r < 16 ? base[0] : base[1]) + (r & 15) * kRow;
    else return pool + shfl64(off, r);
  }
  __device__ __forceinline__ const half_t* scale_of(const uint8_t* pool, uint32_t r) const {
    if constexpr (UNI)
      return reinterpret_cast<const half_t*>(pool + (r < 16 ? base[0] + scales[0] : base[1] + scales[1]) + (r & 15) * (DD / 16));
    else return reinterpret_cast<const half_t*>(pool + shfl64(off, r) + (uint32_t)__shfl((int)sc, r));
  }
  // The row of key 16 h + r, and its scales.
  __device__ __forceinline__ const uint8_t* row(const uint8_t* pool, int h, uint32_t r) const {
    if constexpr (UNI) return pool + base[h] + r * kRow;
    else return pool + shfl64(off, 16 * h + r);
  }
  __device__ __forceinline__ const half_t* scale(const uint8_t* pool, int h, uint32_t r) const {
    if constexpr (UNI) return reinterpret_cast<const half_t*>(pool + base[h] + scales[h] + r * (DD / 16));
    else return reinterpret_cast<const half_t*>(pool + shfl64(off, 16 * h + r) + (uint32_t)__shfl((int)sc, 16 * h + r));
  }
};

// Eight codes as f16: 0x64cc is 1024 + cc, so (code + 128) goes into the low byte
// and 1152 off again (exact); times the scale, rounded once to f16.
__device__ __forceinline__ half8 dequant8(uint2 w, half_t d) {
  const half2v off = {(half_t)1152.0f, (half_t)1152.0f}, dd = {d, d};
  half8 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t x = (i ? w.y : w.x) ^ 0x80808080u;
    const half2v lo = (__builtin_bit_cast(half2v, __builtin_amdgcn_perm(x, 0x64646464u, 0x00050004u)) - off) * dd;
    const half2v hi = (__builtin_bit_cast(half2v, __builtin_amdgcn_perm(x, 0x64646464u, 0x00070006u)) - off) * dd;
    r[4 * i] = lo[0];
    r[4 * i + 1] = lo[1];
    r[4 * i + 2] = hi[0];
    r[4 * i + 3] = hi[1];
  }
  return r;
}
__device__ __forceinline__ bool any_not_finite(half8 x) {
  const u32x4 u = __builtin_bit_cast(u32x4, x);
  uint32_t bad = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) bad |= (uint32_t)((u[i] & 0x7C00u) == 0x7C00u) | (uint32_t)((u[i] & 0x7C000000u) == 0x7C000000u);
  return bad != 0;
}

// Sum / max over the 4 lanes of a column (lanes n, n + 16, n + 32, n + 48) or the
// 2 of one (n, n + 32) with the swaps of lane rows; s_nop covers the wait states
// between a VALU write and a permlane read.
template <bool ROW32>
__device__ __forceinline__ float2s lane_swap(float v) {
  float a = v, b = v;
  if constexpr (ROW32) asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
  else asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
  return float2s{a, b};
}
__device__ __forceinline__ float max2(float v) {
  const float2s r = lane_swap<true>(v);
  return fmaxf(r[0], r[1]);
}
__device__ __forceinline__ float sum2(float v) {
  const float2s r = lane_swap<true>(v);
  return r[0] + r[1];
}
__device__ __forceinline__ float max4(float v) {
  const float2s r = lane_swap<false>(v);
  return max2(fmaxf(r[0], r[1]));
}
__device__ __forceinline__ float sum4(float v) {
  const float2s r = lane_swap<false>(v);
  return sum2(r[0] + r[1]);
}

// The f16 weights carry 2^kWeightLog2, which keeps the small ones out of the
// subnormal range (it is divided out with the sum); the reference maximum may lag
// the running one by 2^kLagLog2 before the sums are rescaled, so weights stay
// below 2^15.
constexpr float kWeightLog2 = 7.f, kLagLog2 = 8.f;

// What is taken off the scores in the weights' exponents, for a running maximum `m` and
// weights times 2^`log2`.  Finite while every score so far is -inf: those weigh
// exp2(-inf) = 0, where -inf - -inf would be NaN.
__device__ __forceinline__ float exponent_base(float m, float log2) { return m == -INFINITY ? 0.f : m - log2; }

typedef short short4v __attribute__((ext_vector_type(4)));
// ds_read_b64_tr_b16: among each 16 lanes, lane i receives element i % 4 of the 8
// bytes that lane 4e + i / 4 addresses, as its element e.
__device__ __forceinline__ uint2 read_tr(const half_t* p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)p));
}

// ---- few query rows: keys split over the waves, f16 ----------------------------------
//
// Single tokens and short chunks, where the cache is read once and the time is
// that of reading it.  A workgroup takes up to 16 NT query rows of one KV head
// and one split of the keys; its four waves take 32-key tiles in turn, each on
// its own, and merge at the end.  Per tile:
//  * S^T[key][row] = K . Q^T on v_mfma_f32_16x16x32_f16: a lane loads the 8 dims
//    of its key that are its A operand straight from the cache (16 bytes; I8: 16
//    codes are the operands of two steps, the order of the dims being free);
//  * base-2 online softmax per row;
//  * O^T[dim][row] += V^T . P^T: the weights are the B operand as S^T leaves them,
//    rounded to f16 (2^-11 of each, the size of the output's own rounding); V
//    goes through the wave's own part of LDS (no workgroup barrier), from where
//    transposing reads fetch the A operand.
// An 8-bit cache becomes f16 in registers, code * scale rounded once, as a gather
// into f16 rows would.
// A weight of 0 times a value that is not finite is NaN inside the MFMA, so values
// that no row sees are stored as zeros, and a tile that has a value that is not
// finite and a row that does not see some key of it takes the vector ALU, which
// skips the pairs that are masked.
// Bound by HBM at f16 (64 sequences of up to 8192 positions, 8 KV heads of 128: 1.35 GB
// in 262 us, 5.2 TB/s, where a copy of 2 GiB reaches 4.9), by it and the conversion's
// instructions at I8 (4 of up to 131072: 0.83 GB in 158 to 166 us, 5.1 TB/s); with 20 rows
// a sequence by the conversion (16 of up to 4096: 91 MB in 31 us).
template <PoolType PT, int DD, int NT, bool UNI>
__global__ __launch_bounds__(256, 2) void chunk_narrow_kernel(Chunk c) {
  constexpr bool I8 = PT == PoolType::I8;
  constexpr int KSTEP = DD / 32, DB = DD / 16;
  // LDS row (halves): 8 dwords past a multiple of 64 or an odd multiple of 8, so that
  // the 8 rows that 32 lanes of a transposing read touch lie in different banks
  constexpr int VP = DD + 16;
  constexpr int VC = I8 ? 16 : 8;                    // elements per 16-byte chunk
  constexpr int CPR = DD / VC, NV = 32 * CPR / 64;   // chunks per row, per lane and tile
  constexpr int NP = KSTEP / 2;                      // I8: 16-code loads per key row
  __shared__ __attribute__((aligned(16))) half_t vs[4][32 * VP];
  __shared__ __attribute__((aligned(16))) float ps[4][32][16];
  __shared__ float wm[4][16 * NT], wl[4][16 * NT];
  static_assert(sizeof(float) * 16 * DD <= sizeof(half_t) * 32 * VP, "a wave's rows merge in its part of vs");

  const uint32_t sp = blockIdx.x % c.splits, kvh = blockIdx.y;
  RowTile t;
  if (!find_tile(c.b, blockIdx.x / c.splits, c.group, 16 * NT, c.lo, c.hi, t)) return;
  const uint32_t ns = splits_of(c, t.len);
  if (sp >= ns) return;
  const uint32_t G = c.group, H = c.n_heads;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t live = t.rows - t.first < 16u * NT ? t.rows - t.first : 16u * NT;
  // positions of the tile's rows, first to last
  const int pos_lo = t.pos0 + (int)(t.first / G), pos_hi = t.pos0 + (int)((t.first + live - 1) / G);
  const int begin = (int)(sp * c.keys_per_split);
  int end = pos_hi + 1 < t.len ? pos_hi + 1 : t.len;  // keys below it
  if (end > begin + (int)c.keys_per_split) end = begin + (int)c.keys_per_split;
  end = __builtin_amdgcn_readfirstlane(end);

  half8 qb[NT][KSTEP];
  int pos[NT];
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    const uint32_t r = t.first + 16 * u + n < t.rows ? t.first + 16 * u + n : t.rows - 1;
    pos[u] = t.pos0 + (int)(r / G);
    const half_t* qr = static_cast<const half_t*>(c.q) + ((uint64_t)(t.start + r / G) * H + kvh * G + r % G) * DD;
#pragma unroll
    for (int s = 0; s < KSTEP; ++s) {
      const int d = !I8 || s >= 2 * NP ? 32 * s + 8 * g : 64 * (s / 2) + 16 * g + 8 * (s % 2);
      qb[u][s] = *reinterpret_cast<const half8*>(qr + d);
    }
  }
  float4v ot[NT][DB];
  float m[NT], l[NT];
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    m[u] = -INFINITY;
    l[u] = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d) ot[u][d] = float4v{0.f, 0.f, 0.f, 0.f};
  }

  u32x4 kraw[2][I8 ? (NP > 0 ? NP : 1) : KSTEP];
  uint2 kodd[2];       // I8, odd KSTEP: the last 32 dims
  half_t kd[2][KSTEP]; // I8: scales
  u32x4 vraw[NV];
  half_t vd[NV];
  Rows<PT, DD, 2, UNI> rows(c.b, t.seq, kvh, end);
  auto fetch = [&]() {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint8_t* kr = rows.row(c.k, j, n);
      if constexpr (I8) {
        const half_t* sc = rows.scale(c.k, j, n);
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          kraw[j][p] = *reinterpret_cast<const u32x4*>(kr + 64 * p + 16 * g);
          kd[j][2 * p] = sc[2 * p + (g >> 1)];
        }
        if constexpr (KSTEP % 2) {
          kodd[j] = *reinterpret_cast<const uint2*>(kr + 64 * NP + 8 * g);
          kd[j][KSTEP - 1] = sc[KSTEP - 1];
        }
      } else {
#pragma unroll
        for (int s = 0; s < KSTEP; ++s) kraw[j][s] = *reinterpret_cast<const u32x4*>(kr + 64 * s + 16 * g);
      }
    }
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int ch = lane + 64 * u, r = ch / CPR, col = ch % CPR;
      if constexpr (16 * CPR % 64 == 0) {  // the 64 chunks of a load lie in one group of 16 keys
        const int h = 64 * u / (16 * CPR);
        vraw[u] = *reinterpret_cast<const u32x4*>(rows.row(c.v, h, r - 16 * h) + 16 * col);
        if constexpr (I8) vd[u] = rows.scale(c.v, h, r - 16 * h)[col / 2];
      } else {
        vraw[u] = *reinterpret_cast<const u32x4*>(rows.row_of(c.v, r) + 16 * col);
        if constexpr (I8) vd[u] = rows.scale_of(c.v, r)[col / 2];
      }
    }
  };

  half_t* const vw = vs[w];
  const half_t* const vtr = vw + (4 * g + n / 4) * VP + 4 * (n % 4);
  int t0 = begin + 32 * w;
  if (t0 < end) {
    rows.look(t0);
    rows.take(t0);
    fetch();
    if (t0 + 128 < end) rows.look(t0 + 128);
  }
  auto next = [&]() {
    if (t0 + 128 >= end) return;
    rows.take(t0 + 128);
    fetch();
    if (t0 + 256 < end) rows.look(t0 + 256);
  };
  // One tile; OPEN: every row sees every key, and no check is needed.
  auto tile = [&](uint32_t seen, auto open_c) {
    constexpr bool OPEN = decltype(open_c)::value;
    // scores
    float4v sc[NT][2];
    {
      half8 ka[2][KSTEP];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if constexpr (I8) {
#pragma unroll
          for (int p = 0; p < NP; ++p) {
            ka[j][2 * p] = dequant8(uint2{kraw[j][p][0], kraw[j][p][1]}, kd[j][2 * p]);
            ka[j][2 * p + 1] = dequant8(uint2{kraw[j][p][2], kraw[j][p][3]}, kd[j][2 * p]);
          }
          if constexpr (KSTEP % 2) ka[j][KSTEP - 1] = dequant8(kodd[j], kd[j][KSTEP - 1]);
        } else {
#pragma unroll
          for (int s = 0; s < KSTEP; ++s) ka[j][s] = __builtin_bit_cast(half8, kraw[j][s]);
        }
      }
#pragma unroll
      for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          sc[u][j] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < KSTEP; ++s)
            sc[u][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[j][s], qb[u][s], sc[u][j], 0, 0, 0);
        }
    }
    // (the scheduling barriers keep the compiler from starting on one phase's operands
    // while it holds another's: they do not fit the registers together)
    __builtin_amdgcn_sched_barrier(0);
    // values into the wave's part of LDS, rows without storage as zeros
    bool bad = false;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int ch = lane + 64 * u, r = ch / CPR, col = ch % CPR;
      half8 x[I8 ? 2 : 1];
      if constexpr (I8) {
        x[0] = dequant8(uint2{vraw[u][0], vraw[u][1]}, vd[u]);
        x[1] = dequant8(uint2{vraw[u][2], vraw[u][3]}, vd[u]);
      } else {
        x[0] = __builtin_bit_cast(half8, vraw[u]);
      }
#pragma unroll
      for (int e = 0; e < VC / 8; ++e) {
        if constexpr (!OPEN) {
          if (!((seen >> r) & 1)) x[e] = half8{};
          bad = bad || any_not_finite(x[e]);
        }
        *reinterpret_cast<half8*>(vw + r * VP + VC * col + 8 * e) = x[e];
      }
    }
    const bool alu = !OPEN && __ballot(bad) != 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the wave's LDS accesses stay in order
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_sched_barrier(0);
    if (OPEN) next();
    __builtin_amdgcn_sched_barrier(0);
    half8 pb[NT];
    float pv[NT][2][4];
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = 16 * j + 4 * g + i;
          if (!OPEN && (!((seen >> k) & 1) || t0 + k > pos[u])) sc[u][j][i] = -INFINITY;
          top = fmaxf(top, sc[u][j][i]);
        }
      top = max4(top) * c.scale_log2;
      if (__ballot(top > m[u] + kLagLog2) != 0) {  // uniform
        const float mn = fmaxf(m[u], top);
        const float corr = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[u] - mn);
        l[u] *= corr;
#pragma unroll
        for (int d = 0; d < DB; ++d) ot[u][d] *= corr;
        m[u] = mn;
      }
      const float mb = exponent_base(m[u], kWeightLog2);
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          pv[u][j][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[u][j][i], c.scale_log2, -mb));
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const half2v h = __builtin_convertvector(float2s{pv[u][k / 2][2 * (k % 2)], pv[u][k / 2][2 * (k % 2) + 1]}, half2v);
        pb[u][2 * k] = h[0];
        pb[u][2 * k + 1] = h[1];
        sum = __builtin_amdgcn_fdot2(h, half2v{(half_t)1.f, (half_t)1.f}, sum, false);
      }
      l[u] += sum4(sum);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (!alu) {
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        if (d % 4 == 0) __builtin_amdgcn_sched_barrier(0);
        const uint2 lo = read_tr(vtr + 16 * d), hi = read_tr(vtr + 16 * VP + 16 * d);
        const half8 av = __builtin_bit_cast(half8, u32x4{lo.x, lo.y, hi.x, hi.y});
#pragma unroll
        for (int u = 0; u < NT; ++u) ot[u][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, pb[u], ot[u][d], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int u = 0; u < NT; ++u) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) ps[w][16 * j + 4 * g + i][n] = pv[u][j][i];
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 1
        for (int k = 0; k < 32; ++k) {
          if (!((seen >> k) & 1) || t0 + k > pos[u]) continue;
          const float p = ps[w][k][n];
#pragma unroll
          for (int d = 0; d < DB; ++d) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 4; ++i) ot[u][d][i] += p * (float)vw[k * VP + 16 * d + 4 * g + i];
          }
        }
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the next tile's values come after these reads
    __builtin_amdgcn_wave_barrier();
    if (!OPEN) next();
  };
  // The open tiles come first: those that every row sees whole, up to the first that
  // has a hole.  Two loops, as one with both bodies does not fit the registers.
  while (t0 < end && (uint32_t)rows.have() == ~0u && t0 + 31 <= pos_lo) {  // uniform
    tile(~0u, std::true_type{});
    t0 += 128;
  }
  while (t0 < end) {
    tile((uint32_t)rows.have(), std::false_type{});
    t0 += 128;
  }

  // merge the waves, 16 rows at a time; write the output (a lone split) or the partial
#pragma unroll
  for (int u = 0; u < NT; ++u)
    if (g == 0) {
      wm[w][16 * u + n] = m[u];
      wl[w][16 * u + n] = l[u];
    }
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    if (u > 0) __syncthreads();
    float* mine = reinterpret_cast<float*>(vw);
#pragma unroll
    for (int d = 0; d < DB; ++d) *reinterpret_cast<float4v*>(mine + n * DD + 16 * d + 4 * g) = ot[u][d];
    __syncthreads();
    for (int idx = tid; idx < 16 * DD / 4; idx += 256) {
      const int r = idx / (DD / 4), d = idx % (DD / 4) * 4;
      const uint32_t row = t.first + 16 * u + r;
      if (row >= t.rows) break;
      float M = -INFINITY, L = 0.f;
#pragma unroll
      for (int v = 0; v < 4; ++v) M = fmaxf(M, wm[v][16 * u + r]);
      float4v A = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float mv = wm[v][16 * u + r];
        const float f = mv == M ? 1.f : __builtin_amdgcn_exp2f(mv - M);
        L += f * wl[v][16 * u + r];
        A += f * *reinterpret_cast<const float4v*>(reinterpret_cast<const float*>(vs[v]) + r * DD + d);
      }
      const uint64_t o = (uint64_t)(t.start + row / G) * H + kvh * G + row % G;
      if (ns == 1) {
        const float inv = L == 0.f ? 0.f : 1.0f / L;
        half2v a = {(half_t)(A[0] * inv), (half_t)(A[1] * inv)}, bb = {(half_t)(A[2] * inv), (half_t)(A[3] * inv)};
        *reinterpret_cast<uint2*>(static_cast<half_t*>(c.out) + o * DD + d) =
            uint2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, bb)};
      } else {
        const uint64_t p = o * c.splits + sp;
        if (d == 0) *reinterpret_cast<float2s*>(c.ml + 2 * p) = float2s{M, L};
        *reinterpret_cast<float4v*>(c.acc + p * DD + d) = A;
      }
    }
  }
}

// The splits of every query row whose sequence has more than one, where they are few:
// a wave per row.
constexpr uint32_t kFewSplits = 8;
template <typename T, int DD>
__global__ __launch_bounds__(256) void chunk_combine_few_kernel(Chunk c) {
  constexpr int R = (DD + 63) / 64;
  const uint32_t o = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  uint32_t seq;
  int64_t pos;
  if (o >= c.b.rows * c.n_heads || !find_row_wave(c.b, o / c.n_heads, seq, pos)) return;  // uniform
  const int len = c.b.lens[seq];
  const uint32_t ns = splits_of(c, len < (int)c.b.limit ? len : (int)c.b.limit);
  if (ns == 1) return;
  const uint64_t first = (uint64_t)o * c.splits;
  const float2s* ml = reinterpret_cast<const float2s*>(c.ml) + first;
  float x[kFewSplits][R], M = -INFINITY, L = 0.f, A[R] = {};
  float2s v[kFewSplits];
#pragma unroll
  for (uint32_t s = 0; s < kFewSplits; ++s) {
    const uint32_t at = s < ns ? s : ns - 1;
    v[s] = ml[at];
#pragma unroll
    for (int r = 0; r < R; ++r) x[s][r] = c.acc[(first + at) * DD + (lane + 64 * r < DD ? lane + 64 * r : DD - 1)];
  }
#pragma unroll
  for (uint32_t s = 0; s < kFewSplits; ++s) M = fmaxf(M, v[s][0]);
#pragma unroll
  for (uint32_t s = 0; s < kFewSplits; ++s) {
    if (s >= ns || v[s][1] == 0.f) continue;  // no key: its row may be anything
    const float f = v[s][0] == M ? 1.f : __builtin_amdgcn_exp2f(v[s][0] - M);
    L += f * v[s][1];
#pragma unroll
    for (int r = 0; r < R; ++r) A[r] += f * x[s][r];
  }
  const float inv = L == 0.f ? 0.f : 1.0f / L;
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (lane + 64 * r < DD) static_cast<T*>(c.out)[(uint64_t)o * DD + lane + 64 * r] = (T)(A[r] * inv);
}

// The same for many splits.  A workgroup per row: the splits' weights exp2(m - M) are
// formed once, then each wave sums every fourth split's row (a wave per row, which took
// them one after the other, needed 54 us for 64 splits of 128 rows of 128; for few
// splits this kernel is the slower one: three ragged f32 chunks of up to 389 tokens
// with 2000 positions 136 us, with a wave per row 117).
constexpr int kSplitsAtOnce = 256;
template <typename T, int DD>
__global__ __launch_bounds__(256) void chunk_combine_kernel(Chunk c) {
  constexpr int R = (DD + 63) / 64;
  __shared__ float weight[kSplitsAtOnce];
  __shared__ float part[4][64 * R];
  __shared__ float wave_m[4], wave_l[4];
  const uint32_t o = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint32_t seq;
  int64_t pos;
  if (!find_row_wave(c.b, o / c.n_heads, seq, pos)) return;  // uniform
  const int l = c.b.lens[seq];
  const uint32_t ns = splits_of(c, l < (int)c.b.limit ? l : (int)c.b.limit);
  if (ns == 1) return;
  const uint64_t first = (uint64_t)o * c.splits;
  const float2s* ml = reinterpret_cast<const float2s*>(c.ml) + first;
  float M = -INFINITY, L = 0.f;
  for (uint32_t s = tid; s < ns; s += 256) M = fmaxf(M, ml[s][0]);
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) M = fmaxf(M, __shfl_xor(M, k));
  if (lane == 0) wave_m[wave] = M;
  __syncthreads();
  M = fmaxf(fmaxf(wave_m[0], wave_m[1]), fmaxf(wave_m[2], wave_m[3]));
  float A[R] = {};
  for (uint32_t s0 = 0; s0 < ns; s0 += kSplitsAtOnce) {
    if (s0) __syncthreads();
    if (s0 + tid < ns) {
      const float2s v = ml[s0 + tid];
      const float f = v[0] == M ? 1.f : __builtin_amdgcn_exp2f(v[0] - M);
      weight[tid] = v[1] == 0.f ? 0.f : f;  // no key: its row may be anything
      L += v[1] == 0.f ? 0.f : f * v[1];
    }
    __syncthreads();
    const uint32_t n = ns - s0 < (uint32_t)kSplitsAtOnce ? ns - s0 : kSplitsAtOnce;
#pragma unroll 4
    for (uint32_t s = wave; s < n; s += 4) {
      const float f = weight[s];
      const float* a = c.acc + (first + s0 + s) * DD;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float x = a[lane + 64 * r < DD ? lane + 64 * r : DD - 1];
        A[r] += f == 0.f ? 0.f : f * x;
      }
    }
  }
  L = wave_sum(L);
  if (lane == 0) wave_l[wave] = L;
#pragma unroll
  for (int r = 0; r < R; ++r) part[wave][lane + 64 * r] = A[r];
  __syncthreads();
  L = (wave_l[0] + wave_l[1]) + (wave_l[2] + wave_l[3]);
  const float inv = L == 0.f ? 0.f : 1.0f / L;
  for (uint32_t d = tid; d < DD; d += 256)
    static_cast<T*>(c.out)[(uint64_t)o * DD + d] = (T)(((part[0][d] + part[1][d]) + (part[2][d] + part[3][d])) * inv);
}

// Workgroup x of a wide kernel -> KV head and row tile, late tiles (most keys) first.
// Workgroup x runs on XCD x % 8, and each XCD has its own L2: the tiles of a KV head go
// to one XCD where heads are a multiple of 8, else in turn to the XCDs that share the
// head (in halves of the tiles, one XCD had the long sequences: 165 us for three
// ragged f32 chunks, 133 so).
__device__ __forceinline__ bool wide_tile(const Chunk& c, uint32_t& kvh, uint32_t& idx) {
  const uint32_t xcd = blockIdx.x % 8, i = blockIdx.x / 8, n_kv = c.b.n_kv;
  uint32_t tile;
  if (n_kv % 8 == 0) {
    kvh = xcd * (n_kv / 8) + i / c.tiles;
    tile = i % c.tiles;
  } else if (8 % n_kv == 0) {
    const uint32_t share = 8 / n_kv;
    kvh = xcd / share;
    tile = i * share + xcd % share;
  } else {
    kvh = blockIdx.x % n_kv;
    tile = blockIdx.x / n_kv;
  }
  idx = c.tiles - 1 - tile;
  return tile < c.tiles && kvh < n_kv;
}
// Workgroups for it.
inline uint32_t wide_grid(uint32_t tiles, uint32_t n_kv) {
  return 8 % n_kv == 0 ? 8 * ((tiles + 8 / n_kv - 1) / (8 / n_kv)) : tiles * n_kv;
}

// ---- many query rows, f16 --------------------------------------------------------------
//
// A workgroup takes 128 query rows of one KV head, 32 per wave (and one split of
// the keys); 64-key tiles of K and V are staged row-major in LDS for all of them
// (an 8-bit cache becomes f16 there), the next tile's loads in flight meanwhile.
// The matrices are transposed as in the narrow kernel, on
// v_mfma_f32_32x32x16_f16: S^T[key][row] = K . Q^T with the queries held in
// registers; a lane then has half of its row's scores, and the weights, rounded to
// f16, are the B operand of O^T[dim][row] += V^T . P^T as they are.
// Masking, the lazy rescale and values that are not finite: as above; tiles that
// every row of the workgroup sees whole skip all of it.
// No unit bounds it by itself: a wave takes scores, exponentials and P.V one after the
// other.  Two sequences of 2048 tokens behind 6144, 32 heads of 128, 481 GFLOP in 604 to
// 638 us (several cards), 750 to 800 TFLOP/s, where a matrix product of 8192 in each size
// reaches 1093; the MFMA pipes are busy 32 % of the cycles, and without its softmax and
// staging this kernel took 364 us.  From I8 594 to 631 us: half the bytes to stage, the
// conversion beside the MFMAs.
template <PoolType PT, int DD, bool UNI>
__global__ __launch_bounds__(256, 2) void chunk_wide_kernel(Chunk c) {
  constexpr bool I8 = PT == PoolType::I8;
  constexpr int KS = DD / 16, DB = DD / 32, KP = DD + 8;
  // V rows 16 or 48 dwords past a multiple of 64: the 4 rows and 32 dims that 32 lanes
  // of a transposing read touch then lie in different banks (in rows of KP, pairs
  // of them share; 685 and 671 us at the size below)
  constexpr int VP = DD == 96 ? 96 : DD + 32;
  constexpr int VC = I8 ? 16 : 8;
  constexpr int CPR = DD / VC;
  constexpr int NU = (64 * CPR + 255) / 256;
  // two buffers for the open tiles; the masked ones use the first, and the second for
  // the weights of the vector ALU
  constexpr int BUF = 64 * (KP + VP);
  static_assert(BUF * sizeof(half_t) >= 4 * 32 * 32 * sizeof(float), "a buffer holds the weights");
  __shared__ __attribute__((aligned(16))) half_t lds[2 * BUF];
  __shared__ int tile_bad[2];
  half_t* const ks = lds;
  half_t* const vs = lds + 64 * KP;
  float(*const ps)[32][32] = reinterpret_cast<float(*)[32][32]>(lds + BUF);

  uint32_t kvh, idx;
  if (!wide_tile(c, kvh, idx)) return;
  const uint32_t sp = blockIdx.y;
  RowTile t;
  if (!find_tile(c.b, idx, c.group, 128, c.lo, c.hi, t)) return;
  const uint32_t ns = splits_of(c, t.len);
  if (sp >= ns) return;
  const uint32_t G = c.group, H = c.n_heads;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, hf = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t last = (t.first + 128 < t.rows ? t.first + 128 : t.rows) - 1;
  const int pos_lo = t.pos0 + (int)(t.first / G), pos_hi = t.pos0 + (int)(last / G);
  const int begin = (int)(sp * c.keys_per_split);
  int end = pos_hi + 1 < t.len ? pos_hi + 1 : t.len;
  if (end > begin + (int)c.keys_per_split) end = begin + (int)c.keys_per_split;
  end = __builtin_amdgcn_readfirstlane(end);

  const uint32_t r0 = t.first + 32 * w;
  const bool wave_live = r0 < t.rows;
  const uint32_t row = r0 + n < t.rows ? r0 + n : t.rows - 1;
  const uint64_t orow = (uint64_t)(t.start + row / G) * H + kvh * G + row % G;
  const int pos = t.pos0 + (int)(row / G);
  const int w_hi = __builtin_amdgcn_readfirstlane(t.pos0 + (int)((r0 + 31 < t.rows ? r0 + 31 : t.rows - 1) / G));
  half8 qb[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s)
    qb[s] = *reinterpret_cast<const half8*>(static_cast<const half_t*>(c.q) + orow * DD + 16 * s + 8 * hf);
  f32x16 ot[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) ot[d][i] = 0.f;
  float m = -INFINITY, l = 0.f, mb = 0.f;  // mb: exponent_base of m

  u32x4 kraw[NU], vraw[NU];
  half_t kd[NU], vd[NU];
  Rows<PT, DD, 4, UNI> rows(c.b, t.seq, kvh, end);
  auto fetch = [&]() {
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int ch = tid + 256 * u < 64 * CPR ? tid + 256 * u : 64 * CPR - 1;
      const int r = ch / CPR, col = ch % CPR;
      if constexpr (!UNI) {
        kraw[u] = *reinterpret_cast<const u32x4*>(rows.row(c.k, 0, r) + 16 * col);
        vraw[u] = *reinterpret_cast<const u32x4*>(rows.row(c.v, 0, r) + 16 * col);
        if constexpr (I8) {
          kd[u] = rows.scale(c.k, 0, r)[col / 2];
          vd[u] = rows.scale(c.v, 0, r)[col / 2];
        }
      } else if constexpr (16 * CPR == 256) {
        // F16, 128: the workgroup's 256 chunks lie in one group of 16 keys, known here (612 us at
        // the size above, looked up as the others 640).
        kraw[u] = *reinterpret_cast<const u32x4*>(rows.row(c.k, u, r - 16 * u) + 16 * col);
        vraw[u] = *reinterpret_cast<const u32x4*>(rows.row(c.v, u, r - 16 * u) + 16 * col);
      } else {
        // A wave's 64 lie in one group, or in two.  It looks up those alone, by scalar
        // instructions: a choice among the addresses of all four was made by 64-bit
        // multiplications in the vector ALU (I8, the same size: 953 us, and 594 to 631).
        const int c0 = 64 * (w + 4 * u), h0 = min(c0, 64 * CPR - 1) / (16 * CPR), h1 = min(c0 + 63, 64 * CPR - 1) / (16 * CPR);
        uint32_t so, rr = r - 16 * h0;
        uint64_t ro = rows.place(h0, so);
        if constexpr (CPR % 4 != 0) {
          uint32_t so1;
          const uint64_t ro1 = rows.place(h1, so1);
          if (r >= 16 * h1) {
            rr = r - 16 * h1;
            ro = ro1;
            so = so1;
          }
        }
        kraw[u] = *reinterpret_cast<const u32x4*>(c.k + ro + rr * rows.kRow + 16 * col);
        vraw[u] = *reinterpret_cast<const u32x4*>(c.v + ro + rr * rows.kRow + 16 * col);
        if constexpr (I8) {
          kd[u] = reinterpret_cast<const half_t*>(c.k + ro + so + rr * (DD / 16))[col / 2];
          vd[u] = reinterpret_cast<const half_t*>(c.v + ro + so + rr * (DD / 16))[col / 2];
        }
      }
    }
  };
  auto stage = [&](uint64_t seen, auto open_c, int par, int buf) {
    constexpr bool OPEN = decltype(open_c)::value;
    bool bad = false;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int ch = tid + 256 * u;
      if (64 * CPR % 256 != 0 && ch >= 64 * CPR) break;
      const int r = ch / CPR, col = ch % CPR;
      half8 kx[VC / 8], vx[VC / 8];
      if constexpr (I8) {
        kx[0] = dequant8(uint2{kraw[u][0], kraw[u][1]}, kd[u]);
        kx[1] = dequant8(uint2{kraw[u][2], kraw[u][3]}, kd[u]);
        vx[0] = dequant8(uint2{vraw[u][0], vraw[u][1]}, vd[u]);
        vx[1] = dequant8(uint2{vraw[u][2], vraw[u][3]}, vd[u]);
      } else {
        kx[0] = __builtin_bit_cast(half8, kraw[u]);
        vx[0] = __builtin_bit_cast(half8, vraw[u]);
      }
#pragma unroll
      for (int e = 0; e < VC / 8; ++e) {
        if constexpr (!OPEN) {
          if (!((seen >> r) & 1)) vx[e] = half8{};
          bad = bad || any_not_finite(vx[e]);
        }
        *reinterpret_cast<half8*>(ks + buf + r * KP + VC * col + 8 * e) = kx[e];
        *reinterpret_cast<half8*>(vs + buf + r * VP + VC * col + 8 * e) = vx[e];
      }
    }
    if (!OPEN && bad) tile_bad[par] = 1;
  };
  const half_t* const vtr = vs + (4 * hf + (lane & 15) / 4) * VP + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);

  // The running maximum for scores whose largest is `top`, and the weights in place of
  // the scores, rounded to f16 in pairs and summed as rounded.
  f32x16 sc[2];
  half8 pb[2][2];
  auto rescale = [&](float top) {
    if (__ballot(top > m + kLagLog2) == 0) return;  // uniform
    const float mn = fmaxf(m, top);
    const float corr = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
    l *= corr;
#pragma unroll
    for (int d = 0; d < DB; ++d) ot[d] *= corr;
    m = mn;
    mb = exponent_base(m, kWeightLog2);
  };
  auto weights = [&]() {
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
          sc[j][i + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[j][i + e], c.scale_log2, -mb));
        const half2v h = __builtin_convertvector(float2s{sc[j][i], sc[j][i + 1]}, half2v);
        pb[j][i / 8][i % 8] = h[0];
        pb[j][i / 8][i % 8 + 1] = h[1];
        sum = __builtin_amdgcn_fdot2(h, half2v{(half_t)1.f, (half_t)1.f}, sum, false);
      }
    l += sum2(sum);
  };
  auto value_op = [&](int buf, int j, int k, int d) {
    const uint2 lo = read_tr(vtr + buf + (32 * j + 16 * k) * VP + 32 * d);
    const uint2 hi = read_tr(vtr + buf + (32 * j + 16 * k + 8) * VP + 32 * d);
    return __builtin_bit_cast(half8, u32x4{lo.x, lo.y, hi.x, hi.y});
  };

  // An open tile.  The operands of the next eight MFMAs are under way from LDS while
  // the current four are issued, and the first values before the softmax: left to
  // itself the compiler reads each just before its use (2048 rows behind 6144 keys,
  // two sequences, 32 heads of 128: 677 us, 622 with four ahead, 600 with eight).
  const half_t* const krow = ks + n * KP + 8 * hf;
  auto open_tile = [&](int buf) {
    half8 a[3][4];
    auto keys = [&](int ch) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        a[ch % 3][q] = *reinterpret_cast<const half8*>(krow + buf + 32 * (q & 1) * KP + 16 * (2 * ch + q / 2));
    };
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[j][i] = 0.f;
    keys(0);
    keys(1);
#pragma unroll
    for (int ch = 0; ch < KS / 2; ++ch) {
      if (ch + 2 < KS / 2) keys(ch + 2);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int q = 0; q < 4; ++q)
        sc[q & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[ch % 3][q], qb[2 * ch + q / 2], sc[q & 1], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    half8 av[3][DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      av[0][d] = value_op(buf, 0, 0, d);
      av[1][d] = value_op(buf, 0, 1, d);
    }
    __builtin_amdgcn_sched_barrier(0);
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, sc[j][i]);
    rescale(max2(top) * c.scale_log2);
    weights();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int ch = 0; ch < 4; ++ch) {
      if (ch < 2)
#pragma unroll
        for (int d = 0; d < DB; ++d) av[(ch + 2) % 3][d] = value_op(buf, (ch + 2) / 2, (ch + 2) % 2, d);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int d = 0; d < DB; ++d)
        ot[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(av[ch % 3][d], pb[ch / 2][ch % 2], ot[d], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // A tile with masked pairs or keys without a row.
  auto masked_tile = [&](int t0, uint64_t seen, int par) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[j][i] = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (s % 2 == 0 && j == 0) __builtin_amdgcn_sched_barrier(0);  // bounds the operands that are held at once
        const half8 a = *reinterpret_cast<const half8*>(krow + 32 * j * KP + 16 * s);
        sc[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qb[s], sc[j], 0, 0, 0);
      }
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int k = 32 * j + 8 * (i / 4) + 4 * hf + i % 4;
        if (!((seen >> k) & 1) || t0 + k > pos) sc[j][i] = -INFINITY;
        top = fmaxf(top, sc[j][i]);
      }
    rescale(max2(top) * c.scale_log2);
    weights();
    if (!tile_bad[par]) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int d = 0; d < DB; ++d)
            ot[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(value_op(0, j, k, d), pb[j][k], ot[d], 0, 0, 0);
        }
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int i = 0; i < 16; ++i) ps[w][8 * (i / 4) + 4 * hf + i % 4][n] = sc[j][i];
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 1
        for (int k = 0; k < 32; ++k) {
          if (!((seen >> (32 * j + k)) & 1) || t0 + 32 * j + k > pos) continue;
          const float p = ps[w][k][n];
#pragma unroll
          for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              if (i % 8 == 0) __builtin_amdgcn_sched_barrier(0);
              ot[d][i] += p * (float)vs[(32 * j + k) * VP + 32 * d + 8 * (i / 4) + 4 * hf + i % 4];
            }
        }
      }
    }
  };

  if (tid == 0) tile_bad[0] = tile_bad[1] = 0;
  int t0 = begin;  // the tile in the registers
  if (t0 < end) {
    rows.look(t0);
    rows.take(t0);
    fetch();
    if (t0 + 64 < end) rows.look(t0 + 64);
  }
  auto next = [&]() {
    t0 += 64;
    if (t0 >= end) return;
    rows.take(t0);
    fetch();
    if (t0 + 64 < end) rows.look(t0 + 64);
  };
  // The open tiles come first: those that every row of the workgroup sees whole, up to
  // the first that has a hole.  While one is computed from its buffer, the next is
  // staged into the other and the one after that is loaded.  Two loops, as one with
  // both kinds of tile does not fit the registers.
  auto open = [&]() { return t0 < end && rows.have() == ~0ull && t0 + 63 <= pos_lo; };  // uniform
  if (open()) {
    stage(~0ull, std::true_type{}, 0, 0);
    next();
    __syncthreads();
    for (int buf = 0;; buf = BUF - buf) {
      const bool more = open();
      if (more) {
        stage(~0ull, std::true_type{}, 0, BUF - buf);
        next();
      }
      if (wave_live) open_tile(buf);
      __syncthreads();
      if (!more) break;
    }
  }
  for (int par = 0; t0 < end; par ^= 1) {
    __syncthreads();  // the previous tile's readers are done
    // the other parity's flag was last read before this barrier and is set again
    // only behind the next tile's first barrier
    if (tid == 0) tile_bad[par ^ 1] = 0;
    const uint64_t seen = rows.have();
    stage(seen, std::false_type{}, par, 0);
    __syncthreads();
    if (wave_live && t0 <= w_hi) masked_tile(t0, seen, par);  // uniform
    next();
  }

  if (!wave_live || r0 + n >= t.rows) return;
  if (ns == 1) {
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    half_t* o = static_cast<half_t*>(c.out) + orow * DD;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        half2v a = {(half_t)(ot[d][4 * q] * inv), (half_t)(ot[d][4 * q + 1] * inv)};
        half2v b = {(half_t)(ot[d][4 * q + 2] * inv), (half_t)(ot[d][4 * q + 3] * inv)};
        *reinterpret_cast<uint2*>(o + 32 * d + 8 * q + 4 * hf) =
            uint2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
      }
  } else {
    const uint64_t p = orow * c.splits + sp;
    if (hf == 0) *reinterpret_cast<float2s*>(c.ml + 2 * p) = float2s{m, l};
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<float4v*>(c.acc + p * DD + 32 * d + 8 * q + 4 * hf) =
            float4v{ot[d][4 * q], ot[d][4 * q + 1], ot[d][4 * q + 2], ot[d][4 * q + 3]};
  }
}

// ---- f32 rows -----------------------------------------------------------------------
//
// The same two kernels on v_mfma_f32_16x16x4_f32, whose products and sums are
// those of f32 arithmetic; 8-bit codes become f32 exactly.  The MFMA takes one
// value per lane and operand, so the order in which dims (scores) and keys (P.V)
// are summed is free and every operand comes in 16-byte pieces:
//  * scores: k-step s of lane group g is dim DD/4 g + s, a lane's operand DD/4
//    consecutive elements of its key's row;
//  * P.V: the k-step over keys 16j + 4g + i takes the weight that the scores left
//    in lane (row, g) as element (j, i); row m of output block 4h + e is dim 64h +
//    4m + e, so a lane's operands are 4 consecutive elements of one value row, and
//    it ends with 16 consecutive dims per h.  (DD = 96: half of the second h is
//    not there; its columns are computed and dropped.)

// Eight codes and four codes as f32.
__device__ __forceinline__ void codes8_f32(uint2 w, float d, float* x) {
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = d * (float)(int)(int8_t)((e < 4 ? w.x : w.y) >> (8 * (e & 3)));
}
__device__ __forceinline__ float4v codes4_f32(uint32_t w, float d) {
  return float4v{d * (float)(int)(int8_t)w, d * (float)(int)(int8_t)(w >> 8), d * (float)(int)(int8_t)(w >> 16),
                 d * (float)(int)(int8_t)(w >> 24)};
}

// One row's output or partial, from the layout above.
template <int DD>
__device__ __forceinline__ void store_f32(const Chunk& c, uint64_t orow, uint32_t sp, uint32_t ns, int g, float m, float l,
                                          const float4v* ot) {
  float* dst = ns == 1 ? static_cast<float*>(c.out) + orow * DD : c.acc + (orow * c.splits + sp) * DD;
  const float f = ns > 1 ? 1.0f : l == 0.f ? 0.f : 1.0f / l;
  if (ns > 1 && g == 0) *reinterpret_cast<float2s*>(c.ml + 2 * (orow * c.splits + sp)) = float2s{m, l};
#pragma unroll
  for (int h = 0; h < (DD + 63) / 64; ++h)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (64 * h + 16 * g < DD)
        *reinterpret_cast<float4v*>(dst + 64 * h + 16 * g + 4 * r) =
            float4v{ot[4 * h][r] * f, ot[4 * h + 1][r] * f, ot[4 * h + 2][r] * f, ot[4 * h + 3][r] * f};
}

// Few query rows: 16 a workgroup, its waves take 32-key tiles in turn; K and V go
// from the cache straight into the operands, no LDS before the merge.  A tile
// with a masked pair and a value that is not finite reads the values again, row by
// row, for the pairs that count.  Bound by HBM (8 sequences of up to 4096 positions,
// 8 KV heads of 128: 49 us), at short caches by its latency (one of 101: 6.6 us).
template <PoolType PT, int DD, bool UNI>
__global__ __launch_bounds__(256, 2) void chunk_narrow_f32_kernel(Chunk c) {
  constexpr bool I8 = PT == PoolType::I8;
  constexpr int DG = DD / 4, NH = (DD + 63) / 64, NB = 4 * NH;
  __shared__ __attribute__((aligned(16))) float merge[4][16 * 64 * NH];
  __shared__ float wm[4][16], wl[4][16];
  const uint32_t sp = blockIdx.x % c.splits, kvh = blockIdx.y;
  RowTile t;
  if (!find_tile(c.b, blockIdx.x / c.splits, c.group, 16, c.lo, c.hi, t)) return;
  const uint32_t ns = splits_of(c, t.len);
  if (sp >= ns) return;
  const uint32_t G = c.group, H = c.n_heads;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t last = (t.first + 16 < t.rows ? t.first + 16 : t.rows) - 1;
  const int pos_lo = t.pos0 + (int)(t.first / G), pos_hi = t.pos0 + (int)(last / G);
  const int begin = (int)(sp * c.keys_per_split);
  int end = pos_hi + 1 < t.len ? pos_hi + 1 : t.len;
  if (end > begin + (int)c.keys_per_split) end = begin + (int)c.keys_per_split;
  end = __builtin_amdgcn_readfirstlane(end);
  const uint32_t row = t.first + n < t.rows ? t.first + n : t.rows - 1;
  const uint64_t orow = (uint64_t)(t.start + row / G) * H + kvh * G + row % G;
  const int pos = t.pos0 + (int)(row / G);

  float qb[DG];
#pragma unroll
  for (int s = 0; s < DG / 4; ++s) {
    const float4v x = *reinterpret_cast<const float4v*>(static_cast<const float*>(c.q) + orow * DD + DG * g + 4 * s);
#pragma unroll
    for (int e = 0; e < 4; ++e) qb[4 * s + e] = x[e];
  }
  float4v ot[NB];
#pragma unroll
  for (int d = 0; d < NB; ++d) ot[d] = float4v{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;

  float4v kf[2][I8 ? 1 : DG / 4], vf[2][4][I8 ? 1 : NH];
  uint2 kc[2][I8 ? DG / 8 : 1];
  half_t kd[2][I8 ? DG / 8 : 1], vd[2][4][NH];
  uint32_t vc[2][4][NH];
  Rows<PT, DD, 2, UNI> rows(c.b, t.seq, kvh, end);
  auto fetch_k = [&]() {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint8_t* kr = rows.row(c.k, j, n);
      if constexpr (I8) {
        const half_t* sc = rows.scale(c.k, j, n);
#pragma unroll
        for (int p = 0; p < DG / 8; ++p) {
          kc[j][p] = *reinterpret_cast<const uint2*>(kr + DG * g + 8 * p);
          kd[j][p] = sc[(DG * g + 8 * p) / 32];
        }
      } else {
#pragma unroll
        for (int p = 0; p < DG / 4; ++p) kf[j][p] = *reinterpret_cast<const float4v*>(kr + 4 * (DG * g + 4 * p));
      }
    }
  };
  auto fetch_v = [&]() {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t* vr = rows.row(c.v, j, 4 * g + i);
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          const int d = 64 * h + 4 * n < DD ? 64 * h + 4 * n : 0;
          if constexpr (I8) {
            vc[j][i][h] = *reinterpret_cast<const uint32_t*>(vr + d);
            vd[j][i][h] = rows.scale(c.v, j, 4 * g + i)[d / 32];
          } else {
            vf[j][i][h] = *reinterpret_cast<const float4v*>(vr + 4 * d);
          }
        }
      }
  };

  int t0 = begin + 32 * w;
  if (t0 < end) {
    rows.look(t0);
    rows.take(t0);
    fetch_k();
    fetch_v();
    if (t0 + 128 < end) rows.look(t0 + 128);
  }
  auto next = [&]() {
    if (t0 + 128 >= end) return;
    rows.take(t0 + 128);
    fetch_k();
    if (t0 + 256 < end) rows.look(t0 + 256);
  };
  auto tile = [&](uint32_t seen, auto open_c) {
    constexpr bool OPEN = decltype(open_c)::value;
    float4v sc[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      sc[j] = float4v{0.f, 0.f, 0.f, 0.f};
      float a[DG];
      if constexpr (I8) {
#pragma unroll
        for (int p = 0; p < DG / 8; ++p) codes8_f32(kc[j][p], (float)kd[j][p], a + 8 * p);
      } else {
#pragma unroll
        for (int p = 0; p < DG; ++p) a[p] = kf[j][p / 4][p % 4];
      }
#pragma unroll
      for (int s = 0; s < DG; ++s) sc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], qb[s], sc[j], 0, 0, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (OPEN) next();
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = 16 * j + 4 * g + i;
        if (!OPEN && (!((seen >> k) & 1) || t0 + k > pos)) sc[j][i] = -INFINITY;
        top = fmaxf(top, sc[j][i]);
      }
    top = max4(top) * c.scale_log2;
    if (__ballot(top > m + kLagLog2) != 0) {  // uniform
      const float mn = fmaxf(m, top);
      const float corr = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      l *= corr;
#pragma unroll
      for (int d = 0; d < NB; ++d) ot[d] *= corr;
      m = mn;
    }
    const float mb = exponent_base(m, 0.f);
    float pv[2][4], sum = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        pv[j][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[j][i], c.scale_log2, -mb));
        sum += pv[j][i];
      }
    l += sum4(sum);
    // a key's values, zeros without a row
    auto value = [&](int j, int i, int h) {
      float4v x;
      if constexpr (I8) x = codes4_f32(vc[j][i][h], (float)vd[j][i][h]);
      else x = vf[j][i][h];
      if (!OPEN && !((seen >> (16 * j + 4 * g + i)) & 1)) x = float4v{0.f, 0.f, 0.f, 0.f};
      return x;
    };
    bool alu = false;
    if constexpr (!OPEN) {
      // (again: they do not fit the registers beside the rest of a masked tile)
      __builtin_amdgcn_sched_barrier(0);
      fetch_v();
      bool bad = false;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int h = 0; h < NH; ++h) {
            const float4v x = value(j, i, h);
#pragma unroll
            for (int e = 0; e < 4; ++e) bad = bad || !__builtin_isfinite(x[e]);
          }
      alu = __ballot(bad) != 0;
    }
    if (!alu) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int h = 0; h < NH; ++h) {
            const float4v x = value(j, i, h);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              ot[4 * h + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], pv[j][i], ot[4 * h + e], 0, 0, 0);
          }
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll 1
          for (int gk = 0; gk < 4; ++gk) {
            const int k = 16 * j + 4 * gk + i;
            const float p = __shfl(pv[j][i], 16 * gk + n);
            const uint32_t slot = (uint32_t)(t0 + k) % c.b.block_size;
            const uint8_t* page = rows.row(c.v, j, 4 * gk + i) - (uint64_t)slot * rows.kRow;
            if (!((seen >> k) & 1) || t0 + k > pos) continue;
#pragma unroll
            for (int d = 0; d < NB; ++d)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                if (d % 2 == 0 && r == 0) __builtin_amdgcn_sched_barrier(0);
                const uint32_t dim = 64 * (d / 4) + 16 * g + 4 * r + d % 4;
                if (dim < DD) ot[d][r] += p * page_value<PT>(c.b, page, slot, dim);
              }
          }
    }
    if (!OPEN) next();
    // a tile of values and the next one's do not fit the registers together
    __builtin_amdgcn_sched_barrier(0);
    if (OPEN && t0 + 128 < end) fetch_v();
  };
  // The open tiles first, as in the f16 kernel.
  while (t0 < end && (uint32_t)rows.have() == ~0u && t0 + 31 <= pos_lo) {  // uniform
    tile(~0u, std::true_type{});
    t0 += 128;
  }
  while (t0 < end) {
    tile((uint32_t)rows.have(), std::false_type{});
    t0 += 128;
  }

  if (g == 0) {
    wm[w][n] = m;
    wl[w][n] = l;
  }
  // row n of the wave: dim order of the registers, 4 floats (d = 4h .. 4h + 3, r) at a time
#pragma unroll
  for (int h = 0; h < NH; ++h)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      *reinterpret_cast<float4v*>(&merge[w][(n * NH + h) * 64 + 16 * g + 4 * r]) =
          float4v{ot[4 * h][r], ot[4 * h + 1][r], ot[4 * h + 2][r], ot[4 * h + 3][r]};
  __syncthreads();
  for (int idx = tid; idx < 16 * DD / 4; idx += 256) {
    const int r = idx / (DD / 4), d = idx % (DD / 4) * 4;
    const uint32_t qr = t.first + r;
    if (qr >= t.rows) break;
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int v = 0; v < 4; ++v) M = fmaxf(M, wm[v][r]);
    float4v A = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const float f = wm[v][r] == M ? 1.f : __builtin_amdgcn_exp2f(wm[v][r] - M);
      L += f * wl[v][r];
      A += f * *reinterpret_cast<const float4v*>(&merge[v][r * NH * 64 + d]);
    }
    const uint64_t o = (uint64_t)(t.start + qr / G) * H + kvh * G + qr % G;
    if (ns == 1) {
      const float inv = L == 0.f ? 0.f : 1.0f / L;
      *reinterpret_cast<float4v*>(static_cast<float*>(c.out) + o * DD + d) = A * inv;
    } else {
      const uint64_t p = o * c.splits + sp;
      if (d == 0) *reinterpret_cast<float2s*>(c.ml + 2 * p) = float2s{M, L};
      *reinterpret_cast<float4v*>(c.acc + p * DD + d) = A;
    }
  }
}

// Many query rows: 64 a workgroup, 16 per wave, 32-key tiles of K and V in LDS.
// Bound by the f32 MFMA, busy 55 % of the cycles, and the waits between: one buffer and two
// barriers a tile, few row tiles of unlike length, bank conflicts in 7 % of the cycles.
// Two sequences of 512 tokens with 2048 positions, 32 heads of 128, 293 us; three of up
// to 389 with 2000, 32 heads of 64, 9.5 GFLOP in 117 us with the combine (13 of them),
// where a product of 8192 in each size reaches 153 TFLOP/s.
template <PoolType PT, int DD, bool UNI>
__global__ __launch_bounds__(256, 2) void chunk_wide_f32_kernel(Chunk c) {
  constexpr bool I8 = PT == PoolType::I8;
  constexpr int TK = 32, DP = DD + 4, DG = DD / 4, NH = (DD + 63) / 64, NB = 4 * NH;
  constexpr int EC = I8 ? 8 : 4;                  // elements per chunk (8 or 16 bytes)
  constexpr int CPR = DD / EC, NU = (TK * CPR + 255) / 256;
  static_assert(CPR % 4 == 0, "a wave's 64 chunks of a tile lie in one group of 16 keys");
  __shared__ __attribute__((aligned(16))) float ks[TK * DP];
  __shared__ __attribute__((aligned(16))) float vs[TK * DP + 64 * NH - DD];
  __shared__ __attribute__((aligned(16))) float ps[4][TK][16];
  __shared__ int tile_bad[2];
  uint32_t kvh, idx;
  if (!wide_tile(c, kvh, idx)) return;
  const uint32_t sp = blockIdx.y;
  RowTile t;
  if (!find_tile(c.b, idx, c.group, 64, c.lo, c.hi, t)) return;
  const uint32_t ns = splits_of(c, t.len);
  if (sp >= ns) return;
  const uint32_t G = c.group, H = c.n_heads;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t last = (t.first + 64 < t.rows ? t.first + 64 : t.rows) - 1;
  const int pos_lo = t.pos0 + (int)(t.first / G), pos_hi = t.pos0 + (int)(last / G);
  const int begin = (int)(sp * c.keys_per_split);
  int end = pos_hi + 1 < t.len ? pos_hi + 1 : t.len;
  if (end > begin + (int)c.keys_per_split) end = begin + (int)c.keys_per_split;
  end = __builtin_amdgcn_readfirstlane(end);
  const uint32_t r0 = t.first + 16 * w;
  const bool wave_live = r0 < t.rows;
  const uint32_t row = r0 + n < t.rows ? r0 + n : t.rows - 1;
  const uint64_t orow = (uint64_t)(t.start + row / G) * H + kvh * G + row % G;
  const int pos = t.pos0 + (int)(row / G);
  const int w_hi = __builtin_amdgcn_readfirstlane(t.pos0 + (int)((r0 + 15 < t.rows ? r0 + 15 : t.rows - 1) / G));
  float qb[DG];
#pragma unroll
  for (int s = 0; s < DG / 4; ++s) {
    const float4v x = *reinterpret_cast<const float4v*>(static_cast<const float*>(c.q) + orow * DD + DG * g + 4 * s);
#pragma unroll
    for (int e = 0; e < 4; ++e) qb[4 * s + e] = x[e];
  }
  float4v ot[NB];
#pragma unroll
  for (int d = 0; d < NB; ++d) ot[d] = float4v{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;

  float4v kf[I8 ? 1 : NU], vf[I8 ? 1 : NU];
  uint2 kc[I8 ? NU : 1], vc[I8 ? NU : 1];
  half_t kd[NU], vd[NU];
  Rows<PT, DD, 2, UNI> rows(c.b, t.seq, kvh, end);
  auto fetch = [&]() {
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int ch = tid + 256 * u < TK * CPR ? tid + 256 * u : TK * CPR - 1;
      const int r = ch / CPR, col = ch % CPR;
      auto get = [&](const uint8_t* kr, const uint8_t* vr, const half_t* ksc, const half_t* vsc) {
        if constexpr (I8) {
          kc[u] = *reinterpret_cast<const uint2*>(kr + 8 * col);
          vc[u] = *reinterpret_cast<const uint2*>(vr + 8 * col);
          kd[u] = ksc[col / 4];
          vd[u] = vsc[col / 4];
        } else {
          kf[u] = *reinterpret_cast<const float4v*>(kr + 16 * col);
          vf[u] = *reinterpret_cast<const float4v*>(vr + 16 * col);
        }
      };
      if constexpr (!UNI) {
        get(rows.row(c.k, 0, r), rows.row(c.v, 0, r), rows.scale(c.k, 0, r), rows.scale(c.v, 0, r));
      } else {  // a wave's 64 lie in one group of 16 keys
        const bool whole = 16 * CPR % 256 == 0;  // the workgroup's 256 do
        const int h = whole ? 256 * u / (16 * CPR) : min(w + 4 * u, TK * CPR / 64 - 1) / (CPR / 4);
        uint32_t so = whole ? rows.scales[h] : 0;
        const uint64_t ro = whole ? rows.base[h] : rows.place(h, so);
        const uint32_t rr = r - 16 * h, sr = so + rr * (DD / 16);
        get(c.k + ro + rr * rows.kRow, c.v + ro + rr * rows.kRow, reinterpret_cast<const half_t*>(c.k + ro + sr),
            reinterpret_cast<const half_t*>(c.v + ro + sr));
      }
    }
  };
  auto stage = [&](uint32_t seen, bool closed, int par) {
    bool bad = false;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int ch = tid + 256 * u;
      if (TK * CPR % 256 != 0 && ch >= TK * CPR) break;
      const int r = ch / CPR, col = ch % CPR;
      float kx[EC], vx[EC];
      if constexpr (I8) {
        codes8_f32(kc[u], (float)kd[u], kx);
        codes8_f32(vc[u], (float)vd[u], vx);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          kx[e] = kf[u][e];
          vx[e] = vf[u][e];
        }
      }
#pragma unroll
      for (int e = 0; e < EC; ++e)
        if (closed) {
          if (!((seen >> r) & 1)) vx[e] = 0.f;
          bad = bad || !__builtin_isfinite(vx[e]);
        }
#pragma unroll
      for (int e = 0; e < EC; e += 4) {
        *reinterpret_cast<float4v*>(ks + r * DP + EC * col + e) = float4v{kx[e], kx[e + 1], kx[e + 2], kx[e + 3]};
        *reinterpret_cast<float4v*>(vs + r * DP + EC * col + e) = float4v{vx[e], vx[e + 1], vx[e + 2], vx[e + 3]};
      }
    }
    if (bad) tile_bad[par] = 1;
  };
  auto tile = [&](int t0, uint32_t seen, int par, auto open_c) {
    constexpr bool OPEN = decltype(open_c)::value;
    float4v sc[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      sc[j] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int p = 0; p < DG / 4; ++p) {
        const float4v a = *reinterpret_cast<const float4v*>(ks + (16 * j + n) * DP + DG * g + 4 * p);
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], qb[4 * p + e], sc[j], 0, 0, 0);
      }
    }
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (!OPEN) {
          const int k = 16 * j + 4 * g + i;
          if (!((seen >> k) & 1) || t0 + k > pos) sc[j][i] = -INFINITY;
        }
        top = fmaxf(top, sc[j][i]);
      }
    top = max4(top) * c.scale_log2;
    if (__ballot(top > m + kLagLog2) != 0) {  // uniform
      const float mn = fmaxf(m, top);
      const float corr = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      l *= corr;
#pragma unroll
      for (int d = 0; d < NB; ++d) ot[d] *= corr;
      m = mn;
    }
    const float mb = exponent_base(m, 0.f);
    float pv[2][4], sum = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        pv[j][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[j][i], c.scale_log2, -mb));
        sum += pv[j][i];
      }
    l += sum4(sum);
    if (OPEN || !tile_bad[par]) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int h = 0; h < NH; ++h) {
            const float4v a = *reinterpret_cast<const float4v*>(vs + (16 * j + 4 * g + i) * DP + 4 * n + 64 * h);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              ot[4 * h + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], pv[j][i], ot[4 * h + e], 0, 0, 0);
          }
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) ps[w][16 * j + 4 * g + i][n] = pv[j][i];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      for (int k = 0; k < TK; ++k) {
        if (!((seen >> k) & 1) || t0 + k > pos) continue;
        const float p = ps[w][k][n];
#pragma unroll
        for (int d = 0; d < NB; ++d)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int dim = 64 * (d / 4) + 16 * g + 4 * r + d % 4;
            if (dim < DD) ot[d][r] += p * vs[k * DP + dim];
          }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  };

  if (tid == 0) tile_bad[0] = tile_bad[1] = 0;
  int t0 = begin;
  if (t0 < end) {
    rows.look(t0);
    rows.take(t0);
    fetch();
    if (t0 + TK < end) rows.look(t0 + TK);
  }
  auto next = [&]() {
    if (t0 + TK >= end) return;
    rows.take(t0 + TK);
    fetch();
    if (t0 + 2 * TK < end) rows.look(t0 + 2 * TK);
  };
  // The open tiles first, as in the f16 kernel.
  while (t0 < end && (uint32_t)rows.have() == ~0u && t0 + TK - 1 <= pos_lo) {  // uniform
    __syncthreads();  // the previous tile's readers are done
    stage(~0u, false, 0);
    __syncthreads();
    next();
    tile(t0, ~0u, 0, std::true_type{});
    t0 += TK;
  }
  for (int par = 0; t0 < end; t0 += TK, par ^= 1) {
    __syncthreads();
    if (tid == 0) tile_bad[par ^ 1] = 0;
    const uint32_t seen = (uint32_t)rows.have();
    stage(seen, true, par);
    __syncthreads();
    if (wave_live && t0 <= w_hi) tile(t0, seen, par, std::false_type{});  // uniform
    next();
  }
  if (wave_live && r0 + n < t.rows) store_f32<DD>(c, orow, sp, ns, g, m, l, ot);
}

// ---- launch ------------------------------------------------------------------------------

// Query rows of a sequence, on average, up to which the narrow kernel takes the whole
// batch.  It reads the cache once per 16 or 32 rows and splits it finely; the wide one
// once per 128 (f32: 64).  Narrow and wide, 8 sequences of 4096 positions, 8 KV heads
// of 128:
//   f16, 64 rows 52 and 70 us, 96 rows 70 and 63;
//   I8,  64 rows 37 and 45 us, 96 rows 51 and 44;
//   f32, 36 rows 144 and 100 us, 64 rows 155 and 111; one of 8192, 32 rows: 28 and 33.
template <typename T>
constexpr uint32_t kNarrowRows = std::is_same<T, float>::value ? 32 : 64;
// Where the wide kernel runs, the sequences that go to the narrow one all the same; more
// wait for a kernel with too few workgroups (three sequences of up to 96 rows: 42 us, and
// 54 with the narrow kernel taking those of up to 64).
constexpr uint32_t kFewRows = 32;

template <typename T, PoolType PT, int DD, bool UNI>
hipError_t chunk_mfma_at(const PagedBatch& b, uint32_t n_heads, const void* q, const void* kp, const void* vp, void* out,
                      const nfhip::Workspace& ws, hipStream_t s) {
  Chunk c{};
  c.b = b;
  c.q = q;
  c.k = static_cast<const uint8_t*>(kp);
  c.v = static_cast<const uint8_t*>(vp);
  c.out = out;
  c.n_heads = n_heads;
  c.group = n_heads / b.n_kv;
  c.scale_log2 = 1.4426950408889634f / sqrtf((float)DD);
  const uint64_t rows = (uint64_t)b.rows * c.group;  // query rows per KV head
  // Lengths are known on the device only: each kernel skips the sequences that are the
  // other's.
  const bool wide = rows > (uint64_t)kNarrowRows<T> * b.n_seqs;
  const bool narrow = !wide || b.n_seqs > 1;
  constexpr bool F16 = std::is_same<T, half_t>::value;
  constexpr uint32_t kWideRows = F16 ? 128 : 64;  // a wide workgroup's query rows
  // A narrow workgroup takes 16 rows, or 32 where sequences have more, which then read
  // the cache once (16 I8 sequences of 20 rows behind up to 4096 positions, with the
  // append before it: 48 and 37 us; 64 sequences of 4 rows behind up to 8192, f16:
  // with 16 rows 262 us, with 32 279).
  const uint32_t nt = F16 && (wide || rows > 16ull * b.n_seqs) ? 2 : 1;
  const uint64_t per = wide ? kWideRows : 16 * nt, mean = (rows + b.n_seqs - 1) / b.n_seqs;
  const uint64_t most_tiles = rows / per + b.n_seqs;
  // Splits of the keys, with partials that fit the workspace.  Narrow: two workgroups per
  // CU, not one more (20 sequences of 4096 positions in I8: 41 us; rounded up, a third
  // of the CUs have a third workgroup, 50).  Wide: four where no sequence is cut short by
  // the mask or its length, rounded up (three ragged f32 chunks: 117 us, rounded down
  // 129, with two 129); none where the tiles alone are as many.
  const uint64_t units = b.n_seqs * ((mean + per - 1) / per) * b.n_kv;
  uint64_t splits = wide ? (1024 + units - 1) / units : units < 512 ? 512 / units : 1;
  // fewer keys a split, and reading the partials costs more than they save (one sequence of
  // 28 rows behind 8192 positions: 18 us, with 128 keys 22)
  const uint32_t min_keys = wide || nt == 2 ? 256 : 128;
  const uint64_t most = ws.part ? ws.part_floats / ((uint64_t)b.rows * n_heads * (DD + 4)) : 1;
  if (splits > most) splits = most ? most : 1;
  uint64_t keys = splits > 1 ? (b.limit + splits - 1) / splits : b.limit;
  keys = keys < min_keys ? min_keys : keys;
  keys = (keys + 127) / 128 * 128;
  c.keys_per_split = (uint32_t)keys;
  c.splits = (uint32_t)((b.limit + keys - 1) / keys);
  if (c.splits == 0) c.splits = 1;
  c.ml = ws.part;
  c.acc = ws.part + ((uint64_t)b.rows * n_heads * c.splits * 2 + 3) / 4 * 4;
  if (wide) {
    c.tiles = (uint32_t)most_tiles;
    c.lo = narrow ? kFewRows : 0;
    c.hi = ~0ull;
    const dim3 grid(wide_grid(c.tiles, b.n_kv), c.splits);
    if constexpr (F16) chunk_wide_kernel<PT, DD, UNI><<<grid, 256, 0, s>>>(c);
    else chunk_wide_f32_kernel<PT, DD, UNI><<<grid, 256, 0, s>>>(c);
  }
  if (narrow) {
    c.lo = 0;
    c.hi = wide ? kFewRows : ~0ull;
    c.tiles = (uint32_t)(wide ? b.n_seqs * (kFewRows / (16 * nt)) : most_tiles);
    const dim3 grid(c.splits * c.tiles, b.n_kv);
    if constexpr (!F16) chunk_narrow_f32_kernel<PT, DD, UNI><<<grid, 256, 0, s>>>(c);
    else if (nt == 2) chunk_narrow_kernel<PT, DD, 2, UNI><<<grid, 256, 0, s>>>(c);
    else chunk_narrow_kernel<PT, DD, 1, UNI><<<grid, 256, 0, s>>>(c);
  }
  if (c.splits > 1) {
    if (c.splits <= kFewSplits) chunk_combine_few_kernel<T, DD><<<dim3((b.rows * n_heads + 3) / 4), 256, 0, s>>>(c);
    else chunk_combine_kernel<T, DD><<<dim3(b.rows * n_heads), 256, 0, s>>>(c);
  }
  return hipGetLastError();
}

template <typename T, PoolType PT, int DD>
hipError_t chunk_mfma(const PagedBatch& b, uint32_t n_heads, const void* q, const void* kp, const void* vp, void* out,
                      const nfhip::Workspace& ws, hipStream_t s) {
  return b.block_size >= 16 && (b.block_size & (b.block_size - 1)) == 0 ? chunk_mfma_at<T, PT, DD, true>(b, n_heads, q, kp, vp, out, ws, s)
                                : chunk_mfma_at<T, PT, DD, false>(b, n_heads, q, kp, vp, out, ws, s);
}

template <typename T, PoolType PT>
hipError_t chunk(const PagedBatch& b, uint32_t n_heads, const void* q, const void* kp, const void* vp, void* out,
                 const nfhip::Workspace& ws, hipStream_t s) {
  const uintptr_t all = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(kp) |
                        reinterpret_cast<uintptr_t>(vp) | reinterpret_cast<uintptr_t>(out);
  // 16-byte rows: an I8 page of block_size head_dim 17/16 bytes has to be whole chunks
  if (all % 16 == 0 && n_heads % b.n_kv == 0 && b.blocks > 0 && b.limit > 0 &&
      (PT != PoolType::I8 || b.block_size * b.dim % 256 == 0)) {
    if (b.dim == 128) return chunk_mfma<T, PT, 128>(b, n_heads, q, kp, vp, out, ws, s);
    if (b.dim == 96) return chunk_mfma<T, PT, 96>(b, n_heads, q, kp, vp, out, ws, s);
    if (b.dim == 64) return chunk_mfma<T, PT, 64>(b, n_heads, q, kp, vp, out, ws, s);
  }
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
