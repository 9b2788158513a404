// paged_attention.hpp — kernels of attention of new tokens over a paged cache
// (flash_attention_paged_chunk, flash_attention_paged_prefix): row r of sequence
// s, at position pos, attends to positions 0 .. pos of its sequence,
//   o = sum_p exp(x_p - m) v_p / sum_p exp(x_p - m),  x_p = q . k_p / sqrt(dim),
// with m the running maximum of an online softmax.  Query head h reads KV head
// h * n_kv / n_heads.  A position without storage counts as no key; a row
// without any key gives zeros; rows of no sequence are left as they are.
// lse, where it is wanted: m + ln sum_p exp(x_p - m) of each row and head, -inf
// without a key.
#pragma once

#include <type_traits>

#include "paged.hpp"

namespace nfk {
namespace paged {

// Keys are split for two workgroups a CU.  Where a third fits, some CUs get it and others
// none: four long I8 sequences 216 us, kept to two 158.
#define NF_TWO_PER_CU __attribute__((amdgpu_flat_work_group_size(256, 256), amdgpu_waves_per_eu(2, 2)))

constexpr int kMaxDim = 256;
constexpr int kTile = 64;

// Any head_dim, head ratio and alignment.  A workgroup takes one (row, head);
// its four waves take 64-key tiles in turn: a lane scores one key, then the
// lanes lie over head_dim for the tile's 64 value rows, and the waves' (m, l,
// acc) are merged at the end.  Element loads, which every query head of a KV head
// makes again, and the vector ALU bound it: single tokens of 8 sequences of 4096
// positions with 32 query and 8 KV heads of 80 take 650 us in f16, where heads of 128
// on the MFMA kernel take 31.  SHARE: positions of the sequence's shared prefix are
// looked up in its group's table.
template <typename T, PoolType PT, bool SHARE>
__global__ __launch_bounds__(256) void chunk_any_kernel(PagedBatch b, PagedShared sh, uint32_t n_heads, float scale,
                                                        const T* __restrict__ q, const uint8_t* __restrict__ kp,
                                                        const uint8_t* __restrict__ vp, T* __restrict__ out,
                                                        float* __restrict__ lse) {
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
  const SharedPrefix pre = SHARE ? find_prefix(b, sh, seq) : SharedPrefix{seq, 0};
  float acc[R], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int r = 0; r < R; ++r) acc[r] = 0.0f;
  for (int64_t t0 = (int64_t)wave * kTile; t0 <= last; t0 += NW * kTile) {
    const int64_t p = t0 + lane;
    const uint32_t phys = p <= last ? find_block(b, SHARE && p < pre.len ? pre.seq : seq, p) : ~0u;
    float s = -INFINITY;
    if (phys != ~0u) {
      const uint8_t* page = kp + page_offset<PT>(b, phys, kvh);
      const uint32_t slot = (uint32_t)p % b.block_size;
      float dot = 0.0f;
      for (uint32_t d = 0; d < D; ++d) dot += qs[d] * row_value<T, PT>(b, page, slot, d);
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
        if (d < D) acc[r] += ps[wave][j] * row_value<T, PT>(b, page, slot, d);
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
  if (lse && threadIdx.x == 0) lse[(uint64_t)row * n_heads + h] = L == 0.0f ? -INFINITY : M + logf(L);
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
  // kShared:
  uint32_t pre;               // sequence whose table the shared positions are read through
  int shared;                 // shared positions
  uint32_t last;              // a group's rows: one past its last sequence; else 0
  uint32_t slot, splits;      // of the rows' partials this part's first one; splits of its keys
  uint32_t keys;              // keys of a split
  uint32_t base, stride;      // partials: query row (token, head) of the first, splits of each
  bool all;                   // every row of the group sees all shared positions
  bool wide;                  // of a part of many rows; `rows` is then the tile's end
};

// What a kernel serves: flash_attention_paged_chunk, the same with the rows'
// log-sum-exp, or flash_attention_paged_prefix (with it where it is wanted).
enum Form { kChunk, kLse, kShared };

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
  // kLse, kShared:
  float* lse;    // output, or null
  float* lsum;   // partials, f16: sum of the weights as they were before they were rounded
  // kShared (keys_per_split: the least):
  PagedShared sh;
  bool apart;       // the groups' shared keys are parts of their own
  uint32_t target;  // splits of a KV head's keys that are aimed at
  bool last_round;  // few parts, and partials of all rows do not fit: only the last sequences' keys may be cut
  uint64_t room;    // splits of query rows that do fit
  uint32_t* keys;   // Cuts, for the combination
  const uint2* items;       // large batches: (part, tile and split) of each workgroup, in turn,
  const struct Part* parts; // and the parts; else null
};

// Splits that a sequence of `len` positions takes.
__device__ __forceinline__ uint32_t splits_of(const Chunk& c, int len) {
  return len <= 0 ? 1u : ((uint32_t)len + c.keys_per_split - 1) / c.keys_per_split;
}

// The keys of a sequence with shared positions, as the tiles count them.  A tile lies on
// one side of the border `shared`, and starts at a multiple of 16: the shared keys count
// 0 .. shared - 1, the own ones follow at the next multiple of 64, from the last multiple
// of 16 that is not past the border (the keys between are masked).  Apart: no shared keys.
struct Border {
  int split, shift;  // count from which keys are own, and what is taken off it for the position
  int end;           // counts below it
};
__device__ __forceinline__ Border find_border(bool apart, int shared, int end) {
  if (end <= shared) return {0x7FFFFFFF, 0, apart || end < 0 ? 0 : end};
  const int split = apart ? 0 : (shared + 63) & ~63, shift = split - (shared & ~15);
  return {split, shift, end + shift};
}
// How keys are cut: a group's part into splits of `shared` keys, an own one of `own`; with
// last_round those of the sequences from `seq` on into `pieces`, whose rows begin at
// (token, head) `row`, the others not at all.
struct Cuts {
  uint32_t shared, own, seq, pieces, row;
};
// (A sequence behind `seq` whose rows begin before its, as descending STARTS make one, has
// no partials.)
__device__ __forceinline__ uint32_t own_keys(const Chunk& c, const Cuts& k, uint32_t seq, uint32_t start, int n) {
  if (!c.last_round) return k.own;
  return seq < k.seq || start * c.n_heads < k.row || n <= 0 ? c.keys_per_split : ((uint32_t)n / k.pieces + 64) / 64 * 64;
}
__device__ __forceinline__ Cuts load_cuts(const Chunk& c) { return {c.keys[0], c.keys[1], c.keys[2], c.keys[3], c.keys[4]}; }
__device__ __forceinline__ void store_cuts(const Chunk& c, const Cuts& k) {
  c.keys[0] = k.shared;
  c.keys[1] = k.own;
  c.keys[2] = k.seq;
  c.keys[3] = k.pieces;
  c.keys[4] = k.row;
}
// The first query row that has partials, and the splits of each.
__device__ __forceinline__ uint32_t first_row(const Chunk& c) { return c.last_round ? c.keys[4] : 0; }
__device__ __forceinline__ uint32_t stride_of(const Chunk& c) { return c.last_round ? c.keys[3] : c.splits; }
// Splits of the partials of a row: those of its group's part, then those of its own.
struct Slots {
  uint32_t group, own;
};
__device__ __forceinline__ uint32_t cut(int n, uint32_t keys) { return n <= 0 ? 1u : ((uint32_t)n + keys - 1) / keys; }
__device__ __forceinline__ Slots find_slots(const Chunk& c, const Cuts& k, uint32_t seq, uint32_t start, int shared, int len) {
  const uint32_t group = c.apart && shared > 0 ? cut(shared, k.shared) : 0;
  const int n = find_border(c.apart, shared, len).end;
  return {group, n <= 0 && group ? 0 : cut(n, own_keys(c, k, seq, start, n))};
}

// kShared: the batch as parts, first the groups' shared keys (where they are apart), then
// the sequences.
struct Part {
  uint32_t n, start;        // rows
  uint32_t seq, pre, last;  // as in RowTile
  int len, pos0, shared;
  int keys;                 // that its tiles count
  uint32_t group, splits;   // splits of its keys, and of its group's
  uint32_t all;
};
// Parts of up to FEW query rows are cut into tiles of NARROW, others into as few of up to WIDE
// as there have to be, of like heights: a workgroup of two full tiles is not beside one of
// two nearly empty ones (four groups of 160 rows, 128 and 32 of them a tile: 52 us).
template <uint32_t FEW, uint32_t NARROW, uint32_t WIDE>
struct Cut {
  static __device__ __forceinline__ uint32_t tiles(const Chunk& c, const Part& p) {
    const uint64_t rows = (uint64_t)p.n * c.group;
    return (uint32_t)(rows <= FEW ? (rows + NARROW - 1) / NARROW : (rows + WIDE - 1) / WIDE);
  }
  // The time of a tile's key, that of a narrow one's being 2/5 of a wide one's.
  static __device__ __forceinline__ float cost(const Chunk& c, const Part& p) {
    return (uint64_t)p.n * c.group <= FEW ? 0.4f : 1.f;
  }
  // And what a tile takes besides: finding it, its first keys, its partials; two tiles of 16
  // rows merge one after the other.
  static __device__ __forceinline__ float fixed(const Chunk& c, const Part& p) {
    return (uint64_t)p.n * c.group <= FEW && NARROW == 32 ? 500.f : 200.f;
  }
  // Tile and split k of a part.  All tiles of a split come after each other, so that they
  // share its keys in the caches.
  static __device__ __forceinline__ void tile(const Chunk& c, const Part& p, uint32_t nt, uint32_t k, const Cuts& keys, RowTile& t,
                                              uint32_t& sp) {
    t.keys = p.last ? keys.shared : own_keys(c, keys, p.seq, p.start, p.keys);
    t.base = c.last_round ? keys.row : 0;
    t.stride = c.last_round ? keys.pieces : c.splits;
    sp = k / nt;
    const uint32_t rows = p.n * c.group, wave = WIDE / 4;
    t.wide = rows > FEW;
    const uint32_t per = t.wide ? ((rows + nt - 1) / nt + wave - 1) / wave * wave : NARROW;
    t.first = (k - sp * nt) * per;
    t.rows = t.wide && t.first + per < rows ? t.first + per : rows;
    t.seq = p.seq;
    t.start = p.start;
    t.pos0 = p.pos0;
    t.len = p.len;
    t.pre = p.pre;
    t.shared = p.shared;
    t.last = p.last;
    t.slot = p.group;
    t.splits = p.splits;
    t.all = p.all != 0;
  }
};
// A sequence's part, but for its splits.
__device__ __forceinline__ Part sequence_part(const Chunk& c, uint32_t seq, int64_t a, int64_t z, int32_t l, const SharedPrefix& pre) {
  Part p{};
  if (a < 0 || z <= a || z > (int64_t)c.b.rows) return p;
  p.n = (uint32_t)(z - a);
  p.start = (uint32_t)a;
  p.seq = seq;
  p.pos0 = (int)((uint32_t)l - p.n);
  p.len = l < (int64_t)c.b.limit ? l : (int)c.b.limit;
  p.pre = pre.seq;
  p.shared = (int)pre.len;
  p.keys = find_border(c.apart, p.shared, p.len).end;
  return p;
}
// A group's: r0, r1 the first row of its first sequence and of the one behind its last.
__device__ __forceinline__ Part group_part(const Chunk& c, int32_t a, uint32_t last, int32_t len, int64_t r0, int64_t r1) {
  Part p{};
  if (r0 < 0) r0 = 0;
  if (r1 > (int64_t)c.b.rows) r1 = c.b.rows;
  if (r1 <= r0) return p;
  p.n = (uint32_t)(r1 - r0);
  p.start = (uint32_t)r0;
  p.seq = p.pre = (uint32_t)a;
  p.last = last;
  p.shared = p.len = p.keys = len < (int64_t)c.b.limit ? len : (int)c.b.limit;
  return p;
}
__device__ __forceinline__ bool good_group(const PagedBatch& b, int32_t a, int32_t z, int32_t len) {
  return a >= 0 && z > a && (uint32_t)a < b.n_seqs && len > 0;
}
__device__ __forceinline__ void cut_part(const Chunk& c, const Cuts& keys, Part& p) {
  p.group = 0;
  p.splits = cut(p.shared, keys.shared);
  if (p.last) return;
  const Slots s = find_slots(c, keys, p.seq, p.start, p.shared, p.len);
  p.group = s.group;
  p.splits = s.own;
}

// What the parts' tiles have to do, in keys of a wide tile.
struct Work {
  float shared = 0.f, own = 0.f;                // tiles times keys
  float shared_cost = 0.f, own_cost = 0.f;      // and their time
  float fixed = 0.f;                            // what own tiles take besides
  template <typename CUT>
  __device__ __forceinline__ void add(const Chunk& c, const Part& p) {
    if (p.keys <= 0 || p.n == 0) return;
    const float n = (float)CUT::tiles(c, p), w = n * (float)p.keys, cost = w * CUT::cost(c, p);
    if (p.last) {
      shared += w;
      shared_cost += cost;
    } else {
      own += w;
      own_cost += cost;
      fixed += n * CUT::fixed(c, p);
    }
  }
};
// The keys of a split; only the device knows the lengths.  With S workgroups at once, which
// `target` is for a KV head, split k keys take F + k in time, F = 200 (finding the tile, its
// first keys, its partials: 9 us, 64 keys 2.4), so W shared keys take W / k workgroups that
// long, which leaves the others the time (S - W / k)(F + k).  k is such that the own parts,
// B = own keys and what each tile takes besides, and a fifth more, as they do not fill it
// evenly, just fit:
//   S k^2 + (S F - W - B) k - W F = 0.
// Own keys are cut where their tile would take longer than that, into no more pieces than
// there are workgroups left.  (32 sequences with own parts of up to 1024 positions behind
// 32768 in I8, one head_dim of 128: all keys cut alike 54.8 us, without the fifth 52.7, so 49.6.)
__device__ __forceinline__ Cuts keys_of(const Chunk& c, const Work& w) {
  const float S = (float)c.target, F = 200.f;
  float shared = 0.f, own = w.own / S;
  if (w.shared > 0.f) {
    const float W = w.shared_cost, B = 1.2f * (w.own_cost + w.fixed), b = S * F - W - B;
    const float k = (__builtin_sqrtf(b * b + 4.f * S * W * F) - b) / (2.f * S);
    shared = k * (w.shared / W);
    own = w.own_cost > 0.f ? fmaxf(k * (w.own / w.own_cost), w.own / (fmaxf(S - W / k, 0.f) + 8.f)) : 0.f;
  }
  auto whole = [&](float k) {
    const uint32_t n = k < 1e9f ? ((uint32_t)k + 64) / 64 * 64 : 1u << 30;
    return n > c.keys_per_split ? n : c.keys_per_split;
  };
  return {whole(shared), whole(own), 0xFFFFFFFFu, 1, 0};
}
// With last_round: T tiles of a KV head are q rounds of the S workgroups at once and r more,
// which would take a round of their own.  The last sequences with r tiles between them are
// cut into as many pieces as still fit that round, which then takes 1 / pieces of one (16
// questions of up to 200 tokens behind 8192, 88 tiles, S 64: uncut 700 us, so 608, both before
// wide_rows()'s HINT).
constexpr uint32_t kMostPieces = 4;
__device__ __forceinline__ uint32_t more_tiles(const Chunk& c, uint32_t tiles) {
  return tiles > c.target ? tiles % c.target : 0;
}
__device__ __forceinline__ void cut_last(const Chunk& c, Cuts& k, uint32_t seq, uint32_t tiles, uint32_t token) {
  uint32_t n = tiles ? c.target / tiles : 1;
  if (n > kMostPieces) n = kMostPieces;
  while (n > 1 && (uint64_t)(c.b.rows - token) * c.n_heads * n > c.room) --n;
  if (n <= 1) return;
  k.seq = seq;
  k.pieces = n;
  k.row = token * c.n_heads;
}

// Tile and split `idx` of a KV head, for up to 128 parts and 64 groups: a lane looks at two
// parts, all loads in one round, which is the time that this takes (a search per sequence,
// 64 at a time: 4 us of 22 for 64 sequences behind 64 positions).
constexpr uint32_t kFewParts = 128, kFewGroups = 64;
template <typename CUT>
__device__ __forceinline__ bool find_few(const Chunk& c, uint32_t idx, RowTile& t, uint32_t& sp, Cuts& keys) {
  const PagedBatch& b = c.b;
  const int lane = threadIdx.x & 63;
  const uint32_t groups = c.apart ? c.sh.n_groups : 0;
  int32_t ga = 0, gz = 0, gl = 0;  // lane g: group g
  if ((uint32_t)lane < c.sh.n_groups) {
    ga = c.sh.first[lane];
    gz = c.sh.first[lane + 1];
    gl = c.sh.len[lane];
  }
  // Sequences are at parts groups .. groups + n_seqs - 1.
  int32_t a[2], z[2], l[2];
  uint32_t seq[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t e = 64 * i + lane;
    seq[i] = e - groups;
    a[i] = z[i] = l[i] = 0;
    if (e >= groups && seq[i] < b.n_seqs) {
      a[i] = b.starts[seq[i]];
      z[i] = b.starts[seq[i] + 1];
      l[i] = b.lens[seq[i]];
    }
  }
  // The group of each sequence, as find_prefix() has it: the first whose end is past it.
  SharedPrefix pre[2] = {{seq[0], 0}, {seq[1], 0}};
  bool found[2] = {false, false};
  for (uint32_t g = 0; g < c.sh.n_groups; ++g) {  // uniform
    const int32_t fa = __builtin_amdgcn_readlane(ga, (int)g), fz = __builtin_amdgcn_readlane(gz, (int)g);
    const int32_t n = __builtin_amdgcn_readlane(gl, (int)g);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (!found[i] && (int64_t)fz > (int64_t)seq[i]) {
        found[i] = true;
        if (fa >= 0 && (uint32_t)fa <= seq[i] && n > 0) pre[i] = {(uint32_t)fa, n < (int64_t)b.limit ? n : (int64_t)b.limit};
      }
  }
  Part p[2];
  Work work;
  // A group's rows, from the lanes of its sequences.
  const uint32_t last = (uint32_t)gz < b.n_seqs ? (uint32_t)gz : b.n_seqs;
  const bool good = (uint32_t)lane < groups && good_group(b, ga, gz, gl);
  const uint32_t e0 = good ? groups + (uint32_t)ga : 0, e1 = good ? groups + last - 1 : 0;
  const int32_t x0 = __shfl(a[0], (int)(e0 & 63)), x1 = __shfl(a[1], (int)(e0 & 63));
  const int32_t y0 = __shfl(z[0], (int)(e1 & 63)), y1 = __shfl(z[1], (int)(e1 & 63));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    p[i] = sequence_part(c, seq[i], a[i], z[i], l[i], pre[i]);
    if (i == 0 && good) p[i] = group_part(c, ga, last, gl, e0 < 64 ? x0 : x1, e1 < 64 ? y0 : y1);
    work.add<CUT>(c, p[i]);
  }
  work.shared = wave_sum(work.shared);
  work.own = wave_sum(work.own);
  work.shared_cost = wave_sum(work.shared_cost);
  work.own_cost = wave_sum(work.own_cost);
  work.fixed = wave_sum(work.fixed);
  keys = keys_of(c, work);
  keys.shared = (uint32_t)__builtin_amdgcn_readfirstlane((int)keys.shared);
  keys.own = (uint32_t)__builtin_amdgcn_readfirstlane((int)keys.own);
  if (c.last_round) {  // (all parts are sequences)
    uint32_t up[2], total = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      up[i] = CUT::tiles(c, p[i]);
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t v = __shfl_up(up[i], o);
        if (lane >= o) up[i] += v;
      }
      up[i] += total;
      total = (uint32_t)__builtin_amdgcn_readlane((int)up[i], 63);
    }
    const uint32_t more = more_tiles(c, total);
    auto from = [&](const Part& q, uint32_t before) {  // the last sequence that has `more` tiles from it on
      const uint32_t rest = total - before + CUT::tiles(c, q);
      const uint64_t has = __ballot(q.n > 0 && rest >= more);
      if (has == 0) return false;
      const int at = 63 - __builtin_clzll(has);
      auto of = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, at); };
      cut_last(c, keys, of(q.seq), of(rest), of(q.start));
      return true;
    };
    if (more && !from(p[1], up[1])) from(p[0], up[0]);
  }
  uint32_t done = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    cut_part(c, keys, p[i]);
    const uint32_t tiles = CUT::tiles(c, p[i]), mine = tiles * p[i].splits;
    uint32_t up = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t v = __shfl_up(up, o);
      if (lane >= o) up += v;
    }
    const uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)up, 63);
    if (idx - done < total) {
      const uint32_t k = idx - done;
      const int at = __builtin_ctzll(__ballot(up > k));
      auto of = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, at); };
      Part q;
      q.n = of(p[i].n);
      q.start = of(p[i].start);
      q.seq = of(p[i].seq);
      q.pre = of(p[i].pre);
      q.last = of(p[i].last);
      q.len = (int)of((uint32_t)p[i].len);
      q.pos0 = (int)of((uint32_t)p[i].pos0);
      q.shared = (int)of((uint32_t)p[i].shared);
      q.group = of(p[i].group);
      q.splits = of(p[i].splits);
      q.keys = (int)of((uint32_t)p[i].keys);
      bool all = true;
      if (q.last)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (p[j].last == 0 && p[j].n > 0 && p[j].seq >= q.seq && p[j].seq < q.last)
            all = all && (int64_t)p[j].pos0 + 1 >= (int64_t)q.shared;
      q.all = __ballot(!all) == 0;
      CUT::tile(c, q, of(tiles), k - of(up - mine), keys, t, sp);
      return true;
    }
    done += total;
  }
  return false;
}

// The same from what plan_kernel left.
template <typename CUT>
__device__ __forceinline__ bool find_planned(const Chunk& c, uint32_t idx, RowTile& t, uint32_t& sp) {
  if (idx >= c.keys[5]) return false;
  const uint2 it = c.items[idx];
  const Part p = c.parts[__builtin_amdgcn_readfirstlane((int)it.x)];
  CUT::tile(c, p, CUT::tiles(c, p), (uint32_t)__builtin_amdgcn_readfirstlane((int)it.y), load_cuts(c), t, sp);
  return true;
}

// Large batches: one workgroup writes the parts, and the part and the tile and split of
// each workgroup of the attention to come; keys[5]: workgroups of a KV head, at most `room`.
template <typename CUT>
__global__ __launch_bounds__(1024) void plan_kernel(Chunk c, Part* parts, uint2* items, uint32_t room) {
  __shared__ float sums[5][16];
  __shared__ uint32_t counts[16];
  const PagedBatch& b = c.b;
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t groups = c.apart ? c.sh.n_groups : 0, n = groups + b.n_seqs;
  Work work;
  for (uint32_t e = tid; e < n; e += 1024) {
    Part p{};
    if (e < groups) {
      const int32_t a = c.sh.first[e], z = c.sh.first[e + 1], len = c.sh.len[e];
      if (good_group(b, a, z, len)) {
        const uint32_t last = (uint32_t)z < b.n_seqs ? (uint32_t)z : b.n_seqs;
        p = group_part(c, a, last, len, b.starts[a], b.starts[last]);
        p.all = 1;  // unless a sequence finds otherwise
      }
    } else {
      const uint32_t seq = e - groups;
      p = sequence_part(c, seq, b.starts[seq], b.starts[seq + 1], b.lens[seq], find_prefix(b, c.sh, seq));
    }
    parts[e] = p;
    work.add<CUT>(c, p);
  }
  float* const of[5] = {&work.shared, &work.own, &work.shared_cost, &work.own_cost, &work.fixed};
#pragma unroll
  for (int j = 0; j < 5; ++j) {
    const float x = wave_sum(*of[j]);
    if (lane == 0) sums[j][wave] = x;
  }
  __syncthreads();  // and the parts
#pragma unroll
  for (int j = 0; j < 5; ++j) {
    *of[j] = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) *of[j] += sums[j][i];
  }
  const Cuts keys = keys_of(c, work);
  // A sequence that does not see all of its group's positions says so.
  if (groups)
    for (uint32_t e = groups + tid; e < n; e += 1024) {
      const Part& p = parts[e];
      if (p.n == 0 || p.shared == 0 || (int64_t)p.pos0 + 1 >= (int64_t)p.shared) continue;
      uint32_t lo = 0, hi = groups;  // its group, as in find_prefix()
      while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        if ((int64_t)c.sh.first[mid + 1] <= (int64_t)p.seq) lo = mid + 1;
        else hi = mid;
      }
      if (lo < groups) parts[lo].all = 0;
    }
  __syncthreads();
  uint32_t done = 0;
  for (uint32_t e0 = 0; e0 < n; e0 += 1024) {
    const uint32_t e = e0 + tid;
    uint32_t mine = 0;
    if (e < n) {
      Part p = parts[e];
      cut_part(c, keys, p);
      parts[e].group = p.group;
      parts[e].splits = p.splits;
      mine = CUT::tiles(c, p) * p.splits;
    }
    uint32_t up = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t v = __shfl_up(up, o);
      if ((int)lane >= o) up += v;
    }
    __syncthreads();
    if (lane == 63) counts[wave] = up;
    __syncthreads();
    uint32_t at = done + up - mine;
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i) {
      if (i < wave) at += counts[i];
      done += counts[i];
    }
    for (uint32_t k = 0; k < mine; ++k)
      if (at + k < room) items[at + k] = uint2{e, k};
  }
  if (tid == 0) {
    store_cuts(c, keys);
    c.keys[5] = done < room ? done : room;
  }
}

// The position of a row that sees all keys, of which a sequence in kShared has at most 2^30.
constexpr int kEverywhere = 0x3FFFFFFF;

// Position of a query row's token: of a group's rows, that in whatever sequence it is.
template <Form FORM>
__device__ __forceinline__ int row_pos(const PagedBatch& b, const RowTile& t, uint32_t token, bool all) {
  if (FORM != kShared || t.last == 0) return t.pos0 + (int)token;
  if (all) return kEverywhere;
  uint32_t seq;
  int64_t pos;
  return find_row(b, t.start + token, seq, pos) ? pos < kEverywhere ? (int)pos : kEverywhere : -1;
}

// The keys of a tile of rows, from its first row's token to its last's.
struct Keys {
  Border at;
  int lo;  // every row sees the positions up to it
  int hi;  // none sees one past it
};
template <Form FORM>
__device__ __forceinline__ Keys find_keys(const Chunk& c, const RowTile& t, uint32_t first_token, uint32_t last_token, bool all) {
  const int lo = t.pos0 + (int)first_token, hi = t.pos0 + (int)last_token;
  const int end = hi + 1 < t.len ? hi + 1 : t.len;
  if constexpr (FORM == kShared) {
    if (t.last) return {{0x7FFFFFFF, 0, t.shared}, all ? kEverywhere : -1, kEverywhere};
    return {find_border(c.apart, t.shared, end), lo, hi};
  }
  return {{0, 0, end}, lo, hi};
}

// Where the keys of a split from `begin` on end.  (begin + keys may not fit 31 bits.)
__device__ __forceinline__ int cut_end(int begin, int end, uint32_t keys) {
  return end > begin && (uint32_t)(end - begin) > keys ? begin + (int)keys : end;
}

// A query row's partial of split `sp` of a tile's part.
template <bool SHARE>
__device__ __forceinline__ uint64_t part_of(const Chunk& c, const RowTile& t, uint64_t orow, uint32_t sp) {
  if constexpr (SHARE) return (orow - t.base) * t.stride + t.slot + sp;
  else return orow * c.splits + sp;
}

// ln of a sum of weights 2^(x - m + log2), times the sum that m stands for.
__device__ __forceinline__ float lse_of(float m, float l, float log2) {
  return l == 0.f ? -INFINITY : (m + (__builtin_amdgcn_logf(l) - log2)) * 0.6931471805599453f;
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
// SHARE: keys are counted as Border says; at() is the position of a tile's first key.
template <PoolType PT, int DD, int N, bool UNI, bool SHARE>
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

  const uint32_t* common;  // SHARE: the table of the shared keys
  Border border;
  int shared;

  __device__ __forceinline__ Rows(const PagedBatch& b_, const RowTile& t, uint32_t kvh, int end_, const Border& at_)
      : b(b_), table(b_.table + (uint64_t)t.seq * b_.width),
        page((uint32_t)nfhip::page_bytes(PT, (uint64_t)b_.block_size * DD)), block((uint64_t)b_.n_kv * page),
        head((uint64_t)kvh * page), end(end_), shift(__builtin_ctz(b_.block_size)) {
    if constexpr (SHARE) {
      common = b_.table + (uint64_t)t.pre * b_.width;
      border = at_;
      shared = t.shared;
    }
  }
  __device__ __forceinline__ bool own(int t0) const { return !SHARE || t0 >= border.split; }
  __device__ __forceinline__ int at(int t0) const { return SHARE && own(t0) ? t0 - border.shift : t0; }
  // The table of a tile's keys, and the position below which they lie.
  __device__ __forceinline__ const uint32_t* table_of(int t0) const { return own(t0) ? table : common; }
  __device__ __forceinline__ int end_of(int t0) const {
    return !SHARE ? end : own(t0) ? end - border.shift : shared < end ? shared : end;
  }
  // The keys of a tile that are not before the border, as bits.
  __device__ __forceinline__ uint64_t behind(int t0) const {
    if (!SHARE || !own(t0)) return ~0ull;
    const int before = shared - at(t0);  // at most 15
    return before <= 0 ? ~0ull : ~0ull << before;
  }
  // From a key's row to its scales.
  __device__ __forceinline__ uint32_t to_scales(uint32_t at) const {
    return PT == PoolType::I8 ? (b.block_size - at) * DD + at * (DD / 16) : 0;
  }
  __device__ __forceinline__ void look(int t0) {
    if constexpr (UNI) {
      const int p = at(t0) + 16 * (int)(threadIdx.x & (N - 1));
      entry = table_of(t0)[(uint32_t)min(p, end_of(t0) - 1) >> shift];  // past the end: the last key's block, whose bits are cleared
    } else {
      const int p = at(t0) + (int)(threadIdx.x & (16 * N - 1));
      next_off = 0;
      next_sc = 0;
      bool ok = false;
      if (p < end_of(t0)) {
        const uint32_t k = (uint32_t)p / b.block_size, at = (uint32_t)p - k * b.block_size, phys = table_of(t0)[k];
        ok = phys < b.blocks;
        if (ok) {
          next_off = phys * block + head + at * kRow;
          next_sc = to_scales(at);
        }
      }
      next_valid = __ballot(ok) & behind(t0);
      if constexpr (N < 4) next_valid &= (1ull << (16 * N)) - 1;
    }
  }
  __device__ __forceinline__ void take(int t0) {
    if constexpr (UNI) {
      cur = at(t0);
      valid = 0;
#pragma unroll
      for (int h = 0; h < N; ++h) {
        const uint32_t phys = (uint32_t)__builtin_amdgcn_readlane((int)entry, h);
        const uint32_t at = (uint32_t)(cur + 16 * h) & (b.block_size - 1);
        const bool ok = phys < b.blocks;
        base[h] = ok ? phys * block + head + at * kRow : 0;
        scales[h] = ok ? to_scales(at) : 0;
        valid |= (uint64_t)(ok ? 0xFFFFu : 0u) << (16 * h);
      }
      const int left = end_of(t0) - cur;
      if (left < 16 * N) valid &= SHARE && left <= 0 ? 0 : (1ull << left) - 1;
      valid &= behind(t0);
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
//    rounded to f16 (2^-11 of each, the size of the output's own rounding: attention of
//    normal rows is 2.8e-4 to 2.9e-4 from 64 bits, the rounding of the output alone 2.1e-4;
//    a second product for what is rounded off would be half of all MFMAs again); V
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
// kLse, kShared: the log-sum-exp takes the weights as they were before they are rounded.
template <int DD, int NT, bool LSE>
struct NarrowLds {
  __attribute__((aligned(16))) half_t vs[4][32 * (DD + 16)];
  __attribute__((aligned(16))) float ps[4][32][16];
  float wm[4][16 * NT], wl[4][16 * NT], wx[LSE ? 4 : 1][16 * NT];
};
template <PoolType PT, int DD, int NT, bool UNI, Form FORM>
__device__ __forceinline__ void narrow_tile(const Chunk& c, const RowTile& t, uint32_t sp, uint32_t ns, uint32_t kvh,
                                            NarrowLds<DD, NT, FORM != kChunk>& lds) {
  constexpr bool SHARE = FORM == kShared, LSE = FORM != kChunk;
  constexpr bool I8 = PT == PoolType::I8;
  constexpr int KSTEP = DD / 32, DB = DD / 16;
  // LDS row (halves): 8 dwords past a multiple of 64 or an odd multiple of 8, so that
  // the 8 rows that 32 lanes of a transposing read touch lie in different banks
  constexpr int VP = DD + 16;
  constexpr int VC = I8 ? 16 : 8;                    // elements per 16-byte chunk
  constexpr int CPR = DD / VC, NV = 32 * CPR / 64;   // chunks per row, per lane and tile
  constexpr int NP = KSTEP / 2;                      // I8: 16-code loads per key row
  auto& vs = lds.vs;
  auto& ps = lds.ps;
  auto& wm = lds.wm;
  auto& wl = lds.wl;
  auto& wx = lds.wx;
  static_assert(sizeof(float) * 16 * DD <= sizeof(half_t) * 32 * VP, "a wave's rows merge in its part of vs");

  const uint32_t G = c.group, H = c.n_heads;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t live = t.rows - t.first < 16u * NT ? t.rows - t.first : 16u * NT;
  const bool all = SHARE && t.last && t.all;
  const Keys keys = find_keys<FORM>(c, t, t.first / G, (t.first + live - 1) / G, all);
  const uint32_t cut_keys = SHARE ? t.keys : c.keys_per_split;
  const int pos_lo = keys.lo, begin = (int)(sp * cut_keys);
  int end = keys.at.end;  // keys below it
  end = cut_end(begin, end, cut_keys);
  end = __builtin_amdgcn_readfirstlane(end);

  half8 qb[NT][KSTEP];
  int pos[NT];
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    const uint32_t r = t.first + 16 * u + n < t.rows ? t.first + 16 * u + n : t.rows - 1;
    pos[u] = row_pos<FORM>(c.b, t, r / G, all);
    const half_t* qr = static_cast<const half_t*>(c.q) + ((uint64_t)(t.start + r / G) * H + kvh * G + r % G) * DD;
#pragma unroll
    for (int s = 0; s < KSTEP; ++s) {
      const int d = !I8 || s >= 2 * NP ? 32 * s + 8 * g : 64 * (s / 2) + 16 * g + 8 * (s % 2);
      qb[u][s] = *reinterpret_cast<const half8*>(qr + d);
    }
  }
  float4v ot[NT][DB];
  float m[NT], l[NT], lx[NT];
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    m[u] = -INFINITY;
    l[u] = lx[u] = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d) ot[u][d] = float4v{0.f, 0.f, 0.f, 0.f};
  }

  u32x4 kraw[2][I8 ? (NP > 0 ? NP : 1) : KSTEP];
  uint2 kodd[2];       // I8, odd KSTEP: the last 32 dims
  half_t kd[2][KSTEP]; // I8: scales
  u32x4 vraw[NV];
  half_t vd[NV];
  Rows<PT, DD, 2, UNI, SHARE> rows(c.b, t, kvh, end, keys.at);
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
          if (!OPEN && (!((seen >> k) & 1) || rows.at(t0) + k > pos[u])) sc[u][j][i] = -INFINITY;
          top = fmaxf(top, sc[u][j][i]);
        }
      top = max4(top) * c.scale_log2;
      if (__ballot(top > m[u] + kLagLog2) != 0) {  // uniform
        const float mn = fmaxf(m[u], top);
        const float corr = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[u] - mn);
        l[u] *= corr;
        lx[u] *= corr;
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
      if constexpr (LSE)
        lx[u] += sum4(((pv[u][0][0] + pv[u][0][1]) + (pv[u][0][2] + pv[u][0][3])) +
                      ((pv[u][1][0] + pv[u][1][1]) + (pv[u][1][2] + pv[u][1][3])));
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
          if (!((seen >> k) & 1) || rows.at(t0) + k > pos[u]) continue;
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
  while (t0 < end && (uint32_t)rows.have() == ~0u && rows.at(t0) + 31 <= pos_lo) {  // uniform
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
      if constexpr (LSE) wx[w][16 * u + n] = lx[u];
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
      float M = -INFINITY, L = 0.f, X = 0.f;
#pragma unroll
      for (int v = 0; v < 4; ++v) M = fmaxf(M, wm[v][16 * u + r]);
      float4v A = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float mv = wm[v][16 * u + r];
        const float f = mv == M ? 1.f : __builtin_amdgcn_exp2f(mv - M);
        L += f * wl[v][16 * u + r];
        if constexpr (LSE) X += f * wx[v][16 * u + r];
        A += f * *reinterpret_cast<const float4v*>(reinterpret_cast<const float*>(vs[v]) + r * DD + d);
      }
      const uint64_t o = (uint64_t)(t.start + row / G) * H + kvh * G + row % G;
      if (ns == 1) {
        const float inv = L == 0.f ? 0.f : 1.0f / L;
        half2v a = {(half_t)(A[0] * inv), (half_t)(A[1] * inv)}, bb = {(half_t)(A[2] * inv), (half_t)(A[3] * inv)};
        *reinterpret_cast<uint2*>(static_cast<half_t*>(c.out) + o * DD + d) =
            uint2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, bb)};
        if (LSE && c.lse && d == 0) c.lse[o] = lse_of(M, X, kWeightLog2);
      } else {
        const uint64_t p = part_of<SHARE>(c, t, o, sp);
        if (d == 0) *reinterpret_cast<float2s*>(c.ml + 2 * p) = float2s{M, L};
        if (LSE && d == 0) c.lsum[p] = X;
        *reinterpret_cast<float4v*>(c.acc + p * DD + d) = A;
      }
    }
  }
}

template <PoolType PT, int DD, int NT, bool UNI, Form FORM>
__global__ NF_TWO_PER_CU void chunk_narrow_kernel(Chunk c) {
  const uint32_t sp = blockIdx.x % c.splits, kvh = blockIdx.y;
  RowTile t;
  if (!find_tile(c.b, blockIdx.x / c.splits, c.group, 16 * NT, c.lo, c.hi, t)) return;
  const uint32_t ns = splits_of(c, t.len);
  __shared__ NarrowLds<DD, NT, FORM != kChunk> lds;
  if (sp < ns) narrow_tile<PT, DD, NT, UNI, FORM>(c, t, sp, ns, kvh, lds);
}

// The splits of every query row whose sequence has more than one, where they are few:
// a wave per row.
constexpr uint32_t kFewSplits = 8;
//
// Splits of a row's partials, 1 where its tile has written the output itself.
template <Form FORM>
__device__ __forceinline__ uint32_t row_splits(const Chunk& c, uint32_t seq) {
  const int l = c.b.lens[seq], len = l < (int)c.b.limit ? l : (int)c.b.limit;
  if constexpr (FORM == kShared) {
    const Slots s = find_slots(c, load_cuts(c), seq, (uint32_t)c.b.starts[seq], (int)find_prefix(c.b, c.sh, seq).len, len);
    return s.group + s.own;
  }
  return splits_of(c, len);
}
// Whether they are to be combined.
template <Form FORM>
__device__ __forceinline__ bool row_direct(const Chunk& c, uint32_t seq, uint32_t ns) {
  return ns == 1 && (FORM != kShared || !c.apart || find_prefix(c.b, c.sh, seq).len == 0);
}
template <typename T, int DD, Form FORM>
__global__ __launch_bounds__(256) void chunk_combine_few_kernel(Chunk c) {
  constexpr bool HALF = std::is_same<T, half_t>::value, LSE = FORM != kChunk;
  constexpr int R = (DD + 63) / 64;
  const uint32_t o = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  uint32_t seq;
  int64_t pos;
  if (o >= c.b.rows * c.n_heads || !find_row_wave(c.b, o / c.n_heads, seq, pos)) return;  // uniform
  const uint32_t ns = row_splits<FORM>(c, seq);
  if (row_direct<FORM>(c, seq, ns)) return;
  const uint64_t first = (uint64_t)o * c.splits;
  const float2s* ml = reinterpret_cast<const float2s*>(c.ml) + first;
  float x[kFewSplits][R], M = -INFINITY, L = 0.f, X = 0.f, A[R] = {};
  float2s v[kFewSplits];
  float vx[kFewSplits];
#pragma unroll
  for (uint32_t s = 0; s < kFewSplits; ++s) {
    const uint32_t at = s < ns ? s : ns - 1;
    v[s] = ml[at];
    if (LSE) vx[s] = HALF ? c.lsum[first + at] : v[s][1];
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
    if (LSE) X += f * vx[s];
#pragma unroll
    for (int r = 0; r < R; ++r) A[r] += f * x[s][r];
  }
  if (LSE && c.lse && lane == 0) c.lse[o] = lse_of(M, X, HALF ? kWeightLog2 : 0.f);
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
template <typename T, int DD, Form FORM>
__global__ __launch_bounds__(256) void chunk_combine_kernel(Chunk c) {
  constexpr bool HALF = std::is_same<T, half_t>::value, LSE = FORM != kChunk;
  constexpr int R = (DD + 63) / 64;
  __shared__ float weight[kSplitsAtOnce];
  __shared__ float part[4][64 * R];
  __shared__ float wave_m[4], wave_l[4], wave_x[4];
  const uint32_t o = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint32_t seq;
  int64_t pos;
  if (!find_row_wave(c.b, o / c.n_heads, seq, pos)) return;  // uniform
  const uint32_t ns = row_splits<FORM>(c, seq);
  if (row_direct<FORM>(c, seq, ns)) return;
  const uint64_t first = (uint64_t)o * c.splits;
  const float2s* ml = reinterpret_cast<const float2s*>(c.ml) + first;
  float M = -INFINITY, L = 0.f, X = 0.f;
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
      if (LSE) X += v[1] == 0.f ? 0.f : f * (HALF ? c.lsum[first + s0 + tid] : v[1]);
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
  if (LSE) {
    X = wave_sum(X);
    if (lane == 0) wave_x[wave] = X;
  }
#pragma unroll
  for (int r = 0; r < R; ++r) part[wave][lane + 64 * r] = A[r];
  __syncthreads();
  L = (wave_l[0] + wave_l[1]) + (wave_l[2] + wave_l[3]);
  if (LSE && c.lse && tid == 0)
    c.lse[o] = lse_of(M, (wave_x[0] + wave_x[1]) + (wave_x[2] + wave_x[3]), HALF ? kWeightLog2 : 0.f);
  const float inv = L == 0.f ? 0.f : 1.0f / L;
  for (uint32_t d = tid; d < DD; d += 256)
    static_cast<T*>(c.out)[(uint64_t)o * DD + d] = (T)(((part[0][d] + part[1][d]) + (part[2][d] + part[3][d])) * inv);
}

// kShared, many rows: a wave per row, whose lanes form its splits' weights; the rows of
// eight splits are in flight.  (Five tokens of 32 sequences behind four prompts, 5120 rows
// of some 8 partials: a workgroup per row 13 us, so 6.6; 1024 rows of 44: 8.0 and 8.6.)
// So many rows have at most 60 splits: more do not fit the workspace.
constexpr uint32_t kManyRows = 2048;
template <typename T, int DD>
__global__ __launch_bounds__(256) void shared_combine_kernel(Chunk c) {
  constexpr bool HALF = std::is_same<T, half_t>::value;
  constexpr int R = (DD + 63) / 64, AHEAD = 8;
  const uint32_t lane = threadIdx.x & 63, row0 = first_row(c), o = row0 + blockIdx.x * 4 + (threadIdx.x >> 6);
  uint32_t seq;
  int64_t pos;
  if (o >= c.b.rows * c.n_heads || !find_row_wave(c.b, o / c.n_heads, seq, pos)) return;  // uniform
  const uint32_t ns = row_splits<kShared>(c, seq);
  if (row_direct<kShared>(c, seq, ns)) return;
  const uint64_t first = (uint64_t)(o - row0) * stride_of(c);
  const float2s* ml = reinterpret_cast<const float2s*>(c.ml) + first;
  const float2s v = lane < ns ? ml[lane] : float2s{-INFINITY, 0.f};
  float M = v[0], L = 0.f, X = 0.f, A[R] = {}, f = 0.f;
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) M = fmaxf(M, __shfl_xor(M, k));
  if (v[1] != 0.f) {  // else no key: its row may be anything
    f = v[0] == M ? 1.f : __builtin_amdgcn_exp2f(v[0] - M);
    L = f * v[1];
    X = f * (HALF ? c.lsum[first + lane] : v[1]);
  }
  for (uint32_t s = 0; s < ns; s += AHEAD) {
    float x[AHEAD][R];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
#pragma unroll
      for (int r = 0; r < R; ++r)
        x[i][r] = c.acc[(first + (s + i < ns ? s + i : ns - 1)) * DD + (lane + 64 * r < DD ? lane + 64 * r : DD - 1)];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const float fi = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), (int)((s + i) & 63)));
      if (s + i < ns && fi != 0.f)  // uniform
#pragma unroll
        for (int r = 0; r < R; ++r) A[r] += fi * x[i][r];
    }
  }
  L = wave_sum(L);
  X = wave_sum(X);
  if (c.lse && lane == 0) c.lse[o] = lse_of(M, X, HALF ? kWeightLog2 : 0.f);
  const float inv = L == 0.f ? 0.f : 1.0f / L;
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (lane + 64 * r < DD) static_cast<T*>(c.out)[(uint64_t)o * DD + lane + 64 * r] = (T)(A[r] * inv);
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
// f16 as there, are the B operand of O^T[dim][row] += V^T . P^T as they are.
// Masking, the lazy rescale and values that are not finite: as above; tiles that
// every row of the workgroup sees whole skip all of it.
// No unit bounds it by itself: a wave takes scores, exponentials and P.V one after the
// other.  Two sequences of 2048 tokens behind 6144, 32 heads of 128, 481 GFLOP in 604 to
// 638 us (several cards), 750 to 800 TFLOP/s, where a matrix product of 8192 in each size
// reaches 1093; the MFMA pipes are busy 32 % of the cycles, and without its softmax and
// staging this kernel took 364 us.  From I8 594 to 631 us: half the bytes to stage, the
// conversion beside the MFMAs.
// V rows 16 or 48 dwords past a multiple of 64: the 4 rows and 32 dims that 32 lanes
// of a transposing read touch then lie in different banks (in rows of DD + 8, pairs
// of them share; 685 and 671 us at the size above).  Two buffers for the open tiles; the
// masked ones use the first, and the second for the weights of the vector ALU.
template <int DD>
struct WideLds {
  static constexpr int KP = DD + 8, VP = DD == 96 ? 96 : DD + 32, BUF = 64 * (KP + VP);
  __attribute__((aligned(16))) half_t lds[2 * BUF];
  int tile_bad[2];
};
// HINT: the open loop's test of the end is a branch of its own, unlikely to be taken.  In
// kShared, f16 and 128 dims, 16 chunks of up to 200 tokens behind 8192 positions take 520 us
// without and 476 with it, eight of 60 behind 5000 110 and 101, five tokens of 32 sequences 58 and
// 52.5, but single tokens of 64 53.8 and 55.6; I8 and 64 dims alike within 0.5 %.
// In kChunk two chunks of 2048 tokens behind 6144, f16, 128 dims, 638 and 624, but four of up
// to 512, 64 dims, 110 and 111.5; I8 and 96 dims alike within 0.5 %.
template <PoolType PT, int DD, bool UNI, Form FORM, bool HINT = false>
__device__ __forceinline__ void wide_rows(const Chunk& c, const RowTile& t, uint32_t sp, uint32_t ns, uint32_t kvh,
                                          WideLds<DD>& mem) {
  constexpr bool SHARE = FORM == kShared, LSE = FORM != kChunk;
  constexpr bool I8 = PT == PoolType::I8;
  constexpr int KS = DD / 16, DB = DD / 32, KP = WideLds<DD>::KP, VP = WideLds<DD>::VP, BUF = WideLds<DD>::BUF;
  constexpr int VC = I8 ? 16 : 8;
  constexpr int CPR = DD / VC;
  constexpr int NU = (64 * CPR + 255) / 256;
  static_assert(BUF * sizeof(half_t) >= 4 * 32 * 32 * sizeof(float), "a buffer holds the weights");
  half_t* const lds = mem.lds;
  auto& tile_bad = mem.tile_bad;
  half_t* const ks = lds;
  half_t* const vs = lds + 64 * KP;
  float(*const ps)[32][32] = reinterpret_cast<float(*)[32][32]>(lds + BUF);

  const uint32_t G = c.group, H = c.n_heads;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, hf = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t last = (t.first + 128 < t.rows ? t.first + 128 : t.rows) - 1;
  const bool all = SHARE && t.last && t.all;
  const Keys keys = find_keys<FORM>(c, t, t.first / G, last / G, all);
  const uint32_t cut_keys = SHARE ? t.keys : c.keys_per_split;
  const int pos_lo = keys.lo, begin = (int)(sp * cut_keys);
  int end = keys.at.end;
  end = cut_end(begin, end, cut_keys);
  end = __builtin_amdgcn_readfirstlane(end);

  const uint32_t r0 = t.first + 32 * w;
  const bool wave_live = r0 < t.rows;
  const uint32_t row = r0 + n < t.rows ? r0 + n : t.rows - 1;
  const uint64_t orow = (uint64_t)(t.start + row / G) * H + kvh * G + row % G;
  const int pos = row_pos<FORM>(c.b, t, row / G, all);
  const int w_hi = SHARE && t.last ? kEverywhere
                                   : __builtin_amdgcn_readfirstlane(t.pos0 + (int)((r0 + 31 < t.rows ? r0 + 31 : t.rows - 1) / G));
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
  float lx = 0.f;  // LSE: the sum of the weights as they were before they are rounded

  u32x4 kraw[NU], vraw[NU];
  half_t kd[NU], vd[NU];
  Rows<PT, DD, 4, UNI, SHARE> rows(c.b, t, kvh, end, keys.at);
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
    lx *= corr;
#pragma unroll
    for (int d = 0; d < DB; ++d) ot[d] *= corr;
    m = mn;
    mb = exponent_base(m, kWeightLog2);
  };
  auto weights = [&]() {
    float sum = 0.f, whole = 0.f;
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
        if constexpr (LSE) whole += sc[j][i] + sc[j][i + 1];
      }
    l += sum2(sum);
    if constexpr (LSE) lx += sum2(whole);
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
        if (!((seen >> k) & 1) || rows.at(t0) + k > pos) sc[j][i] = -INFINITY;
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
          if (!((seen >> (32 * j + k)) & 1) || rows.at(t0) + 32 * j + k > pos) continue;
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
  auto open = [&]() {  // uniform
    if (HINT && __builtin_expect(t0 >= end, 0)) return false;
    return t0 < end && rows.have() == ~0ull && rows.at(t0) + 63 <= pos_lo;
  };
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
    if (wave_live && rows.at(t0) <= w_hi) masked_tile(t0, seen, par);  // uniform
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
    if (LSE && c.lse && hf == 0) c.lse[orow] = lse_of(m, lx, kWeightLog2);
  } else {
    const uint64_t p = part_of<SHARE>(c, t, orow, sp);
    if (hf == 0) *reinterpret_cast<float2s*>(c.ml + 2 * p) = float2s{m, l};
    if (LSE && hf == 0) c.lsum[p] = lx;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<float4v*>(c.acc + p * DD + 32 * d + 8 * q + 4 * hf) =
            float4v{ot[d][4 * q], ot[d][4 * q + 1], ot[d][4 * q + 2], ot[d][4 * q + 3]};
  }
}

template <PoolType PT, int DD, bool UNI, Form FORM>
__global__ __launch_bounds__(256, 2) void chunk_wide_kernel(Chunk c) {
  uint32_t kvh, idx;
  if (!wide_tile(c, kvh, idx)) return;
  const uint32_t sp = blockIdx.y;
  RowTile t;
  if (!find_tile(c.b, idx, c.group, 128, c.lo, c.hi, t)) return;
  const uint32_t ns = splits_of(c, t.len);
  __shared__ WideLds<DD> lds;
  if (sp < ns) wide_rows<PT, DD, UNI, FORM, FORM == kChunk && PT == PoolType::F16 && DD == 128>(c, t, sp, ns, kvh, lds);
}

// kShared: narrow and wide tiles in one launch, whose workgroups find out which theirs is, so
// that the groups' parts and the sequences' run beside each other.
// `ns` of a part: 1 says that no other has partials of its rows.
template <PoolType PT, int DD, int NT, bool UNI>
__global__ NF_TWO_PER_CU void shared_kernel(Chunk c) {
  __shared__ union {
    NarrowLds<DD, NT, true> narrow;
    WideLds<DD> wide;
  } lds;
  RowTile t;
  uint32_t sp;
  const uint32_t kvh = blockIdx.x, idx = blockIdx.z * gridDim.y + blockIdx.y;
  using C = Cut<64, 16 * NT, 128>;
  if (c.items) {
    if (!find_planned<C>(c, idx, t, sp)) return;
  } else {
    Cuts keys;
    if (!find_few<C>(c, idx, t, sp, keys)) return;
    if (idx == 0 && kvh == 0 && threadIdx.x == 0) store_cuts(c, keys);
  }
  const uint32_t ns = t.last == 0 && t.slot == 0 ? t.splits : t.splits + 1;
  if (!t.wide) narrow_tile<PT, DD, NT, UNI, kShared>(c, t, sp, ns, kvh, lds.narrow);
  else wide_rows<PT, DD, UNI, kShared, NT == 2>(c, t, sp, ns, kvh, lds.wide);
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
template <int DD, Form FORM>
__device__ __forceinline__ void store_f32(const Chunk& c, uint64_t orow, uint64_t part, uint32_t ns, int g, float m, float l,
                                          const float4v* ot) {
  float* dst = ns == 1 ? static_cast<float*>(c.out) + orow * DD : c.acc + part * DD;
  const float f = ns > 1 ? 1.0f : l == 0.f ? 0.f : 1.0f / l;
  if (FORM != kChunk && ns == 1 && c.lse && g == 0) c.lse[orow] = lse_of(m, l, 0.f);
  if (ns > 1 && g == 0) *reinterpret_cast<float2s*>(c.ml + 2 * part) = float2s{m, l};
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
template <int DD>
struct NarrowLdsF32 {
  __attribute__((aligned(16))) float merge[4][16 * 64 * ((DD + 63) / 64)];
  float wm[4][16], wl[4][16];
};
template <PoolType PT, int DD, bool UNI, Form FORM>
__device__ __forceinline__ void narrow_f32_tile(const Chunk& c, const RowTile& t, uint32_t sp, uint32_t ns, uint32_t kvh,
                                                NarrowLdsF32<DD>& lds) {
  constexpr bool SHARE = FORM == kShared;
  constexpr bool I8 = PT == PoolType::I8;
  constexpr int DG = DD / 4, NH = (DD + 63) / 64, NB = 4 * NH;
  auto& merge = lds.merge;
  auto& wm = lds.wm;
  auto& wl = lds.wl;
  const uint32_t G = c.group, H = c.n_heads;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t last = (t.first + 16 < t.rows ? t.first + 16 : t.rows) - 1;
  const bool all = SHARE && t.last && t.all;
  const Keys keys = find_keys<FORM>(c, t, t.first / G, last / G, all);
  const uint32_t cut_keys = SHARE ? t.keys : c.keys_per_split;
  const int pos_lo = keys.lo, begin = (int)(sp * cut_keys);
  int end = keys.at.end;
  end = cut_end(begin, end, cut_keys);
  end = __builtin_amdgcn_readfirstlane(end);
  const uint32_t row = t.first + n < t.rows ? t.first + n : t.rows - 1;
  const uint64_t orow = (uint64_t)(t.start + row / G) * H + kvh * G + row % G;
  const int pos = row_pos<FORM>(c.b, t, row / G, all);

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
  Rows<PT, DD, 2, UNI, SHARE> rows(c.b, t, kvh, end, keys.at);
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
        if (!OPEN && (!((seen >> k) & 1) || rows.at(t0) + k > pos)) sc[j][i] = -INFINITY;
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
            const uint32_t slot = (uint32_t)(rows.at(t0) + k) % c.b.block_size;
            const uint8_t* page = rows.row(c.v, j, 4 * gk + i) - (uint64_t)slot * rows.kRow;
            if (!((seen >> k) & 1) || rows.at(t0) + k > pos) continue;
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
  while (t0 < end && (uint32_t)rows.have() == ~0u && rows.at(t0) + 31 <= pos_lo) {  // uniform
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
      if (FORM != kChunk && c.lse && d == 0) c.lse[o] = lse_of(M, L, 0.f);
    } else {
      const uint64_t p = part_of<SHARE>(c, t, o, sp);
      if (d == 0) *reinterpret_cast<float2s*>(c.ml + 2 * p) = float2s{M, L};
      *reinterpret_cast<float4v*>(c.acc + p * DD + d) = A;
    }
  }
}

template <PoolType PT, int DD, bool UNI, Form FORM>
__global__ __launch_bounds__(256, 2) void chunk_narrow_f32_kernel(Chunk c) {
  const uint32_t sp = blockIdx.x % c.splits, kvh = blockIdx.y;
  RowTile t;
  if (!find_tile(c.b, blockIdx.x / c.splits, c.group, 16, c.lo, c.hi, t)) return;
  const uint32_t ns = splits_of(c, t.len);
  __shared__ NarrowLdsF32<DD> lds;
  if (sp < ns) narrow_f32_tile<PT, DD, UNI, FORM>(c, t, sp, ns, kvh, lds);
}

// Many query rows: 64 a workgroup, 16 per wave, 32-key tiles of K and V in LDS.
// Bound by the f32 MFMA, busy 55 % of the cycles, and the waits between: one buffer and two
// barriers a tile, few row tiles of unlike length, bank conflicts in 7 % of the cycles.
// Two sequences of 512 tokens with 2048 positions, 32 heads of 128, 293 us; three of up
// to 389 with 2000, 32 heads of 64, 9.5 GFLOP in 117 us with the combine (13 of them),
// where a product of 8192 in each size reaches 153 TFLOP/s.
template <int DD>
struct WideLdsF32 {
  __attribute__((aligned(16))) float ks[32 * (DD + 4)];
  __attribute__((aligned(16))) float vs[32 * (DD + 4) + 64 * ((DD + 63) / 64) - DD];
  __attribute__((aligned(16))) float ps[4][32][16];
  int tile_bad[2];
};
template <PoolType PT, int DD, bool UNI, Form FORM>
__device__ __forceinline__ void wide_f32_rows(const Chunk& c, const RowTile& t, uint32_t sp, uint32_t ns, uint32_t kvh,
                                              WideLdsF32<DD>& lds) {
  constexpr bool SHARE = FORM == kShared;
  constexpr bool I8 = PT == PoolType::I8;
  constexpr int TK = 32, DP = DD + 4, DG = DD / 4, NH = (DD + 63) / 64, NB = 4 * NH;
  constexpr int EC = I8 ? 8 : 4;                  // elements per chunk (8 or 16 bytes)
  constexpr int CPR = DD / EC, NU = (TK * CPR + 255) / 256;
  static_assert(CPR % 4 == 0, "a wave's 64 chunks of a tile lie in one group of 16 keys");
  static_assert(TK == 32, "as in WideLdsF32");
  auto& ks = lds.ks;
  auto& vs = lds.vs;
  auto& ps = lds.ps;
  auto& tile_bad = lds.tile_bad;
  const uint32_t G = c.group, H = c.n_heads;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t last = (t.first + 64 < t.rows ? t.first + 64 : t.rows) - 1;
  const bool all = SHARE && t.last && t.all;
  const Keys keys = find_keys<FORM>(c, t, t.first / G, last / G, all);
  const uint32_t cut_keys = SHARE ? t.keys : c.keys_per_split;
  const int pos_lo = keys.lo, begin = (int)(sp * cut_keys);
  int end = keys.at.end;
  end = cut_end(begin, end, cut_keys);
  end = __builtin_amdgcn_readfirstlane(end);
  const uint32_t r0 = t.first + 16 * w;
  const bool wave_live = r0 < t.rows;
  const uint32_t row = r0 + n < t.rows ? r0 + n : t.rows - 1;
  const uint64_t orow = (uint64_t)(t.start + row / G) * H + kvh * G + row % G;
  const int pos = row_pos<FORM>(c.b, t, row / G, all);
  const int w_hi = SHARE && t.last ? kEverywhere
                                   : __builtin_amdgcn_readfirstlane(t.pos0 + (int)((r0 + 15 < t.rows ? r0 + 15 : t.rows - 1) / G));
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
  Rows<PT, DD, 2, UNI, SHARE> rows(c.b, t, kvh, end, keys.at);
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
          if (!((seen >> k) & 1) || rows.at(t0) + k > pos) sc[j][i] = -INFINITY;
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
        if (!((seen >> k) & 1) || rows.at(t0) + k > pos) continue;
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
  while (t0 < end && (uint32_t)rows.have() == ~0u && rows.at(t0) + TK - 1 <= pos_lo) {  // uniform
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
    if (wave_live && rows.at(t0) <= w_hi) tile(t0, seen, par, std::false_type{});  // uniform
    next();
  }
  if (wave_live && r0 + n < t.rows) store_f32<DD, FORM>(c, orow, part_of<SHARE>(c, t, orow, sp), ns, g, m, l, ot);
}

template <PoolType PT, int DD, bool UNI, Form FORM>
__global__ __launch_bounds__(256, 2) void chunk_wide_f32_kernel(Chunk c) {
  uint32_t kvh, idx;
  if (!wide_tile(c, kvh, idx)) return;
  const uint32_t sp = blockIdx.y;
  RowTile t;
  if (!find_tile(c.b, idx, c.group, 64, c.lo, c.hi, t)) return;
  const uint32_t ns = splits_of(c, t.len);
  __shared__ WideLdsF32<DD> lds;
  if (sp < ns) wide_f32_rows<PT, DD, UNI, FORM>(c, t, sp, ns, kvh, lds);
}
template <PoolType PT, int DD, bool UNI>
__global__ NF_TWO_PER_CU void shared_f32_kernel(Chunk c) {
  __shared__ union {
    NarrowLdsF32<DD> narrow;
    WideLdsF32<DD> wide;
  } lds;
  RowTile t;
  uint32_t sp;
  const uint32_t kvh = blockIdx.x, idx = blockIdx.z * gridDim.y + blockIdx.y;
  using C = Cut<32, 16, 64>;
  if (c.items) {
    if (!find_planned<C>(c, idx, t, sp)) return;
  } else {
    Cuts keys;
    if (!find_few<C>(c, idx, t, sp, keys)) return;
    if (idx == 0 && kvh == 0 && threadIdx.x == 0) store_cuts(c, keys);
  }
  const uint32_t ns = t.last == 0 && t.slot == 0 ? t.splits : t.splits + 1;
  if (!t.wide) narrow_f32_tile<PT, DD, UNI, kShared>(c, t, sp, ns, kvh, lds.narrow);
  else wide_f32_rows<PT, DD, UNI, kShared>(c, t, sp, ns, kvh, lds.wide);
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

// Partials take this many floats for each split of a query row: its maximum, its sums and
// the output row, and what aligns them.
constexpr uint32_t kPartFloats = 4;
inline void place_parts(Chunk& c, const nfhip::Workspace& ws, uint32_t dim, uint64_t n) {  // for n of them
  c.ml = ws.part;
  c.acc = ws.part + (n * 2 + 3) / 4 * 4;
  c.lsum = c.acc + n * dim;
}

struct Operands {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  float* lse;
};
inline Chunk chunk_of(const PagedBatch& b, uint32_t n_heads, const Operands& o) {
  Chunk c{};
  c.b = b;
  c.q = o.q;
  c.k = static_cast<const uint8_t*>(o.k);
  c.v = static_cast<const uint8_t*>(o.v);
  c.out = o.out;
  c.lse = o.lse;
  c.n_heads = n_heads;
  c.group = n_heads / b.n_kv;
  c.scale_log2 = 1.4426950408889634f / sqrtf((float)b.dim);
  return c;
}

template <typename T, PoolType PT, int DD, bool UNI, Form FORM>
hipError_t chunk_mfma_at(const PagedBatch& b, uint32_t n_heads, const Operands& o, const nfhip::Workspace& ws, hipStream_t s) {
  Chunk c = chunk_of(b, n_heads, o);
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
  const uint64_t most = ws.part ? ws.part_floats / ((uint64_t)b.rows * n_heads * (DD + kPartFloats)) : 1;
  if (splits > most) splits = most ? most : 1;
  uint64_t keys = splits > 1 ? (b.limit + splits - 1) / splits : b.limit;
  keys = keys < min_keys ? min_keys : keys;
  keys = (keys + 127) / 128 * 128;
  c.keys_per_split = (uint32_t)keys;
  c.splits = (uint32_t)((b.limit + keys - 1) / keys);
  if (c.splits == 0) c.splits = 1;
  place_parts(c, ws, DD, (uint64_t)b.rows * n_heads * c.splits);
  if (wide) {
    c.tiles = (uint32_t)most_tiles;
    c.lo = narrow ? kFewRows : 0;
    c.hi = ~0ull;
    const dim3 grid(wide_grid(c.tiles, b.n_kv), c.splits);
    if constexpr (F16) chunk_wide_kernel<PT, DD, UNI, FORM><<<grid, 256, 0, s>>>(c);
    else chunk_wide_f32_kernel<PT, DD, UNI, FORM><<<grid, 256, 0, s>>>(c);
  }
  if (narrow) {
    c.lo = 0;
    c.hi = wide ? kFewRows : ~0ull;
    c.tiles = (uint32_t)(wide ? b.n_seqs * (kFewRows / (16 * nt)) : most_tiles);
    const dim3 grid(c.splits * c.tiles, b.n_kv);
    if constexpr (!F16) chunk_narrow_f32_kernel<PT, DD, UNI, FORM><<<grid, 256, 0, s>>>(c);
    else if (nt == 2) chunk_narrow_kernel<PT, DD, 2, UNI, FORM><<<grid, 256, 0, s>>>(c);
    else chunk_narrow_kernel<PT, DD, 1, UNI, FORM><<<grid, 256, 0, s>>>(c);
  }
  if (c.splits > 1) {
    if (c.splits <= kFewSplits) chunk_combine_few_kernel<T, DD, FORM><<<dim3((b.rows * n_heads + 3) / 4), 256, 0, s>>>(c);
    else chunk_combine_kernel<T, DD, FORM><<<dim3(b.rows * n_heads), 256, 0, s>>>(c);
  }
  return hipGetLastError();
}

// Blocks of a power of two of at least 16 positions.
inline bool uniform_blocks(const PagedBatch& b) { return b.block_size >= 16 && (b.block_size & (b.block_size - 1)) == 0; }

// 16-byte rows, and whole groups of query heads: what the MFMA kernels take.  An I8 page of
// block_size head_dim 17/16 bytes has to be whole chunks.
template <PoolType PT>
bool pieces_fit(const PagedBatch& b, uint32_t n_heads, const Operands& o) {
  const uintptr_t all = reinterpret_cast<uintptr_t>(o.q) | reinterpret_cast<uintptr_t>(o.k) |
                        reinterpret_cast<uintptr_t>(o.v) | reinterpret_cast<uintptr_t>(o.out);
  return all % 16 == 0 && n_heads % b.n_kv == 0 && b.blocks > 0 && b.limit > 0 &&
         (PT != PoolType::I8 || b.block_size * b.dim % 256 == 0) && (b.dim == 128 || b.dim == 96 || b.dim == 64);
}

template <typename T, PoolType PT, Form FORM>
hipError_t chunk(const PagedBatch& b, uint32_t n_heads, const Operands& o, const nfhip::Workspace& ws, hipStream_t s) {
  if (pieces_fit<PT>(b, n_heads, o)) {
    const bool uni = uniform_blocks(b);
    if (b.dim == 128) return (uni ? chunk_mfma_at<T, PT, 128, true, FORM> : chunk_mfma_at<T, PT, 128, false, FORM>)(b, n_heads, o, ws, s);
    if (b.dim == 96) return (uni ? chunk_mfma_at<T, PT, 96, true, FORM> : chunk_mfma_at<T, PT, 96, false, FORM>)(b, n_heads, o, ws, s);
    return (uni ? chunk_mfma_at<T, PT, 64, true, FORM> : chunk_mfma_at<T, PT, 64, false, FORM>)(b, n_heads, o, ws, s);
  }
  const float scale = 1.0f / sqrtf((float)b.dim);
  chunk_any_kernel<T, PT, false><<<dim3(b.rows, n_heads), 256, 0, s>>>(b, PagedShared{}, n_heads, scale, (const T*)o.q,
                                                                       (const uint8_t*)o.k, (const uint8_t*)o.v, (T*)o.out, o.lse);
  return hipGetLastError();
}

// The chunk attention of one form, for all types.
template <Form FORM>
hipError_t chunk_all(nfhip::EType t, PoolType pool, const PagedBatch& b, uint32_t n_heads, const Operands& o,
                     const nfhip::Workspace& ws, hipStream_t s) {
  if (t == nfhip::EType::F16)
    return pool == PoolType::I8 ? chunk<half_t, PoolType::I8, FORM>(b, n_heads, o, ws, s)
                                : chunk<half_t, PoolType::F16, FORM>(b, n_heads, o, ws, s);
  return pool == PoolType::I8 ? chunk<float, PoolType::I8, FORM>(b, n_heads, o, ws, s)
                              : chunk<float, PoolType::F32, FORM>(b, n_heads, o, ws, s);
}
hipError_t chunk_lse(nfhip::EType t, PoolType pool, const PagedBatch& b, uint32_t n_heads, const Operands& o,
                     const nfhip::Workspace& ws, hipStream_t s);  // paged_lse.hip

}  // namespace paged
}  // namespace nfk
