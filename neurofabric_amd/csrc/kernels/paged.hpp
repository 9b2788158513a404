// paged.hpp — device helpers of the ops on a paged key / value cache.
//
// A batch is n_seqs sequences.  Rows starts[s] .. starts[s + 1] - 1 of the dense
// operands belong to sequence s and are its last positions, up to lens[s] - 1.
// Position p of a sequence lies in block table[s][p / block_size], slot p %
// block_size; a block holds one page per KV head.  Starts, lengths and tables
// are device data that the host never sees, so every index made from them is
// checked here: a row before starts[0] or behind the last start belongs to no
// sequence, nor does one of a sequence whose rows are not all rows of the batch,
// and a position below 0, at or past `limit`, or in a block past the
// pools has no storage.
#pragma once

#include "../launch.hpp"
#include "common.hpp"

namespace nfk {
namespace paged {

using nfhip::PagedBatch;
using nfhip::PagedShared;
using nfhip::PoolType;

// Sequence and position of row `row`; false when it belongs to none.
__device__ __forceinline__ bool find_row(const PagedBatch& b, uint32_t row, uint32_t& seq, int64_t& pos) {
  uint32_t lo = 0, hi = b.n_seqs;  // first s with starts[s + 1] > row
  while (lo < hi) {
    const uint32_t mid = (lo + hi) / 2;
    if ((int64_t)b.starts[mid + 1] <= (int64_t)row) lo = mid + 1;
    else hi = mid;
  }
  if (lo >= b.n_seqs) return false;
  const int64_t a = b.starts[lo], e = b.starts[lo + 1];
  if (a < 0 || a > (int64_t)row || e > (int64_t)b.rows) return false;
  seq = lo;
  pos = (int64_t)b.lens[lo] - (e - (int64_t)row);
  return true;
}

// The same for a row that is the same in all lanes: up to 64 sequences in one
// round of loads, where the search takes one for each of its steps.
__device__ __forceinline__ bool find_row_wave(const PagedBatch& b, uint32_t row, uint32_t& seq, int64_t& pos) {
  if (b.n_seqs > 64) return find_row(b, row, seq, pos);
  const uint32_t s = threadIdx.x & 63;
  int32_t a = -1, e = -1, len = 0;
  if (s < b.n_seqs) {
    a = b.starts[s];
    e = b.starts[s + 1];
    len = b.lens[s];
  }
  const uint64_t mine = __ballot(a >= 0 && (int64_t)a <= (int64_t)row && (int64_t)row < (int64_t)e && (int64_t)e <= (int64_t)b.rows);
  if (mine == 0) return false;
  const int at = __builtin_ctzll(mine);
  seq = at;
  pos = (int64_t)__shfl(len, at) - ((int64_t)__shfl(e, at) - (int64_t)row);
  return true;
}

// The shared positions of a sequence, read through the table of sequence `seq`: none
// (len 0) for a sequence in no group.  `first` and the prefixes are device data too.
struct SharedPrefix {
  uint32_t seq;
  int64_t len;
};
__device__ __forceinline__ SharedPrefix find_prefix(const PagedBatch& b, const PagedShared& sh, uint32_t seq) {
  uint32_t lo = 0, hi = sh.n_groups;  // first g with first[g + 1] > seq
  while (lo < hi) {
    const uint32_t mid = (lo + hi) / 2;
    if ((int64_t)sh.first[mid + 1] <= (int64_t)seq) lo = mid + 1;
    else hi = mid;
  }
  if (lo >= sh.n_groups) return {seq, 0};
  const int32_t a = sh.first[lo], n = sh.len[lo];
  if (a < 0 || (uint32_t)a > seq || n <= 0) return {seq, 0};
  return {(uint32_t)a, n < (int64_t)b.limit ? n : (int64_t)b.limit};
}

// Physical block of position `pos` of sequence `seq`, or ~0 without storage.
__device__ __forceinline__ uint32_t find_block(const PagedBatch& b, uint32_t seq, int64_t pos) {
  if (pos < 0 || pos >= (int64_t)b.limit) return ~0u;
  const uint32_t phys = b.table[(uint64_t)seq * b.width + (uint32_t)pos / b.block_size];
  return phys < b.blocks ? phys : ~0u;
}

// The page of KV head `kvh` in a pool.
template <PoolType PT>
__device__ __forceinline__ uint64_t page_offset(const PagedBatch& b, uint32_t phys, uint32_t kvh) {
  return ((uint64_t)phys * b.n_kv + kvh) * nfhip::page_bytes(PT, (uint64_t)b.block_size * b.dim);
}

// Element `d` of row `slot` of a page, as the f32 value it stands for (exact).
template <PoolType PT>
__device__ __forceinline__ float page_value(const PagedBatch& b, const uint8_t* page, uint32_t slot, uint32_t d) {
  const uint32_t i = slot * b.dim + d;
  if constexpr (PT == PoolType::F32) return reinterpret_cast<const float*>(page)[i];
  else if constexpr (PT == PoolType::F16) return (float)reinterpret_cast<const half_t*>(page)[i];
  else
    return (float)(int)reinterpret_cast<const int8_t*>(page)[i] *
           (float)reinterpret_cast<const half_t*>(page + b.block_size * b.dim)[i / 32];
}

// The same as rows of type T see it: an I8 pool's values are rounded to f16 once for f16
// rows.
template <typename T, PoolType PT>
__device__ __forceinline__ float row_value(const PagedBatch& b, const uint8_t* page, uint32_t slot, uint32_t d) {
  const float x = page_value<PT>(b, page, slot, d);
  return PT == PoolType::I8 ? (float)(T)x : x;
}

// The fp16 scale of 32 elements of type T and largest magnitude `amax`:
// fp16(amax / 127), at most the largest finite fp16.  Finite f16 elements stay
// finite where they are read as f16: amax = 65504 would take 516, whose multiple
// 127 * 516 rounds to infinity, and takes the next scale below.
template <typename T>
__device__ __forceinline__ half_t scale_of(float amax) {
  const half_t d = (half_t)(amax / 127.0f);
  if (sizeof(T) == 2 && amax <= 65504.0f && d > (half_t)515.5f) return (half_t)515.5f;
  return __builtin_isinf((float)d) ? (half_t)65504.0f : d;
}

// x / d to the nearest integer, ties to even, limited to +-127; 0 for NaN and
// for d = 0.  `inv` = 1 / d.  x * inv may be off in its last bits, so the
// quotient next to a border between two codes is corrected from its remainder
// r = x - q d, which is exact: q and the border are within a factor of two of
// x, or q = 0.
__device__ __forceinline__ int code_of_value(float x, float d, float inv) {
  float q = __builtin_rintf(x * inv);
  q = fminf(fmaxf(q, -128.0f), 128.0f);
  const float r = __builtin_fmaf(-q, d, x);
  // |r| > d / 2, or |r| = d / 2 and q odd
  const uint32_t over = __builtin_bit_cast(uint32_t, __builtin_fabsf(r)) + ((uint32_t)(int)q & 1u);
  if (over > __builtin_bit_cast(uint32_t, 0.5f * d)) q += __builtin_copysignf(1.0f, r);
  q = fminf(fmaxf(q, -127.0f), 127.0f);
  return x == x ? (int)q : 0;
}

}  // namespace paged
}  // namespace nfk
