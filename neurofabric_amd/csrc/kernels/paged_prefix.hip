// paged_prefix.hip — flash_attention_paged_prefix: attention over a paged cache of
// sequences in groups, each of which shares its first positions.
//
// Where the sequences bring few rows each, a group's shared keys are a part of their own:
// all rows of the group attend to them together, so that they are read once for up to 128
// query rows, and each sequence's own keys are another part; the parts leave partials (m, l,
// acc), which are combined as those of split keys are:
//   m = max m_i,  l = sum l_i 2^(m_i - m),  acc likewise.
// Where they bring many, each sequence's tiles go through the shared keys and its own ones
// after them: a tile's rows are then a sequence's anyway.
//
// The tiles are those of the chunk attention.  What bounds it, 32 heads over 8 KV heads of
// 128 (kernel times):
//   64 single tokens behind 8192 positions, up to 512 of their own, f16: 43 us, combination
//   6; 119 MB, of which a copy takes 24 us (each sequence reading all: 2.2 GB, 440 us).  A
//   workgroup takes 9 us for finding its rows, the first keys and the partials and 2.1 to 2.7
//   for 64 keys, so that more splits would not help.
//   32 behind 32768, up to 1024 of their own, I8: 50 + 8 us, the codes' conversion besides.
//   Five tokens of 32 behind four prompts of 4096: 46 + 7 us.
//   16 questions of up to 200 behind 8192: 457 to 486 us a pass (four cards), 700 TFLOP/s; the
//   softmax between the products, and a last round of workgroups that does not fill the chip.
#include "../paged_tiles.hpp"
#include "paged_attention.hpp"

namespace nfk {
namespace paged {

// Query rows of a sequence (and KV head), on average, up to which the shared keys are apart.
// 16 sequences behind 4096 positions, f16, with the combination, apart and not, both
// without wide_rows()'s HINT: 32 rows 43
// and 49 us, 64 rows 60 and 78, 96 rows 88 and 87; behind two prefixes of 2048, I8: 64 rows
// 40 and 47, 96 rows 52 and 60 (each tile converts its keys).
template <PoolType PT>
constexpr uint32_t kApartRows = PT == PoolType::I8 ? 96 : 64;
// Workgroups that run at once, two on each CU, and the fewest keys that one takes: 256 and
// 128, the attention alone and the combination, three chunks of 154 tokens with 833 positions,
// I8, 42.9 + 8.3 and 38.9 + 8.3 us; six tokens of 53 sequences with up to 1260, I8, 24.2 + 5.4
// and 25.1 + 5.6; one chunk of 493 with 1197, f16, 47.8 + 8.6 and 48.0 + 8.6; single tokens of
// 40 behind 700, 64 dims, 12.8 + 4.1 and 12.3 + 5.4; three of 24 behind 1000, f32, 64 dims, 22.9
// + 5.2 and 20.5 + 5.2.
constexpr uint32_t kResident = 512;
constexpr uint32_t kMinKeys = 256;

template <typename T, PoolType PT, int DD, bool UNI>
hipError_t prefix_at(const PagedBatch& b, const PagedShared& sh, uint32_t n_heads, const Operands& o,
                     const nfhip::Workspace& ws, hipStream_t s) {
  constexpr bool F16 = std::is_same<T, half_t>::value;
  constexpr uint32_t kWideRows = F16 ? 128 : 64, kFew = F16 ? 64 : 32;
  Chunk c = chunk_of(b, n_heads, o);
  c.sh = sh;
  const uint64_t rows = (uint64_t)b.rows * c.group, mean = (rows + b.n_seqs - 1) / b.n_seqs;
  const uint32_t nt = F16 && mean > 16 ? 2 : 1;
  c.target = (kResident + b.n_kv - 1) / b.n_kv;
  // At most so many tiles and splits of a KV head: those of all parts, and what keys_of() and
  // cut_last() may add to them.
  auto tiles = [&](uint64_t parts) { return nfhip::most_tiles(rows, parts, c.group, kFew, 16 * nt, kWideRows); };
  auto items_of = [&](bool apart) { return tiles(b.n_seqs) + (apart ? tiles(sh.n_groups) : 0) + c.target + 16; };
  // The workspace's end: a few numbers, and the plan of a large batch.
  auto plan_floats = [&](bool apart) {
    const uint64_t n = b.n_seqs + (apart ? sh.n_groups : 0);
    return n <= kFewParts && sh.n_groups <= kFewGroups ? 8 : 8 + n * (sizeof(Part) / 4) + items_of(apart) * 2;
  };
  auto splits_in = [&](uint64_t used) {  // of all rows' keys
    return ws.part_floats > used ? (ws.part_floats - used) / ((uint64_t)b.rows * n_heads * (DD + kPartFloats)) : 0;
  };
  c.apart = sh.n_groups > 0 && sh.n_groups < b.n_seqs && mean <= kApartRows<PT> && splits_in(plan_floats(true)) >= 4;
  const uint64_t used = plan_floats(c.apart), most = splits_in(used), items = items_of(c.apart);
  if (!ws.part || ws.part_floats < used) return hipErrorOutOfMemory;
  // The fewest keys of a split for which the partials fit (`limit` as Border counts); a row
  // has them of two parts at most.
  const uint64_t limit = (uint64_t)b.limit + 80, parts = c.apart ? 2 : 0;
  uint64_t keys = most >= 2 ? (limit + most - parts - 1) / (most - parts) : limit;
  if (keys < kMinKeys) keys = kMinKeys;
  keys = (keys + 127) / 128 * 128;
  c.keys_per_split = (uint32_t)keys;
  c.splits = (uint32_t)((limit + keys - 1) / keys + parts);
  c.last_round = most < 2 && used == 8;
  c.room = (ws.part_floats - used) / (DD + kPartFloats);
  place_parts(c, ws, DD, c.last_round ? c.room : (uint64_t)b.rows * n_heads * c.splits);
  c.keys = reinterpret_cast<uint32_t*>(ws.part + (ws.part_floats - used) / 4 * 4);
  if (used > 8) {
    Part* const plan = reinterpret_cast<Part*>(c.keys + 8);
    uint2* const list = reinterpret_cast<uint2*>(plan + b.n_seqs + (c.apart ? sh.n_groups : 0));
    if (nt == 2) plan_kernel<Cut<kFew, 32, kWideRows>><<<1, 1024, 0, s>>>(c, plan, list, (uint32_t)items);
    else plan_kernel<Cut<kFew, 16, kWideRows>><<<1, 1024, 0, s>>>(c, plan, list, (uint32_t)items);
    c.parts = plan;
    c.items = list;
  }
  const uint64_t y = items < 32768 ? items : 32768;
  const dim3 grid(b.n_kv, (unsigned)y, (unsigned)((items + y - 1) / y));
  if constexpr (!F16) shared_f32_kernel<PT, DD, UNI><<<grid, 256, 0, s>>>(c);
  else if (nt == 2) shared_kernel<PT, DD, 2, UNI><<<grid, 256, 0, s>>>(c);
  else shared_kernel<PT, DD, 1, UNI><<<grid, 256, 0, s>>>(c);
  if (c.splits > 1 || c.last_round) {
    // of the last sequences, where only they have partials: as many rows as those of two splits fit
    const uint64_t all = (uint64_t)b.rows * n_heads;
    const uint32_t outs = (uint32_t)(c.last_round && all > c.room / 2 ? c.room / 2 : all);
    if (c.last_round) shared_combine_kernel<T, DD><<<dim3((outs + 3) / 4), 256, 0, s>>>(c);
    else if (c.splits <= kFewSplits) chunk_combine_few_kernel<T, DD, kShared><<<dim3((outs + 3) / 4), 256, 0, s>>>(c);
    else if (outs >= kManyRows) shared_combine_kernel<T, DD><<<dim3((outs + 3) / 4), 256, 0, s>>>(c);
    else chunk_combine_kernel<T, DD, kShared><<<dim3(outs), 256, 0, s>>>(c);
  }
  return hipGetLastError();
}

template <typename T, PoolType PT>
hipError_t prefix(const PagedBatch& b, const PagedShared& sh, uint32_t n_heads, const Operands& o, const nfhip::Workspace& ws,
                  hipStream_t s) {
  if (pieces_fit<PT>(b, n_heads, o)) {
    const bool uni = uniform_blocks(b);
    if (b.dim == 128) return (uni ? prefix_at<T, PT, 128, true> : prefix_at<T, PT, 128, false>)(b, sh, n_heads, o, ws, s);
    if (b.dim == 96) return (uni ? prefix_at<T, PT, 96, true> : prefix_at<T, PT, 96, false>)(b, sh, n_heads, o, ws, s);
    return (uni ? prefix_at<T, PT, 64, true> : prefix_at<T, PT, 64, false>)(b, sh, n_heads, o, ws, s);
  }
  const float scale = 1.0f / sqrtf((float)b.dim);
  chunk_any_kernel<T, PT, true><<<dim3(b.rows, n_heads), 256, 0, s>>>(b, sh, n_heads, scale, (const T*)o.q, (const uint8_t*)o.k,
                                                                      (const uint8_t*)o.v, (T*)o.out, o.lse);
  return hipGetLastError();
}

}  // namespace paged
}  // namespace nfk

namespace nfhip {

hipError_t launch_paged_prefix(EType t, PoolType pool, const PagedBatch& b, const PagedShared& sh, uint32_t n_heads,
                               const void* q, const void* k_pool, const void* v_pool, void* out, float* lse,
                               const Workspace& ws, hipStream_t s) {
  using namespace nfk;
  if (b.rows == 0 || b.n_seqs == 0) return hipSuccess;
  const paged::Operands o{q, k_pool, v_pool, out, lse};
  if (t == EType::F16)
    return pool == PoolType::I8 ? paged::prefix<half_t, PoolType::I8>(b, sh, n_heads, o, ws, s)
                                : paged::prefix<half_t, PoolType::F16>(b, sh, n_heads, o, ws, s);
  return pool == PoolType::I8 ? paged::prefix<float, PoolType::I8>(b, sh, n_heads, o, ws, s)
                              : paged::prefix<float, PoolType::F32>(b, sh, n_heads, o, ws, s);
}

}  // namespace nfhip
