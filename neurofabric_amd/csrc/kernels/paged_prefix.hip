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
#include "paged_attention.hpp"

namespace nfk {
namespace paged {

// Query rows of a sequence, on average, up to which the shared keys are apart.
constexpr uint32_t kApartRows = 64;
// Workgroups of a launch: two on each CU.
constexpr uint32_t kResident = 512;

template <typename T, PoolType PT, int DD, bool UNI>
hipError_t prefix_at(const PagedBatch& b, const PagedShared& sh, uint32_t n_heads, const Operands& o,
                     const nfhip::Workspace& ws, hipStream_t s) {
  constexpr bool F16 = std::is_same<T, half_t>::value;
  constexpr uint32_t kWideRows = F16 ? 128 : 64;
  Chunk c = chunk_of(b, n_heads, o);
  c.sh = sh;
  const uint64_t rows = (uint64_t)b.rows * c.group, mean = (rows + b.n_seqs - 1) / b.n_seqs;
  const uint64_t most = ws.part ? ws.part_floats / ((uint64_t)b.rows * n_heads * (DD + kPartFloats)) : 1;
  c.apart = sh.n_groups > 0 && sh.n_groups < b.n_seqs && mean <= kApartRows && most >= 4;
  const uint32_t nt = F16 && mean > 16 ? 2 : 1;
  const bool wide = rows > kNarrowRows<T>;
  const uint64_t per = (c.apart ? wide : mean > kNarrowRows<T>) ? kWideRows : 16 * nt;
  // Tiles that share the keys between them; a row has partials of two parts at most.
  const uint64_t tiles = (c.apart ? (rows + per - 1) / per : b.n_seqs * ((mean + per - 1) / per)) * b.n_kv;
  uint64_t splits = tiles < kResident ? kResident / tiles : 1;
  const uint64_t limit = (uint64_t)b.limit + 80, parts = c.apart ? 2 : 0;  // (as Border counts)
  if (splits > most - parts && most >= parts + 1) splits = most - parts;
  if (!c.apart && most < 2) splits = 1;
  uint64_t keys = (limit + splits - 1) / splits;
  if (keys < 256) keys = 256;
  keys = (keys + 127) / 128 * 128;
  c.keys_per_split = (uint32_t)keys;
  c.splits = (uint32_t)((limit + keys - 1) / keys + parts);
  place_parts(c, ws, DD);
  auto grid = [&](uint64_t at) {  // workgroups for tiles of `at` rows
    const uint64_t n = ((c.apart ? 2 : 1) * (rows / at + b.n_seqs) + sh.n_groups) * c.splits * b.n_kv;
    return dim3((unsigned)(n < kResident ? n : kResident));
  };
  if (wide) {
    c.lo = kNarrowRows<T>;
    c.hi = ~0ull;
    if constexpr (F16) shared_wide_kernel<PT, DD, UNI><<<grid(kWideRows), 256, 0, s>>>(c);
    else shared_wide_f32_kernel<PT, DD, UNI><<<grid(kWideRows), 256, 0, s>>>(c);
  }
  if (!wide || b.n_seqs > 1) {
    c.lo = 0;
    c.hi = kNarrowRows<T>;
    if constexpr (!F16) shared_narrow_f32_kernel<PT, DD, UNI><<<grid(16), 256, 0, s>>>(c);
    else if (nt == 2) shared_narrow_kernel<PT, DD, 2, UNI><<<grid(32), 256, 0, s>>>(c);
    else shared_narrow_kernel<PT, DD, 1, UNI><<<grid(16), 256, 0, s>>>(c);
  }
  if (c.splits > 1) {
    if (c.splits <= kFewSplits) chunk_combine_few_kernel<T, DD, kShared><<<dim3((b.rows * n_heads + 3) / 4), 256, 0, s>>>(c);
    else chunk_combine_kernel<T, DD, kShared><<<dim3(b.rows * n_heads), 256, 0, s>>>(c);
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
