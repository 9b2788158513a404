// paged_attention.hip — flash_attention_paged_chunk: choice and launch of the kernels.
#include "paged_attention.hpp"

namespace nfk {
namespace paged {

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
hipError_t chunk(const PagedBatch& b, uint32_t n_heads, const void* q, const void* kp, const void* vp, void* out, float* lse,
                 const nfhip::Workspace& ws, hipStream_t s) {
  const uintptr_t all = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(kp) |
                        reinterpret_cast<uintptr_t>(vp) | reinterpret_cast<uintptr_t>(out);
  // 16-byte rows: an I8 page of block_size head_dim 17/16 bytes has to be whole chunks
  if (!lse && all % 16 == 0 && n_heads % b.n_kv == 0 && b.blocks > 0 && b.limit > 0 &&
      (PT != PoolType::I8 || b.block_size * b.dim % 256 == 0)) {
    if (b.dim == 128) return chunk_mfma<T, PT, 128>(b, n_heads, q, kp, vp, out, ws, s);
    if (b.dim == 96) return chunk_mfma<T, PT, 96>(b, n_heads, q, kp, vp, out, ws, s);
    if (b.dim == 64) return chunk_mfma<T, PT, 64>(b, n_heads, q, kp, vp, out, ws, s);
  }
  const float scale = 1.0f / sqrtf((float)b.dim);
  chunk_any_kernel<T, PT, false><<<dim3(b.rows, n_heads), 256, 0, s>>>(b, PagedShared{}, n_heads, scale, (const T*)q,
                                                                       (const uint8_t*)kp, (const uint8_t*)vp, (T*)out, lse);
  return hipGetLastError();
}

}  // namespace paged
}  // namespace nfk

namespace nfhip {

hipError_t launch_paged_chunk(EType t, PoolType pool, const PagedBatch& b, uint32_t n_heads, const void* q,
                              const void* k_pool, const void* v_pool, void* out, float* lse, const Workspace& ws,
                              hipStream_t s) {
  using namespace nfk;
  if (b.rows == 0 || b.n_seqs == 0) return hipSuccess;
  if (t == EType::F16)
    return pool == PoolType::I8 ? paged::chunk<half_t, PoolType::I8>(b, n_heads, q, k_pool, v_pool, out, lse, ws, s)
                                : paged::chunk<half_t, PoolType::F16>(b, n_heads, q, k_pool, v_pool, out, lse, ws, s);
  return pool == PoolType::I8 ? paged::chunk<float, PoolType::I8>(b, n_heads, q, k_pool, v_pool, out, lse, ws, s)
                              : paged::chunk<float, PoolType::F32>(b, n_heads, q, k_pool, v_pool, out, lse, ws, s);
}

}  // namespace nfhip
