// paged_prefix.hip — flash_attention_paged_prefix: attention over a paged cache of
// sequences in groups, each of which shares its first positions.
#include "paged_attention.hpp"

namespace nfk {
namespace paged {

template <typename T, PoolType PT>
hipError_t prefix(const PagedBatch& b, const PagedShared& sh, uint32_t n_heads, const void* q, const void* kp,
                  const void* vp, void* out, float* lse, const nfhip::Workspace& ws, hipStream_t s) {
  (void)ws;
  const float scale = 1.0f / sqrtf((float)b.dim);
  chunk_any_kernel<T, PT, true><<<dim3(b.rows, n_heads), 256, 0, s>>>(b, sh, n_heads, scale, (const T*)q, (const uint8_t*)kp,
                                                                      (const uint8_t*)vp, (T*)out, lse);
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
  if (t == EType::F16)
    return pool == PoolType::I8 ? paged::prefix<half_t, PoolType::I8>(b, sh, n_heads, q, k_pool, v_pool, out, lse, ws, s)
                                : paged::prefix<half_t, PoolType::F16>(b, sh, n_heads, q, k_pool, v_pool, out, lse, ws, s);
  return pool == PoolType::I8 ? paged::prefix<float, PoolType::I8>(b, sh, n_heads, q, k_pool, v_pool, out, lse, ws, s)
                              : paged::prefix<float, PoolType::F32>(b, sh, n_heads, q, k_pool, v_pool, out, lse, ws, s);
}

}  // namespace nfhip
