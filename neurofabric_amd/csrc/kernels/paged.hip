// paged.hip — new key and value rows written into a paged cache
// (paged_kv_append), quantised to 8 bits when the pools are, and rows read back
// (paged_kv_gather).
//
// I8 pools hold, for 32 consecutive elements x of a row, the scale d =
// fp16(max|x| / 127) and the codes q = x / d to the nearest integer (ties to
// even); the cache then stands for q d.  Values beyond 127 of the largest fp16
// scale saturate, a NaN is held as 0.
#include <type_traits>

#include "paged.hpp"

namespace nfk {
namespace paged {

// Any head_dim and alignment: a thread per element, or per 32 elements of an
// I8 pool.  blockIdx.y: 0 = K, 1 = V.
template <typename T, PoolType PT>
__global__ __launch_bounds__(256) void append_any_kernel(PagedBatch b, const T* __restrict__ kn,
                                                         const T* __restrict__ vn, uint8_t* __restrict__ kp,
                                                         uint8_t* __restrict__ vp) {
  constexpr uint32_t U = PT == PoolType::I8 ? 32 : 1;
  const uint64_t id = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const uint32_t per_head = b.dim / U, per_row = b.n_kv * per_head;
  if (id >= (uint64_t)b.rows * per_row) return;
  const uint32_t row = (uint32_t)(id / per_row), u = (uint32_t)(id % per_row);
  const uint32_t kvh = u / per_head, d0 = u % per_head * U;
  uint32_t seq;
  int64_t pos;
  if (!find_row(b, row, seq, pos)) return;
  const uint32_t phys = find_block(b, seq, pos);
  if (phys == ~0u) return;
  const uint32_t slot = (uint32_t)pos % b.block_size;
  const T* src = (blockIdx.y ? vn : kn) + ((uint64_t)row * b.n_kv + kvh) * b.dim + d0;
  uint8_t* page = (blockIdx.y ? vp : kp) + page_offset<PT>(b, phys, kvh);
  if constexpr (PT != PoolType::I8) {
    reinterpret_cast<T*>(page)[slot * b.dim + d0] = src[0];
  } else {
    float amax = 0.0f;
    for (uint32_t i = 0; i < U; ++i) amax = fmaxf(amax, __builtin_fabsf((float)src[i]));
    const half_t d = scale_of(amax);
    const float df = (float)d, inv = df > 0.0f ? 1.0f / df : 0.0f;
    for (uint32_t i = 0; i < U; ++i)
      page[slot * b.dim + d0 + i] = (uint8_t)(df > 0.0f ? code_of_value((float)src[i], df, inv) : 0);
    reinterpret_cast<half_t*>(page + b.block_size * b.dim)[(slot * b.dim + d0) / 32] = d;
  }
}

// A thread per element.  Rows without storage become zeros; rows of no
// sequence stay as they are.
template <typename T, PoolType PT>
__global__ __launch_bounds__(256) void gather_any_kernel(PagedBatch b, const uint8_t* __restrict__ kp,
                                                         const uint8_t* __restrict__ vp, T* __restrict__ ko,
                                                         T* __restrict__ vo) {
  const uint64_t id = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  const uint32_t per_row = b.n_kv * b.dim;
  if (id >= (uint64_t)b.rows * per_row) return;
  const uint32_t row = (uint32_t)(id / per_row), u = (uint32_t)(id % per_row);
  uint32_t seq;
  int64_t pos;
  if (!find_row(b, row, seq, pos)) return;
  const uint32_t phys = find_block(b, seq, pos);
  float x = 0.0f;
  if (phys != ~0u)
    x = page_value<PT>(b, (blockIdx.y ? vp : kp) + page_offset<PT>(b, phys, u / b.dim),
                       (uint32_t)pos % b.block_size, u % b.dim);
  (blockIdx.y ? vo : ko)[id] = (T)x;
}

template <typename T, PoolType PT>
hipError_t append(const PagedBatch& b, const void* kn, const void* vn, void* kp, void* vp, hipStream_t s) {
  const uint64_t n = (uint64_t)b.rows * b.n_kv * (PT == PoolType::I8 ? b.dim / 32 : b.dim);
  append_any_kernel<T, PT><<<dim3((unsigned)((n + 255) / 256), 2), 256, 0, s>>>(
      b, (const T*)kn, (const T*)vn, (uint8_t*)kp, (uint8_t*)vp);
  return hipGetLastError();
}

template <typename T, PoolType PT>
hipError_t gather(const PagedBatch& b, const void* kp, const void* vp, void* ko, void* vo, hipStream_t s) {
  const uint64_t n = (uint64_t)b.rows * b.n_kv * b.dim;
  gather_any_kernel<T, PT><<<dim3((unsigned)((n + 255) / 256), 2), 256, 0, s>>>(
      b, (const uint8_t*)kp, (const uint8_t*)vp, (T*)ko, (T*)vo);
  return hipGetLastError();
}

}  // namespace paged
}  // namespace nfk

namespace nfhip {

hipError_t launch_paged_append(EType t, PoolType pool, const PagedBatch& b, const void* k, const void* v, void* k_pool,
                               void* v_pool, hipStream_t s) {
  using namespace nfk;
  if (b.rows == 0 || b.n_seqs == 0) return hipSuccess;
  if (t == EType::F16)
    return pool == PoolType::I8 ? paged::append<half_t, PoolType::I8>(b, k, v, k_pool, v_pool, s)
                                : paged::append<half_t, PoolType::F16>(b, k, v, k_pool, v_pool, s);
  return pool == PoolType::I8 ? paged::append<float, PoolType::I8>(b, k, v, k_pool, v_pool, s)
                              : paged::append<float, PoolType::F32>(b, k, v, k_pool, v_pool, s);
}

hipError_t launch_paged_gather(EType t, PoolType pool, const PagedBatch& b, const void* k_pool, const void* v_pool,
                               void* k, void* v, hipStream_t s) {
  using namespace nfk;
  if (b.rows == 0 || b.n_seqs == 0) return hipSuccess;
  if (t == EType::F16)
    return pool == PoolType::I8 ? paged::gather<half_t, PoolType::I8>(b, k_pool, v_pool, k, v, s)
                                : paged::gather<half_t, PoolType::F16>(b, k_pool, v_pool, k, v, s);
  return pool == PoolType::I8 ? paged::gather<float, PoolType::I8>(b, k_pool, v_pool, k, v, s)
                              : paged::gather<float, PoolType::F32>(b, k_pool, v_pool, k, v, s);
}

}  // namespace nfhip
