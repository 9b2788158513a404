// paged.hip — new key and value rows written into a paged cache
// (paged_kv_append), quantised to 8 bits when the pools are, and rows read back
// (paged_kv_gather).
//
// I8 pools hold, for 32 consecutive elements x of a row, the scale d =
// fp16(max|x| / 127) and the codes q = x / d to the nearest integer (ties to
// even); the cache then stands for q d.  Values beyond 127 of the largest fp16
// scale saturate, a NaN is held as 0.  Finite f16 rows take scales of at most 515.5,
// so that what the cache stands for is finite in f16 too.
#include <type_traits>

#include "paged.hpp"

namespace nfk {
namespace paged {

// Any head_dim and alignment: a thread per element, or per 32 elements of an
// I8 pool, each of which looks its row up, which is what bounds it (32768 rows of 8 heads
// of 100 appended in f16 and read back: 682 us).  blockIdx.y: 0 = K, 1 = V.
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
    const half_t d = scale_of<T>(amax);
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

// 16-byte pieces of the dense rows (4 f32, 8 f16), a wave per row: K and V of up to
// kPieces pieces a lane are loaded before the row's place is looked up, so the two
// latencies overlap.  I8: the 8 (f32) or 4 (f16) lanes of 32 elements find their
// largest together.  Bound by HBM: four prompts of up to 2048 rows of 8 heads of 128
// appended in f16, 55 MB in 9.6 us (the last-level cache holds them between calls), 32768 rows of f32 to
// I8 in 76 us and back in 46 (512 MB in 119 together, 4.3 TB/s), 65536 of I8 to f16 in 82
// (411 MB, 5.0 TB/s; a copy of 2 GiB reaches 4.9).  A step's few rows take 3 us each way,
// the chain start - table - row.
// SPREAD, for batches too small to fill the chip: a wave takes 64 pieces of K or of V
// (blockIdx.y: 2 slice + which), which cuts the instructions that one after the other
// make up such a call (appended to I8 and read back: 4 rows 7.8 us, 7.2 spread; 512
// rows 9.3 and 7.3); at large ones more waves look the same rows up (8192 rows: 30 us
// and 33; 1024 rows, where either does: 9.6 and 8.7).
constexpr int kPieces = 2;
constexpr uint32_t kSpreadRows = 512;

template <typename T>
struct Piece {
  static constexpr int kElems = 16 / sizeof(T);
  typedef T type __attribute__((ext_vector_type(kElems)));
};

template <typename T>
__device__ __forceinline__ void put_codes(typename Piece<T>::type x, uint8_t* codes, half_t* scale, bool first) {
  constexpr int E = Piece<T>::kElems;
  float amax = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) amax = fmaxf(amax, __builtin_fabsf((float)x[e]));
#pragma unroll
  for (int o = 1; o < 32 / E; o <<= 1) amax = fmaxf(amax, __shfl_xor(amax, o));
  const half_t d = scale_of<T>(amax);
  const float df = (float)d, inv = df > 0.0f ? 1.0f / df : 0.0f;
  uint32_t w[E / 4] = {};
#pragma unroll
  for (int e = 0; e < E; ++e)
    w[e / 4] |= (uint32_t)(uint8_t)(df > 0.0f ? code_of_value((float)x[e], df, inv) : 0) << (8 * (e % 4));
  if constexpr (E == 8) *reinterpret_cast<uint2*>(codes) = uint2{w[0], w[1]};
  else *reinterpret_cast<uint32_t*>(codes) = w[0];
  if (first) *scale = d;
}

template <typename T, PoolType PT, bool SPREAD>
__global__ __launch_bounds__(256) void append_kernel(PagedBatch b, const T* __restrict__ kn, const T* __restrict__ vn,
                                                     uint8_t* __restrict__ kp, uint8_t* __restrict__ vp) {
  constexpr uint32_t E = Piece<T>::kElems;
  typedef typename Piece<T>::type vec;
  const uint32_t row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= b.rows) return;
  const uint32_t per_head = b.dim / E, pieces = b.n_kv * per_head;
  const vec* ks = reinterpret_cast<const vec*>(kn) + (uint64_t)row * pieces;
  const vec* vs = reinterpret_cast<const vec*>(vn) + (uint64_t)row * pieces;
  constexpr int P = SPREAD ? 1 : kPieces;
  const uint32_t first = SPREAD ? blockIdx.y / 2 * 64 : 0, last = SPREAD ? min(first + 64, pieces) : pieces;
  vec kx[P], vx[P];
  auto load = [&](uint32_t u0) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const uint32_t u = u0 + 64 * i + lane < pieces ? u0 + 64 * i + lane : pieces - 1;
      if (SPREAD) {
        kx[i] = (blockIdx.y & 1 ? vs : ks)[u];
      } else {
        kx[i] = ks[u];
        vx[i] = vs[u];
      }
    }
  };
  load(first);
  uint32_t seq;
  int64_t pos;
  if (!find_row_wave(b, row, seq, pos)) return;  // uniform
  const uint32_t phys = find_block(b, seq, pos);
  if (phys == ~0u) return;
  const uint32_t slot = (uint32_t)pos % b.block_size;
  const uint64_t page = nfhip::page_bytes(PT, (uint64_t)b.block_size * b.dim), block = (uint64_t)phys * b.n_kv * page;
  uint8_t* const p0 = SPREAD && (blockIdx.y & 1) ? vp : kp;
  for (uint32_t u0 = first; u0 < last; u0 += 64 * P) {
    if (u0 != first) load(u0);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const uint32_t u = u0 + 64 * i + lane;
      const uint32_t head = u / per_head, d = (u - head * per_head) * E;
      const uint64_t at = block + head * page;
      if constexpr (PT != PoolType::I8) {
        if (u >= pieces) break;
        const uint64_t to = at + (uint64_t)(slot * b.dim + d) * sizeof(T);
        *reinterpret_cast<vec*>(p0 + to) = kx[i];
        if (!SPREAD) *reinterpret_cast<vec*>(vp + to) = vx[i];
      } else {
        if (u0 + 64 * i >= pieces) break;  // uniform: groups of 32 elements are never split
        const uint32_t el = slot * b.dim + d;
        const uint64_t sc = at + (uint64_t)b.block_size * b.dim + el / 16;
        if (u >= pieces) continue;
        put_codes<T>(kx[i], p0 + at + el, reinterpret_cast<half_t*>(p0 + sc), d % 32 == 0);
        if (!SPREAD) put_codes<T>(vx[i], vp + at + el, reinterpret_cast<half_t*>(vp + sc), d % 32 == 0);
      }
    }
  }
}

template <typename T, PoolType PT, bool SPREAD>
__global__ __launch_bounds__(256) void gather_kernel(PagedBatch b, const uint8_t* __restrict__ kp,
                                                     const uint8_t* __restrict__ vp, T* __restrict__ ko,
                                                     T* __restrict__ vo) {
  constexpr uint32_t E = Piece<T>::kElems;
  typedef typename Piece<T>::type vec;
  typedef typename std::conditional<E == 8, uint2, uint32_t>::type codes_t;
  const uint32_t row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= b.rows) return;
  uint32_t seq;
  int64_t pos;
  if (!find_row_wave(b, row, seq, pos)) return;  // uniform
  const uint32_t phys = find_block(b, seq, pos);
  const uint32_t per_head = b.dim / E, pieces = b.n_kv * per_head;
  vec* kd = reinterpret_cast<vec*>(ko) + (uint64_t)row * pieces;
  vec* vd = reinterpret_cast<vec*>(vo) + (uint64_t)row * pieces;
  constexpr int P = SPREAD ? 1 : kPieces, W = SPREAD ? 1 : 2;  // pieces a lane, and K and V of each
  const uint32_t first = SPREAD ? blockIdx.y / 2 * 64 : 0, last = SPREAD ? min(first + 64, pieces) : pieces;
  vec* const d0 = SPREAD && (blockIdx.y & 1) ? vd : kd;
  const uint8_t* const p0 = SPREAD && (blockIdx.y & 1) ? vp : kp;
  if (phys == ~0u) {
    for (uint32_t u = first + lane; u < last; u += 64) {
      d0[u] = vec{};
      if (!SPREAD) vd[u] = vec{};
    }
    return;
  }
  const uint32_t slot = (uint32_t)pos % b.block_size;
  const uint64_t page = nfhip::page_bytes(PT, (uint64_t)b.block_size * b.dim), block = (uint64_t)phys * b.n_kv * page;
  for (uint32_t u0 = first; u0 < last; u0 += 64 * P) {
    vec x[P][W];
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const uint32_t u = u0 + 64 * i + lane < pieces ? u0 + 64 * i + lane : pieces - 1;
      const uint32_t head = u / per_head, el = slot * b.dim + (u - head * per_head) * E;
      const uint64_t at = block + head * page;
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const uint8_t* p = (j ? vp : p0) + at;
        if constexpr (PT != PoolType::I8) {
          x[i][j] = *reinterpret_cast<const vec*>(p + (uint64_t)el * sizeof(T));
        } else {
          const codes_t c = *reinterpret_cast<const codes_t*>(p + el);
          const float d = (float)*reinterpret_cast<const half_t*>(p + (uint64_t)b.block_size * b.dim + el / 32 * 2);
#pragma unroll
          for (uint32_t e = 0; e < E; ++e) {
            uint32_t word;
            if constexpr (E == 8) word = e < 4 ? c.x : c.y;
            else word = c;
            x[i][j][e] = (T)(d * (float)(int)(int8_t)(word >> (8 * (e % 4))));
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const uint32_t u = u0 + 64 * i + lane;
      if (u < last) {
        d0[u] = x[i][0];
        if (!SPREAD) vd[u] = x[i][W - 1];
      }
    }
  }
}

// Whole 16-byte pieces in rows and pages, and for I8 codes at multiples of 8 bytes.
template <typename T, PoolType PT>
bool pieces_fit(const PagedBatch& b, const void* k, const void* v, const void* kp, const void* vp) {
  const uintptr_t all = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                        reinterpret_cast<uintptr_t>(kp) | reinterpret_cast<uintptr_t>(vp);
  return all % 16 == 0 && b.dim % Piece<T>::kElems == 0 &&
         (PT != PoolType::I8 || nfhip::page_bytes(PT, (uint64_t)b.block_size * b.dim) % 8 == 0);
}

// Slices of 64 pieces in a row.
template <typename T>
uint32_t slices(const PagedBatch& b) {
  return (b.n_kv * (b.dim / Piece<T>::kElems) + 63) / 64;
}

template <typename T, PoolType PT>
hipError_t append(const PagedBatch& b, const void* kn, const void* vn, void* kp, void* vp, hipStream_t s) {
  if (pieces_fit<T, PT>(b, kn, vn, kp, vp)) {
    const bool spread = b.rows <= kSpreadRows && slices<T>(b) <= 32767;  // the grid's y ends at 65535
    auto* kernel = spread ? append_kernel<T, PT, true> : append_kernel<T, PT, false>;
    kernel<<<dim3((b.rows + 3) / 4, spread ? 2 * slices<T>(b) : 1), 256, 0, s>>>(b, (const T*)kn, (const T*)vn,
                                                                                 (uint8_t*)kp, (uint8_t*)vp);
    return hipGetLastError();
  }
  const uint64_t n = (uint64_t)b.rows * b.n_kv * (PT == PoolType::I8 ? b.dim / 32 : b.dim);
  append_any_kernel<T, PT><<<dim3((unsigned)((n + 255) / 256), 2), 256, 0, s>>>(
      b, (const T*)kn, (const T*)vn, (uint8_t*)kp, (uint8_t*)vp);
  return hipGetLastError();
}

template <typename T, PoolType PT>
hipError_t gather(const PagedBatch& b, const void* kp, const void* vp, void* ko, void* vo, hipStream_t s) {
  if (pieces_fit<T, PT>(b, ko, vo, kp, vp)) {
    const bool spread = b.rows <= kSpreadRows && slices<T>(b) <= 32767;  // the grid's y ends at 65535
    auto* kernel = spread ? gather_kernel<T, PT, true> : gather_kernel<T, PT, false>;
    kernel<<<dim3((b.rows + 3) / 4, spread ? 2 * slices<T>(b) : 1), 256, 0, s>>>(b, (const uint8_t*)kp,
                                                                                 (const uint8_t*)vp, (T*)ko, (T*)vo);
    return hipGetLastError();
  }
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
