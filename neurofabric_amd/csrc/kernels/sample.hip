// sample.hip — the next token of each row of logits from a given random number
// (sample_token).
//
// With x the row's logits, T its temperature and m = max x, token i has the
// weight w_i = rint(2^40 exp((x_i - m) / T)), an integer, formed in 64 bits.
// Sums of weights are integer sums, so no result depends on the order in which
// threads add, and a token less likely than 2^-41 of the likeliest is never
// drawn.  In the order of x descending, index ascending:
//   1. the first top_k tokens stay (top_k <= 0 or >= n: all);
//   2. of them the shortest prefix whose weights sum to top_p of theirs
//      (top_p >= 1: all; at least one);
//   3. of them those with w_i >= min_p 2^40.
// With S the weights' sum of what stays, the token is the first in index order
// whose running sum exceeds floor(u S); the probability returned is w_i / S.
// T <= 0 takes the first largest logit.  A logit of +inf counts as the largest
// finite value; NaN and -inf are never drawn, and a row of nothing else gives
// token -1 with probability 0.
#include "../launch.hpp"
#include "common.hpp"

namespace nfk {
namespace sample {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 2048;
constexpr double kOne = 1099511627776.0;  // 2^40

// Unsigned keys in the order of the logits; 0 for a logit that is never drawn.
// Adding 0 makes -0 the same as +0.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (!(x > -INFINITY)) return 0u;
  const uint32_t u = __builtin_bit_cast(uint32_t, fminf(x + 0.0f, 3.402823466e38f));
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

struct Shared {
  uint64_t mass[kBins];
  uint32_t count[kBins];
  uint64_t scan[kWaves];
  uint64_t found_mass;
  uint32_t found, found_count;
};

template <typename T>
struct Row {
  const T* x;
  uint32_t n;
  float top;        // largest logit
  double inv_t;     // 1 / T
  uint32_t cut;     // tokens of a key above `cut` stay, and those of key `cut`
  uint32_t cut_at;  // at an index of at most `cut_at`
  uint64_t least;   // smallest weight that stays
  __device__ __forceinline__ uint32_t key(uint32_t i) const { return key_of((float)x[i]); }
  __device__ __forceinline__ bool in(uint32_t k, uint32_t i) const { return k > cut || (k == cut && i <= cut_at); }
  __device__ __forceinline__ uint64_t weight(uint32_t k) const {
    if (k == 0) return 0;
    return (uint64_t)rint(exp(((double)value_of(k) - (double)top) * inv_t) * kOne);
  }
  __device__ __forceinline__ uint64_t kept(uint32_t i) const {
    const uint32_t k = key(i);
    if (!in(k, i)) return 0;
    const uint64_t w = weight(k);
    return w >= least ? w : 0;
  }
};

__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor((unsigned long long)v, o);
  return v;
}
// Inclusive sum over the wave's lanes up to this one.
__device__ __forceinline__ uint64_t wave_scan64(uint64_t v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t t = __shfl_up((unsigned long long)v, o);
    if (lane >= o) v += t;
  }
  return v;
}

// The first index i whose running sum of f(0) .. f(i) exceeds want(total), for
// want < total; f is non-negative.  The sixteen waves sum a sixteenth of the
// range each, then a sixteenth of the one that holds the index, and so on.
template <class F, class W>
__device__ uint32_t locate(Shared& sh, uint32_t n, F f, W want, uint64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t lo = 0, len = n;
  uint64_t t = 0;
  bool first = true;
  total = 0;
  for (;;) {
    const uint32_t step = (len + kWaves - 1) / kWaves;
    const uint32_t a = min(lo + step * wave, lo + len), e = min(a + step, lo + len);
    uint64_t v = 0;
    for (uint32_t i = a + lane; i < e; i += 64) v += f(i);
    v = wave_sum64(v);
    __syncthreads();
    if (lane == 0) sh.scan[wave] = v;
    __syncthreads();
    if (first) {
      for (int w = 0; w < kWaves; ++w) total += sh.scan[w];
      t = want(total);
      if (t >= total) return n;
      first = false;
    }
    uint64_t before = 0;
    int w = 0;
    for (; w < kWaves - 1; ++w) {
      if (before + sh.scan[w] > t) break;
      before += sh.scan[w];
    }
    t -= before;
    lo += step * w;
    len = min(step, n - lo);
    if (len <= 64) break;
  }
  const uint64_t up = wave_scan64(lane < (int)len ? f(lo + lane) : 0);
  return lo + (uint32_t)__builtin_ctzll(__ballot(up > t));
}

// Of the tokens that `r` keeps so far, the key at which the running sum of
// counts (BY_MASS: of weights) from the largest key down reaches `target`: in
// sh.found, with the sum over the larger keys in sh.found_mass.  Three passes
// over the key's bits, 11, 11 and 10.
template <bool BY_MASS, typename T, class TGT>
__device__ void select(Shared& sh, const Row<T>& r, TGT target) {
  uint32_t prefix = 0;
  uint64_t above = 0;
  double goal = 0;
  int hi = 32;
  for (int level = 0; level < 3; ++level) {
    const int bits = level < 2 ? 11 : 10, lo = hi - bits;
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.mass[i] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < r.n; i += kThreads) {
      const uint32_t k = r.key(i);
      if (k == 0 || !r.in(k, i) || (hi < 32 && (k >> hi) != prefix)) continue;
      atomicAdd((unsigned long long*)&sh.mass[(k >> lo) & ((1u << bits) - 1)], BY_MASS ? r.weight(k) : 1ull);
    }
    __syncthreads();
    // bins from the largest down: thread t has bins 2047 - 2t and 2046 - 2t
    const int b0 = kBins - 1 - 2 * (int)threadIdx.x, b1 = b0 - 1;
    const uint64_t v0 = sh.mass[b0], v1 = sh.mass[b1];
    uint64_t up = wave_scan64(v0 + v1);
    if ((threadIdx.x & 63) == 63) sh.scan[threadIdx.x >> 6] = up;
    __syncthreads();
    uint64_t before = above + up - v0 - v1, total = 0;
    for (int w = 0; w < kWaves; ++w) {
      if (w < (int)(threadIdx.x >> 6)) before += sh.scan[w];
      total += sh.scan[w];
    }
    if (level == 0) goal = target(total);
    if ((double)before < goal && (double)(before + v0) >= goal) {
      sh.found = b0;
      sh.found_mass = before;
    }
    if ((double)(before + v0) < goal && (double)(before + v0 + v1) >= goal) {
      sh.found = b1;
      sh.found_mass = before + v0;
    }
    __syncthreads();
    prefix = hi == 32 ? sh.found : (prefix << bits) | sh.found;
    above = sh.found_mass;
    hi = lo;
    __syncthreads();
  }
  if (threadIdx.x == 0) sh.found = prefix;
  __syncthreads();
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_row_kernel(const T* __restrict__ logits, const float* __restrict__ u,
                                                              const float* __restrict__ params,
                                                              const int32_t* __restrict__ top_k,
                                                              int32_t* __restrict__ token, float* __restrict__ prob,
                                                              uint32_t n) {
  __shared__ Shared sh;
  const uint32_t row = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Row<T> r;
  r.x = logits + (uint64_t)row * n;
  r.n = n;
  const float temp = params[3 * row], top_p = params[3 * row + 1], min_p = params[3 * row + 2];
  const int32_t k = top_k[row];
  // the largest key, and its first index
  uint32_t best = 0;
  for (uint32_t i = threadIdx.x; i < n; i += kThreads) best = max(best, r.key(i));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) best = max(best, (uint32_t)__shfl_xor((int)best, o));
  if (lane == 0) sh.scan[wave] = best;
  __syncthreads();
  best = 0;
  for (int w = 0; w < kWaves; ++w) best = max(best, (uint32_t)sh.scan[w]);
  if (best == 0) {  // nothing to draw
    if (threadIdx.x == 0) {
      token[row] = -1;
      prob[row] = 0.0f;
    }
    return;
  }
  r.top = value_of(best);
  r.cut = 1;  // every key but 0
  r.cut_at = n;
  r.least = 0;
  uint64_t total;
  if (!(temp > 0.0f)) {
    const uint32_t at = locate(sh, n, [&](uint32_t i) -> uint64_t { return r.key(i) == best; },
                               [](uint64_t) -> uint64_t { return 0; }, total);
    if (threadIdx.x == 0) {
      token[row] = (int32_t)at;
      prob[row] = 1.0f;
    }
    return;
  }
  r.inv_t = 1.0 / (double)temp;
  const bool one = top_p <= 0.0f;  // the shortest prefix is the first token
  if (one || (k > 0 && (uint32_t)k < n)) {
    const double want = one ? 1.0 : (double)k;
    __syncthreads();
    select<false>(sh, r, [&](uint64_t valid) { return want < (double)valid ? want : (double)valid; });
    const uint32_t key = sh.found;
    const uint64_t more = (uint64_t)want - sh.found_mass;  // tokens of this key that stay, if there are as many
    const uint32_t at = locate(sh, n, [&](uint32_t i) -> uint64_t { return r.key(i) == key; },
                               [&](uint64_t ties) -> uint64_t { return (more < ties ? more : ties) - 1; }, total);
    r.cut = key;
    r.cut_at = at;
  }
  if (!one && top_p < 1.0f) {
    double goal = 0;
    __syncthreads();
    select<true>(sh, r, [&](uint64_t sum) { return goal = (double)top_p * (double)sum; });
    const uint32_t key = sh.found;
    const uint64_t above = sh.found_mass, w = r.weight(key);
    // the j-th token of this key stays while the sum before it is below the goal
    const uint32_t at = locate(
        sh, n, [&](uint32_t i) -> uint64_t { return r.key(i) == key && r.in(key, i); },
        [&](uint64_t ties) -> uint64_t {
          uint64_t lo = 0, hi = ties - 1;  // the last j with above + j w below the goal
          while (lo < hi) {
            const uint64_t mid = (lo + hi + 1) / 2;
            if ((double)(above + mid * w) < goal) lo = mid;
            else hi = mid - 1;
          }
          return lo;
        },
        total);
    r.cut = key;
    r.cut_at = at;
  }
  if (min_p > 0.0f) r.least = (uint64_t)ceil(fmin((double)min_p, 1.0) * kOne);
  const double draw = (double)u[row];
  const uint32_t at = locate(sh, n, [&](uint32_t i) { return r.kept(i); },
                             [&](uint64_t sum) -> uint64_t {
                               const double t = floor(draw * (double)sum);
                               if (!(t > 0.0)) return 0;
                               return t < (double)sum ? min((uint64_t)t, sum - 1) : sum - 1;
                             },
                             total);
  if (threadIdx.x == 0) {
    token[row] = (int32_t)at;
    prob[row] = (float)((double)r.kept(at) / (double)total);
  }
}

}  // namespace sample
}  // namespace nfk

namespace nfhip {

hipError_t launch_sample(EType t, const void* logits, const float* u, const float* params, const int32_t* top_k,
                         int32_t* token, float* prob, uint32_t rows, uint32_t n, const Workspace&, hipStream_t s) {
  using namespace nfk;
  if (rows == 0) return hipSuccess;
  if (t == EType::F16)
    sample::sample_row_kernel<<<dim3(rows), sample::kThreads, 0, s>>>((const half_t*)logits, u, params, top_k, token,
                                                                      prob, n);
  else
    sample::sample_row_kernel<<<dim3(rows), sample::kThreads, 0, s>>>((const float*)logits, u, params, top_k, token,
                                                                      prob, n);
  return hipGetLastError();
}

}  // namespace nfhip
