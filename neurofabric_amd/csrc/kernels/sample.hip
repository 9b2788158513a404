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
constexpr int kBins = 2048;     // digits of select()
constexpr int kBuckets = 1024;  // buckets of the histogram of a row's logits
constexpr int kList = 2048;     // candidates that are sorted in LDS
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

// exp2 of y <= 0 in 64 bits: 2^n times the Taylor series of 2^r, |r| <= 1/2, to the
// 12th power (the next term is below 2^-52).  Times 2^40 and rounded to an integer
// by the addition of 2^52, whose low bits then hold it.
struct Taylor {
  double c[13];
  constexpr Taylor() : c() {
    c[0] = 1.0;
    for (int k = 1; k < 13; ++k) c[k] = c[k - 1] * 0.693147180559945309417232 / k;
  }
};
__device__ __forceinline__ uint64_t weight_of(double y) {
  if (!(y > -42.0)) return 0;
  constexpr Taylor t;
  const double n = rint(y), r = y - n;
  double p = t.c[12];
#pragma unroll
  for (int k = 11; k >= 0; --k) p = __builtin_fma(p, r, t.c[k]);
  const uint64_t bits = __builtin_bit_cast(uint64_t, p) + ((uint64_t)((int64_t)(int)n + 40) << 52);  // p 2^(n + 40)
  return __builtin_bit_cast(uint64_t, __builtin_bit_cast(double, bits) + 4503599627370496.0) & ((1ull << 52) - 1);
}

// A row and what its parameters ask for.
template <typename T>
struct Row {
  const T* x;
  uint32_t n;
  uint32_t k;        // tokens that top_k leaves; 0: all
  double top_p;      // 1: all
  bool greedy;
  uint64_t least;    // smallest weight that stays
  double log2e_t;    // log2(e) / T
  float inv_width;   // buckets per unit of logit
  uint32_t best;     // largest key
  float top;         // its logit
  uint32_t cut;      // tokens of a key above `cut` stay, and those of key `cut`
  uint32_t cut_at;   // at an index of at most `cut_at`

  __device__ __forceinline__ Row(const T* logits, uint32_t row, uint32_t n_, const float* params, const int32_t* top_k)
      : x(logits + (uint64_t)row * n_), n(n_), cut(1), cut_at(n_) {
    const float temp = params[3 * row], p = params[3 * row + 1], m = params[3 * row + 2];
    const int32_t kk = top_k[row];
    greedy = !(temp > 0.0f);
    k = p <= 0.0f ? 1u : kk > 0 && (uint32_t)kk < n ? (uint32_t)kk : 0u;  // the shortest prefix is the first token
    top_p = p > 0.0f && p < 1.0f ? (double)p : 1.0;
    least = m > 0.0f ? (uint64_t)ceil(fmin((double)m, 1.0) * kOne) : 0;
    log2e_t = 1.4426950408889634074 / (double)temp;
    // kBuckets buckets over the logits that have a weight: exp(-28.5) 2^40 < 1/2
    inv_width = fminf((float)kBuckets / (28.5f * temp), 3.402823466e38f);
  }
  __device__ __forceinline__ void set_top(uint32_t key) {
    best = key;
    top = value_of(key);
  }
  __device__ __forceinline__ uint32_t key(uint32_t i) const { return key_of((float)x[i]); }
  __device__ __forceinline__ bool in(uint32_t k_, uint32_t i) const { return k_ > cut || (k_ == cut && i <= cut_at); }
  __device__ __forceinline__ uint64_t weight(uint32_t k_) const {
    return k_ == 0 ? 0 : weight_of(((double)value_of(k_) - (double)top) * log2e_t);
  }
  __device__ __forceinline__ uint64_t kept(uint32_t i) const {
    const uint32_t k_ = key(i);
    if (!in(k_, i)) return 0;
    const uint64_t w = weight(k_);
    return w >= least ? w : 0;
  }
  // Bucket of a key, 0 at the top, monotone in the logit; kBuckets or more: no weight.
  __device__ __forceinline__ uint32_t bucket(uint32_t k_) const {
    if (k_ == 0) return kBuckets;
    const float z = (top - value_of(k_)) * inv_width;
    return z < (float)kBuckets ? (uint32_t)z : kBuckets;
  }
  __device__ __forceinline__ bool cuts() const { return k != 0 || top_p < 1.0; }
  // Whether the buckets' weights are needed: a top_k that fits the list of
  // candidates finds its sums there.
  __device__ __forceinline__ bool wants_mass() const { return k == 0 || k > kList / 2; }
};

// f(logit, index) for the elements lo .. hi - 1, threads in any order, in 16-byte loads.
template <typename T, class F>
__device__ __forceinline__ void each(const T* x, uint32_t lo, uint32_t hi, F f) {
  constexpr uint32_t E = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(E)));
  const uint32_t tid = threadIdx.x, nt = blockDim.x;
  const uint32_t skew = (uint32_t)(reinterpret_cast<uintptr_t>(x + lo) & 15) / sizeof(T);
  uint32_t head = lo + (skew ? E - skew : 0);
  if (head > hi) head = hi;
  if (lo + tid < head) f((float)x[lo + tid], lo + tid);
  const uint32_t nv = (hi - head) / E;
  const vec* xv = reinterpret_cast<const vec*>(x + head);
#pragma unroll 4
  for (uint32_t v = tid; v < nv; v += nt) {
    const vec t = xv[v];
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) f((float)t[e], head + v * E + e);
  }
  const uint32_t tail = head + nv * E + tid;
  if (tail < hi) f((float)x[tail], tail);
}

__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor((unsigned long long)v, o);
  return v;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
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

struct Shared {
  uint64_t mass[kBins];       // select(): weights or counts by digit; histogram: weights by bucket
  uint32_t count[kBuckets];   // histogram: tokens by bucket
  uint64_t list[kList];       // candidates: key << 32 | ~index, or index << 32 | place
  uint64_t weight[kList];
  uint64_t scan[kWaves];
  uint64_t found_mass;
  uint32_t found, n_list;
};

// Inclusive sum over the workgroup's threads up to this one, and the total.
__device__ __forceinline__ uint64_t block_scan64(Shared& sh, uint64_t v, uint64_t& total) {
  const int wave = threadIdx.x >> 6;
  uint64_t up = wave_scan64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) sh.scan[wave] = up;
  __syncthreads();
  total = 0;
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) up += sh.scan[w];
    total += sh.scan[w];
  }
  return up;
}

// The first index i of [lo, lo + len) whose running sum of f(lo) .. f(i) exceeds
// want(total), for want < total; f is non-negative.  The sixteen waves sum a
// sixteenth of the range each, then a sixteenth of the one that holds the index,
// and so on.
template <class F, class W>
__device__ uint32_t locate(Shared& sh, uint32_t lo, uint32_t len, F f, W want, uint64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t stop = lo + len;
  uint64_t t = 0;
  bool first = true;
  total = 0;
  for (;;) {
    const uint32_t step = (len + kWaves - 1) / kWaves;
    const uint32_t a = min(lo + step * wave, lo + len), e = min(a + step, lo + len);
    uint64_t v = 0;
#pragma unroll 4
    for (uint32_t i = a + lane; i < e; i += 64) v += f(i);
    v = wave_sum64(v);
    __syncthreads();
    if (lane == 0) sh.scan[wave] = v;
    __syncthreads();
    if (first) {
      for (int w = 0; w < kWaves; ++w) total += sh.scan[w];
      t = want(total);
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
    len = min(step, stop - lo);
    if (len <= 64) break;
  }
  const uint64_t up = wave_scan64(lane < (int)len ? f(lo + lane) : 0);
  const uint64_t past = __ballot(up > t);
  return lo + (past ? (uint32_t)__builtin_ctzll(past) : len - 1);
}

// Bitonic sort of list[0 .. n), n a power of two, largest first (DOWN) or last.
template <bool DOWN>
__device__ void sort(uint64_t* list, uint32_t n) {
  for (uint32_t size = 2; size <= n; size <<= 1)
    for (uint32_t d = size >> 1; d > 0; d >>= 1) {
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < n / 2; i += kThreads) {
        const uint32_t a = 2 * i - (i & (d - 1)), b = a + d;
        const uint64_t x = list[a], y = list[b];
        const bool up = ((a & size) == 0) != DOWN;
        if ((x > y) == up) {
          list[a] = y;
          list[b] = x;
        }
      }
    }
  __syncthreads();
}
__device__ __forceinline__ uint32_t pow2_of(uint32_t n) { return n <= 1 ? 1u : 1u << (32 - __builtin_clz(n - 1)); }

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
  __syncthreads();
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
    uint64_t total;
    const uint64_t before = above + block_scan64(sh, v0 + v1, total) - v0 - v1;
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

// The cuts by passes over the row alone, whatever the logits.
template <typename T>
__device__ void cut_by_passes(Shared& sh, Row<T>& r) {
  uint64_t total;
  if (r.k != 0) {
    const double want = (double)r.k;
    select<false>(sh, r, [&](uint64_t valid) { return want < (double)valid ? want : (double)valid; });
    const uint32_t key = sh.found;
    const uint64_t more = r.k - sh.found_mass;  // tokens of this key that stay, if there are as many
    const uint32_t at = locate(sh, 0, r.n, [&](uint32_t i) -> uint64_t { return r.key(i) == key; },
                               [&](uint64_t ties) -> uint64_t { return (more < ties ? more : ties) - 1; }, total);
    r.cut = key;
    r.cut_at = at;
  }
  if (r.top_p < 1.0) {
    double goal = 0;
    select<true>(sh, r, [&](uint64_t sum) { return goal = r.top_p * (double)sum; });
    const uint32_t key = sh.found;
    const uint64_t above = sh.found_mass, w = r.weight(key);
    // the j-th token of this key stays while the sum before it is below the goal
    const uint32_t at = locate(
        sh, 0, r.n, [&](uint32_t i) -> uint64_t { return r.key(i) == key && r.in(key, i); },
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
}

// Candidates of the buckets first .. last into sh.list, sorted, largest first;
// their number (known to be at most kList).
template <typename T>
__device__ uint32_t collect(Shared& sh, const Row<T>& r, uint32_t first, uint32_t last) {
  __syncthreads();
  if (threadIdx.x == 0) sh.n_list = 0;
  __syncthreads();
  each(r.x, 0, r.n, [&](float x, uint32_t i) {
    const uint32_t key = key_of(x), b = r.bucket(key);
    if (b < first || b > last || !r.in(key, i)) return;
    const uint32_t at = atomicAdd(&sh.n_list, 1u);
    if (at < (uint32_t)kList) sh.list[at] = (uint64_t)key << 32 | (uint32_t)~i;
  });
  __syncthreads();
  const uint32_t n = min(sh.n_list, (uint32_t)kList), p = pow2_of(n);
  for (uint32_t i = n + threadIdx.x; i < p; i += kThreads) sh.list[i] = 0;
  sort<true>(sh.list, p);
  return n;
}

// floor(u S), within 0 .. S - 1.
__device__ __forceinline__ uint64_t draw_at(double u, uint64_t sum) {
  const double t = floor(u * (double)sum);
  if (!(t > 0.0)) return 0;
  return t < (double)sum ? min((uint64_t)t, sum - 1) : sum - 1;
}

// The token and its weight from the sorted candidates sh.list[0 .. n), which are
// the first tokens in order; `sum`: the weights that top_p goes by (0: theirs).
template <typename T>
__device__ void draw_from_list(Shared& sh, const Row<T>& r, uint32_t n, uint64_t sum, double u, int32_t* token, float* prob) {
  constexpr int P = kList / kThreads;
  if (r.k != 0 && r.k < n) n = r.k;
  const uint32_t i0 = threadIdx.x * P;
  uint64_t w[P], mine = 0, total;
#pragma unroll
  for (int e = 0; e < P; ++e) {
    w[e] = i0 + e < n ? r.weight((uint32_t)(sh.list[i0 + e] >> 32)) : 0;
    mine += w[e];
  }
  uint64_t before = block_scan64(sh, mine, total) - mine;
  const double goal = r.top_p * (double)(sum ? sum : total);
  mine = 0;
  uint32_t last = 0;  // tokens that stay are among the first `last`
#pragma unroll
  for (int e = 0; e < P; ++e) {
    const bool stays = i0 + e < n && (i0 + e == 0 || r.top_p >= 1.0 || (double)before < goal) && w[e] >= r.least;
    before += w[e];
    if (!stays) w[e] = 0;
    if (w[e]) last = i0 + e + 1;
    mine += w[e];
  }
  block_scan64(sh, mine, total);
  // by index: list = index << 32 | place, weights by place
  last = wave_max(last);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.scan[threadIdx.x >> 6] = last;
  uint64_t entry[P];
#pragma unroll
  for (int e = 0; e < P; ++e) {
    sh.weight[i0 + e] = w[e];
    entry[e] = w[e] ? (uint64_t)(uint32_t)~(uint32_t)sh.list[i0 + e] << 32 | (i0 + e) : ~0ull;
  }
  __syncthreads();
  for (int v = 0; v < kWaves; ++v) last = max(last, (uint32_t)sh.scan[v]);
  const uint32_t p = pow2_of(last);
#pragma unroll
  for (int e = 0; e < P; ++e) sh.list[i0 + e] = entry[e];
  sort<false>(sh.list, p);
  const uint64_t t = draw_at(u, total);
  mine = 0;
#pragma unroll
  for (int e = 0; e < P; ++e) {
    w[e] = i0 + e < p && sh.list[i0 + e] != ~0ull ? sh.weight[(uint32_t)sh.list[i0 + e]] : 0;
    mine += w[e];
  }
  uint64_t all;
  before = block_scan64(sh, mine, all) - mine;
#pragma unroll
  for (int e = 0; e < P; ++e) {
    if (before <= t && before + w[e] > t) {
      *token = (int32_t)(sh.list[i0 + e] >> 32);
      *prob = (float)((double)w[e] / (double)total);
    }
    before += w[e];
  }
}

// A bucket of the histogram in sh: the first whose running sum of counts (BY_MASS: of
// weights) reaches the goal, the sum before it in sh.found_mass; kBuckets if none does.
template <bool BY_MASS>
__device__ uint32_t find_bucket(Shared& sh, double goal, uint64_t& total) {
  static_assert(kBuckets == kThreads, "a bucket per thread");
  const uint64_t v = BY_MASS ? sh.mass[threadIdx.x] : sh.count[threadIdx.x];
  const uint64_t upto = block_scan64(sh, v, total);
  if (threadIdx.x == 0) sh.found = kBuckets;
  __syncthreads();
  if ((double)(upto - v) < goal && (double)upto >= goal) {
    sh.found = threadIdx.x;
    sh.found_mass = upto - v;
  }
  __syncthreads();
  return sh.found;
}

// Cuts the row inside bucket `b` (few enough candidates for the list) so that tokens
// stay while fewer than `more` of it (BY_MASS: weights below `goal` with `above` before
// it) have; the weights of those that stay are returned.
template <bool BY_MASS, typename T>
__device__ uint64_t cut_bucket(Shared& sh, Row<T>& r, uint32_t b, uint64_t above, uint64_t more, double goal) {
  constexpr int P = kList / kThreads;
  const uint32_t n = collect(sh, r, b, b);
  const uint32_t i0 = threadIdx.x * P;
  uint64_t w[P], mine = 0, total;
#pragma unroll
  for (int e = 0; e < P; ++e) {
    w[e] = i0 + e < n ? r.weight((uint32_t)(sh.list[i0 + e] >> 32)) : 0;
    mine += w[e];
  }
  uint64_t before = above + block_scan64(sh, mine, total) - mine;
  uint32_t last = 0;
  mine = 0;
#pragma unroll
  for (int e = 0; e < P; ++e) {
    if (i0 + e < n && (BY_MASS ? (double)before < goal : i0 + e < more)) {
      last = i0 + e + 1;
      mine += w[e];
    }
    before += w[e];
  }
  block_scan64(sh, mine, total);
  last = wave_max(last);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.scan[threadIdx.x >> 6] = last;
  __syncthreads();
  for (int v = 0; v < kWaves; ++v) last = max(last, (uint32_t)sh.scan[v]);
  const uint64_t at = sh.list[last - 1];
  r.cut = (uint32_t)(at >> 32);
  r.cut_at = (uint32_t)~(uint32_t)at;
  return total;
}

// The chunks that the two passes over a row's logits are spread over: each leaves
// its largest key, then its buckets' counts and weights and the sum of its weights
// that min_p leaves.
struct Part {
  uint64_t sum;
  uint64_t mass[kBuckets];
  uint32_t count[kBuckets];
  uint32_t best, pad;
};

template <typename T>
__device__ __forceinline__ uint32_t chunk_best(const Row<T>& r, uint32_t lo, uint32_t hi) {
  uint32_t best = 0;
  each(r.x, lo, hi, [&](float x, uint32_t) { best = max(best, key_of(x)); });
  return wave_max(best);
}

// Counts, and if they are wanted weights, of a chunk into LDS (zeroed); the thread's
// sum of the weights that min_p leaves.
template <typename T>
__device__ __forceinline__ uint64_t chunk_histogram(const Row<T>& r, uint32_t lo, uint32_t hi, uint32_t* count, uint64_t* mass) {
  uint64_t sum = 0;
  if (!r.cuts()) {
    each(r.x, lo, hi, [&](float x, uint32_t) {
      const uint64_t w = r.weight(key_of(x));
      sum += w >= r.least ? w : 0;
    });
  } else if (!r.wants_mass()) {
    each(r.x, lo, hi, [&](float x, uint32_t) {
      const uint32_t b = r.bucket(key_of(x));
      if (b < (uint32_t)kBuckets) atomicAdd(&count[b], 1u);
    });
  } else {
    each(r.x, lo, hi, [&](float x, uint32_t) {
      const uint32_t key = key_of(x), b = r.bucket(key);
      if (b >= (uint32_t)kBuckets) return;
      atomicAdd(&count[b], 1u);
      atomicAdd((unsigned long long*)&mass[b], r.weight(key));
    });
  }
  return sum;
}

constexpr int kChunkThreads = 512;

template <typename T>
__global__ __launch_bounds__(kChunkThreads) void sample_best_kernel(const T* __restrict__ logits,
                                                                    const float* __restrict__ params,
                                                                    const int32_t* __restrict__ top_k, uint32_t n,
                                                                    uint32_t step, Part* __restrict__ parts) {
  __shared__ uint32_t wave_best[kChunkThreads / 64];
  const Row<T> r(logits, blockIdx.y, n, params, top_k);
  const uint32_t lo = blockIdx.x * step, hi = min(n, lo + step);
  const uint32_t best = chunk_best(r, lo, hi);
  if ((threadIdx.x & 63) == 0) wave_best[threadIdx.x >> 6] = best;
  __syncthreads();
  if (threadIdx.x == 0) {
    uint32_t b = 0;
    for (int w = 0; w < kChunkThreads / 64; ++w) b = max(b, wave_best[w]);
    parts[(uint64_t)blockIdx.y * gridDim.x + blockIdx.x].best = b;
  }
}

template <typename T>
__global__ __launch_bounds__(kChunkThreads) void sample_histogram_kernel(const T* __restrict__ logits,
                                                                         const float* __restrict__ params,
                                                                         const int32_t* __restrict__ top_k, uint32_t n,
                                                                         uint32_t step,
                                                                         Part* __restrict__ parts) {
  __shared__ uint64_t mass[kBuckets];
  __shared__ uint32_t count[kBuckets];
  __shared__ uint64_t sums[kChunkThreads / 64];
  Row<T> r(logits, blockIdx.y, n, params, top_k);
  if (r.greedy) return;
  Part* mine = parts + (uint64_t)blockIdx.y * gridDim.x;
  uint32_t best = 0;
  for (uint32_t c = 0; c < gridDim.x; ++c) best = max(best, mine[c].best);
  if (best == 0) return;
  r.set_top(best);
  for (int i = threadIdx.x; i < kBuckets; i += kChunkThreads) {
    mass[i] = 0;
    count[i] = 0;
  }
  __syncthreads();
  const uint32_t lo = blockIdx.x * step, hi = min(n, lo + step);
  const uint64_t sum = wave_sum64(chunk_histogram(r, lo, hi, count, mass));
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum;
  __syncthreads();
  mine += blockIdx.x;
  if (threadIdx.x == 0) {
    uint64_t s = 0;
    for (int w = 0; w < kChunkThreads / 64; ++w) s += sums[w];
    mine->sum = s;
  }
  if (!r.cuts()) return;
  for (int i = threadIdx.x; i < kBuckets; i += kChunkThreads) {
    mine->count[i] = count[i];
    if (r.wants_mass()) mine->mass[i] = mass[i];
  }
}

// A workgroup per row.  Without parts (chunks = 0) it goes over the logits itself.
template <typename T>
__global__ __launch_bounds__(kThreads) void sample_row_kernel(const T* __restrict__ logits, const float* __restrict__ u,
                                                              const float* __restrict__ params,
                                                              const int32_t* __restrict__ top_k,
                                                              int32_t* __restrict__ token, float* __restrict__ prob,
                                                              uint32_t n, uint32_t chunks, uint32_t step,
                                                              const Part* __restrict__ parts) {
  __shared__ Shared sh;
  const uint32_t row = blockIdx.x, tid = threadIdx.x;
  Row<T> r(logits, row, n, params, top_k);
  const Part* mine = parts + (uint64_t)blockIdx.x * chunks;
  uint32_t best = 0;
  if (chunks) {
    for (uint32_t c = tid & 63; c < chunks; c += 64) best = max(best, mine[c].best);
    best = wave_max(best);
  } else {
    best = chunk_best(r, 0, n);
    if ((tid & 63) == 0) sh.scan[tid >> 6] = best;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) best = max(best, (uint32_t)sh.scan[w]);
  }
  if (best == 0) {  // nothing to draw
    if (tid == 0) {
      token[row] = -1;
      prob[row] = 0.0f;
    }
    return;
  }
  r.set_top(best);
  uint64_t total;
  if (r.greedy) {
    uint32_t lo = 0, len = n;
    for (uint32_t c = 0; c < chunks; ++c)
      if (mine[c].best == best) {
        lo = c * step;
        len = min(step, n - lo);
        break;
      }
    const uint32_t at = locate(sh, lo, len, [&](uint32_t i) -> uint64_t { return r.key(i) == best; },
                               [](uint64_t) -> uint64_t { return 0; }, total);
    if (tid == 0) {
      token[row] = (int32_t)at;
      prob[row] = 1.0f;
    }
    return;
  }
  const double draw = (double)u[row];
  if (!r.cuts()) {
    uint32_t lo = 0, len = n;
    uint64_t t = 0, sum = 0;
    if (chunks) {  // the chunk that the running sum passes the draw in
      for (uint32_t c = 0; c < chunks; ++c) sum += mine[c].sum;
      t = draw_at(draw, sum);
      uint64_t before = 0;
      uint32_t c = 0;
      for (; c < chunks - 1; ++c) {
        if (before + mine[c].sum > t) break;
        before += mine[c].sum;
      }
      t -= before;
      lo = c * step;
      len = min(step, n - lo);
    }
    const uint32_t at = locate(sh, lo, len, [&](uint32_t i) { return r.kept(i); },
                               [&](uint64_t s) -> uint64_t { return chunks ? t : draw_at(draw, s); }, total);
    if (tid == 0) {
      token[row] = (int32_t)at;
      prob[row] = (float)((double)r.kept(at) / (double)(chunks ? sum : total));
    }
    return;
  }
  // the histogram
  const bool by_mass = r.wants_mass();
  __syncthreads();
  sh.count[tid] = 0;
  sh.mass[tid] = 0;
  __syncthreads();
  if (chunks) {
    uint32_t cnt = 0;
    uint64_t ms = 0;
    for (uint32_t c = 0; c < chunks; ++c) {
      cnt += mine[c].count[tid];
      if (by_mass) ms += mine[c].mass[tid];
    }
    sh.count[tid] = cnt;
    sh.mass[tid] = ms;
  } else {
    chunk_histogram(r, 0, n, sh.count, sh.mass);
  }
  __syncthreads();
  // the bucket that the first cut ends in, and the candidates up to it
  uint64_t tokens, sum = 0;
  uint32_t b;
  if (r.k) {
    b = find_bucket<false>(sh, (double)r.k, tokens);
  } else {
    uint64_t scanned;
    const uint64_t v = sh.mass[tid];
    block_scan64(sh, v, sum);
    b = find_bucket<true>(sh, r.top_p * (double)sum, scanned);
  }
  uint32_t upto = 0, inside = 0;  // candidates up to bucket b, and in it
  {
    const uint64_t v = tid <= min(b, (uint32_t)kBuckets - 1) ? sh.count[tid] : 0;
    uint64_t all;
    block_scan64(sh, v, all);
    upto = (uint32_t)all;
    inside = b < (uint32_t)kBuckets ? sh.count[b] : 0;
  }
  if (upto <= (uint32_t)kList) {
    const uint32_t c = collect(sh, r, 0, min(b, (uint32_t)kBuckets - 1));
    draw_from_list(sh, r, c, sum, draw, token + row, prob + row);
    return;
  }
  // too many for the list: cut inside the buckets, then draw over the row
  if (inside > (uint32_t)kList || !by_mass) {
    cut_by_passes(sh, r);
  } else {
    const uint64_t above = sh.found_mass;
    if (r.k) {
      if (b < (uint32_t)kBuckets) {
        __syncthreads();
        const uint64_t part = cut_bucket<false>(sh, r, b, 0, r.k - above, 0);
        __syncthreads();
        if (tid == b) sh.mass[tid] = part;
        if (tid > b) sh.mass[tid] = 0;
      }
      if (r.top_p < 1.0) {
        __syncthreads();
        const uint64_t v = sh.mass[tid];
        block_scan64(sh, v, sum);
        const double goal = r.top_p * (double)sum;
        uint64_t scanned;
        const uint32_t bp = find_bucket<true>(sh, goal, scanned);
        if (sh.count[bp] > (uint32_t)kList) cut_by_passes(sh, r);
        else cut_bucket<true>(sh, r, bp, sh.found_mass, 0, goal);
      }
    } else {
      cut_bucket<true>(sh, r, b, above, 0, r.top_p * (double)sum);
    }
  }
  const uint32_t at = locate(sh, 0, n, [&](uint32_t i) { return r.kept(i); },
                             [&](uint64_t s) -> uint64_t { return draw_at(draw, s); }, total);
  if (tid == 0) {
    token[row] = (int32_t)at;
    prob[row] = (float)((double)r.kept(at) / (double)total);
  }
}

template <typename T>
hipError_t launch(const T* logits, const float* u, const float* params, const int32_t* top_k, int32_t* token, float* prob,
                  uint32_t rows, uint32_t n, const nfhip::Workspace& ws, hipStream_t s) {
  const uint64_t fits = ws.part ? ws.part_floats * sizeof(float) / sizeof(Part) : 0;
  // Chunks of a row: enough workgroups for the chip; none where rows alone are, or rows are short.
  uint32_t chunks = rows >= 256 || n <= 8192 ? 0 : (512 + rows - 1) / rows;
  chunks = min(chunks, (n + 4095) / 4096);
  if (chunks <= 1 || fits < (uint64_t)rows * chunks) chunks = 0;
  const uint32_t step = chunks ? ((n + chunks - 1) / chunks + 7) / 8 * 8 : n;
  if (chunks) chunks = (n + step - 1) / step;
  Part* parts = reinterpret_cast<Part*>(ws.part);
  if (chunks) {
    sample_best_kernel<<<dim3(chunks, rows), kChunkThreads, 0, s>>>(logits, params, top_k, n, step, parts);
    sample_histogram_kernel<<<dim3(chunks, rows), kChunkThreads, 0, s>>>(logits, params, top_k, n, step, parts);
  }
  sample_row_kernel<<<dim3(rows), kThreads, 0, s>>>(logits, u, params, top_k, token, prob, n, chunks, step, parts);
  return hipGetLastError();
}

}  // namespace sample
}  // namespace nfk

namespace nfhip {

hipError_t launch_sample(EType t, const void* logits, const float* u, const float* params, const int32_t* top_k,
                         int32_t* token, float* prob, uint32_t rows, uint32_t n, const Workspace& ws, hipStream_t s) {
  using namespace nfk;
  if (rows == 0) return hipSuccess;
  return t == EType::F16 ? sample::launch((const half_t*)logits, u, params, top_k, token, prob, rows, n, ws, s)
                         : sample::launch((const float*)logits, u, params, top_k, token, prob, rows, n, ws, s);
}

}  // namespace nfhip
