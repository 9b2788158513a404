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
// T <= 0 takes the first largest logit; T is taken as at most 1e30.  A logit of +inf
// counts as the largest finite value; NaN and -inf are never drawn, and a row of
// nothing else gives token -1 with probability 0.
#include "../launch.hpp"
#include "common.hpp"

namespace nfk {
namespace sample {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 2048;     // digits of select()
constexpr int kBuckets = 1024;  // buckets of the histogram of a row's logits
constexpr int kList = 2048;     // candidates that are sorted in LDS
// top_k up to which the threads' largest logits bound the candidates (top_k 40 of one row
// of 32000: 13 us, by the histogram 26)
constexpr int kSmallK = 256;
constexpr int kAhead = 2;       // loads a lane has under way while it uses as many
constexpr double kOne = 1099511627776.0;  // 2^40
constexpr float kMostT = 1e30f;  // differences of logits past f32 then have no weight

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
    const float t = params[3 * row], p = params[3 * row + 1], m = params[3 * row + 2];
    const float temp = t > kMostT ? kMostT : t;
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
  __device__ __forceinline__ uint64_t kept(float value, uint32_t i) const {
    const uint32_t k_ = key_of(value);
    if (!in(k_, i)) return 0;
    const uint64_t w = weight(k_);
    return w >= least ? w : 0;
  }
  // Bucket of a logit, 0 at the top, monotone; kBuckets: no weight (or NaN).
  __device__ __forceinline__ uint32_t bucket(float v) const {
    const float z = (top - v) * inv_width;
    return z < (float)kBuckets ? (uint32_t)fmaxf(z, 0.0f) : kBuckets;  // +inf: bucket 0, the largest finite value's
  }
  // The weight of a logit that has a bucket.
  __device__ __forceinline__ uint64_t weight_in(float v) const {
    return weight_of(((double)fminf(v, 3.402823466e38f) - (double)top) * log2e_t);
  }
  __device__ __forceinline__ bool cuts() const { return k != 0 || top_p < 1.0; }
  // A small top_k needs no histogram of the row: see small_k_bound().
  __device__ __forceinline__ bool small_k() const { return k != 0 && k <= (uint32_t)kSmallK; }
};

// f(logits, first index) for groups of 16 bytes of the elements lo .. hi - 1, by the
// threads in any order; what is past hi in the last group is NaN, which is never
// drawn.  Rows start anywhere, and the loads need no alignment.  kAhead loads are under
// way while the kAhead before them are used: a pass is bound by their latency
// otherwise, and a longer body is itself fetched from memory once a launch (with 2, 4
// and 8, a batch of 64 rows of 128256: 70, 72 and 74 us; one row of 32000: 12.6, 12.9
// and 13.5).
template <typename T>
struct Group {
  static constexpr uint32_t kElems = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};
template <typename T, class F>
__device__ __forceinline__ void each_group(const T* x, uint32_t lo, uint32_t hi, F f) {
  constexpr uint32_t E = Group<T>::kElems;
  typedef typename Group<T>::vec vec;
  const uint32_t whole = (hi - lo) / E, nt = blockDim.x;
  const vec* xv = reinterpret_cast<const vec*>(x + lo);
  if (whole) {
    uint32_t g = threadIdx.x;
    vec t[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) t[j] = xv[min(g + j * nt, whole - 1)];
#pragma unroll 1
    for (; g < whole; g += kAhead * nt) {
      vec now[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) now[j] = t[j];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) t[j] = xv[min(g + (kAhead + j) * nt, whole - 1)];
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (g + j * nt < whole) f(now[j], lo + (g + j * nt) * E);
    }
  }
  const uint32_t rest = lo + whole * E;
  if (rest < hi && threadIdx.x == nt - 1) {
    vec t;
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) t[e] = rest + e < hi ? x[rest + e] : (T)__builtin_nanf("");
    f(t, rest);
  }
}

// The lanes' values with the lanes below added, by moves within rows of 16 lanes and
// broadcasts of their last lanes.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp64(uint64_t v) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xF, true);
  return (uint64_t)hi << 32 | lo;
}
// Inclusive sum over the wave's lanes up to this one.
__device__ __forceinline__ uint64_t wave_scan64(uint64_t v) {
  v += dpp64<0x111, 0xF>(v);
  v += dpp64<0x112, 0xF>(v);
  v += dpp64<0x114, 0xF>(v);
  v += dpp64<0x118, 0xF>(v);
  v += dpp64<0x142, 0xA>(v);
  v += dpp64<0x143, 0xC>(v);
  return v;
}
__device__ __forceinline__ uint64_t lane64(uint64_t v, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane) |
         (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane) << 32;
}
__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) { return lane64(wave_scan64(v), 63); }
struct Shared {
  uint64_t mass[kBins];       // weights by bucket, or by index; select(): weights or counts by digit
  uint32_t count[kBuckets];   // tokens by bucket
  uint64_t list[kList];       // candidates: key << 32 | ~index
  uint64_t sub[kBuckets];     // those of one bucket that are left; weights by chunk
  uint64_t sum64[64];         // sum_above()
  uint32_t rank64[64];
  uint64_t scan[2][kWaves];
  uint64_t found_mass, most, least;
  uint32_t found, n_list;
};

// Inclusive sum over the workgroup's threads up to this one, and the total.  `turn`
// alternates between calls, which saves the barrier before the totals are replaced.
__device__ __forceinline__ uint64_t block_scan64(Shared& sh, uint64_t v, uint64_t& total, int turn) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t up = wave_scan64(v);
  if (lane == 63) sh.scan[turn][wave] = up;
  __syncthreads();
  const uint64_t upto = wave_scan64(lane < kWaves ? sh.scan[turn][lane] : 0);
  total = lane64(upto, kWaves - 1);
  return wave ? up + lane64(upto, wave - 1) : up;
}

// The first index i of [lo, lo + len) whose running sum of f(lo) .. f(i) exceeds
// want(total), for want < total; f is non-negative.  The sixteen waves sum a
// sixteenth of the range each, then a sixteenth of the one that holds the index,
// and so on.
template <typename T, class F, class W>
__device__ uint32_t locate(Shared& sh, const T* x, uint32_t lo, uint32_t len, F f, W want, uint64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t stop = lo + len;
  uint64_t t = 0;
  bool first = true;
  total = 0;
  for (;;) {
    const uint32_t step = (len + kWaves - 1) / kWaves;
    const uint32_t a = min(lo + step * wave, lo + len), e = min(a + step, lo + len);
    uint64_t v = 0;
    for (uint32_t i = a + lane; i < e; i += 64 * kAhead) {
      T t[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) t[j] = x[min(i + 64 * j, e - 1)];
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (i + 64 * j < e) v += f((float)t[j], i + 64 * j);
    }
    v = wave_sum64(v);
    __syncthreads();
    if (lane == 0) sh.scan[0][wave] = v;
    __syncthreads();
    if (first) {
      for (int w = 0; w < kWaves; ++w) total += sh.scan[0][w];
      t = want(total);
      first = false;
    }
    uint64_t before = 0;
    int w = 0;
    for (; w < kWaves - 1; ++w) {
      if (before + sh.scan[0][w] > t) break;
      before += sh.scan[0][w];
    }
    t -= before;
    lo += step * w;
    len = min(step, stop - lo);
    if (len <= 64) break;
  }
  const uint64_t up = wave_scan64(lane < (int)len ? f((float)x[lo + lane], lo + lane) : 0);
  const uint64_t past = __ballot(up > t);
  return lo + (past ? (uint32_t)__builtin_ctzll(past) : len - 1);
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
    const uint64_t before = above + block_scan64(sh, v0 + v1, total, 1) - v0 - v1;
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
    const uint32_t at = locate(sh, r.x, 0, r.n, [&](float x, uint32_t) -> uint64_t { return key_of(x) == key; },
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
        sh, r.x, 0, r.n, [&](float x, uint32_t i) -> uint64_t { return key_of(x) == key && r.in(key, i); },
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

// Candidates of the buckets first .. last into sh.list, in no order, as many as fit;
// their number in sh.n_list.
template <typename T>
__device__ __forceinline__ void collect(Shared& sh, const Row<T>& r, uint32_t first, uint32_t last) {
  if (threadIdx.x == 0) sh.n_list = 0;
  __syncthreads();
  // Most logits lie below the last bucket, or above the first: a comparison with a
  // bound that is surely outside sets them aside.
  const float least = r.top - (float)(last + 1) / r.inv_width * 1.00001f;
  const float most = first ? r.top - (float)first / r.inv_width * 0.99999f : INFINITY;
  each_group(r.x, 0, r.n, [&](const typename Group<T>::vec& t, uint32_t i0) {
    bool any = false;
#pragma unroll
    for (uint32_t e = 0; e < Group<T>::kElems; ++e) any |= ((float)t[e] >= least) & ((float)t[e] <= most);
    if (!any) return;
#pragma unroll
    for (uint32_t e = 0; e < Group<T>::kElems; ++e) {
      const uint32_t b = r.bucket((float)t[e]);
      if (b < first || b > last) continue;
      const uint32_t key = key_of((float)t[e]);
      if (!r.in(key, i0 + e)) continue;
      const uint32_t at = atomicAdd(&sh.n_list, 1u);
      if (at < (uint32_t)kList) sh.list[at] = (uint64_t)key << 32 | (uint32_t)~(i0 + e);
    }
  });
  __syncthreads();
}

// floor(u S), within 0 .. S - 1.
__device__ __forceinline__ uint64_t draw_at(double u, uint64_t sum) {
  const double t = floor(u * (double)sum);
  if (!(t > 0.0)) return 0;
  return t < (double)sum ? min((uint64_t)t, sum - 1) : sum - 1;
}

// Of n <= 64 entries, an entry and its weight in lane i of every wave: the sum of the
// weights of those that are larger than the lane's own, and their number.  A wave
// compares all with four of them; the waves' sums meet in LDS.
__device__ __forceinline__ uint64_t sum_above(Shared& sh, uint64_t own, uint64_t w, uint32_t n, uint32_t& rank) {
  const uint32_t tid = threadIdx.x, lane = tid & 63;
  __syncthreads();
  if (tid < 64) {
    sh.sum64[tid] = 0;
    sh.rank64[tid] = 0;
  }
  __syncthreads();
  uint64_t sum = 0;
  uint32_t number = 0;
#pragma unroll
  for (uint32_t i = 0; i < 64 / kWaves; ++i) {
    const uint32_t j = __builtin_amdgcn_readfirstlane(tid >> 6) * (64 / kWaves) + i;
    const bool c = lane64(own, j) > own && j < n;
    sum += c ? lane64(w, j) : 0;
    number += c;
  }
  if (number) {
    atomicAdd((unsigned long long*)&sh.sum64[lane], sum);
    atomicAdd(&sh.rank64[lane], number);
  }
  __syncthreads();
  rank = sh.rank64[lane];
  return sh.sum64[lane];
}

// The token from at most 64 candidates in sh.list.  `sum`: the weights that top_p goes
// by (0: those of the candidates that top_k leaves).
template <typename T>
__device__ void draw_from_few(Shared& sh, const Row<T>& r, uint32_t n, uint64_t sum, double u, int32_t* token, float* prob) {
  const uint32_t lane = threadIdx.x & 63;
  const uint64_t own = lane < n ? sh.list[lane] : 0;
  uint64_t w = lane < n ? r.weight((uint32_t)(own >> 32)) : 0;
  uint32_t rank;
  const uint64_t above = sum_above(sh, own, w, n, rank);
  if (r.k != 0 && rank >= r.k) w = 0;
  const double goal = r.top_p * (double)(sum ? sum : wave_sum64(w));
  if (!((rank == 0 || r.top_p >= 1.0 || (double)above < goal) && w >= r.least)) w = 0;
  const uint64_t total = wave_sum64(w), t = draw_at(u, total);
  // by index: of ~index the larger come first
  const uint64_t before = sum_above(sh, (uint32_t)own, w, n, rank);
  if (threadIdx.x < 64 && before <= t && before + w > t) {
    *token = (int32_t)(uint32_t)~(uint32_t)own;
    *prob = (float)((double)w / (double)total);
  }
}

// The first of sh.count (BY_MASS: sh.mass) whose running sum reaches the goal, in
// sh.found (kBuckets: none does), with the sum before it in sh.found_mass.
template <bool BY_MASS>
__device__ __forceinline__ void find_bucket(Shared& sh, double goal, uint64_t& total) {
  static_assert(kBuckets == kThreads, "a bucket per thread");
  const uint64_t v = BY_MASS ? sh.mass[threadIdx.x] : sh.count[threadIdx.x];
  if (threadIdx.x == 0) sh.found = kBuckets;
  const uint64_t upto = block_scan64(sh, v, total, 0);
  if ((double)(upto - v) < goal && (double)upto >= goal) {
    sh.found = threadIdx.x;
    sh.found_mass = upto - v;
  }
  __syncthreads();
}

// Cuts the row inside bucket `b`, whose candidates are all in sh.list: of them, in
// order, the first `more` stay (BY_MASS: those with less than `goal` before them, the
// sum over the larger buckets being `above`).  Their weights' sum is returned.
// While more than 64 are left, their range is divided into buckets again and the one
// that the cut ends in is kept.
template <bool BY_MASS, typename T>
__device__ uint64_t cut_bucket(Shared& sh, Row<T>& r, uint32_t b, uint64_t above, uint64_t more, double goal) {
  constexpr int P = kList / kThreads;
  const uint32_t tid = threadIdx.x, lane = tid & 63;
  uint64_t c[P], w[P];
  bool left[P], mine[P];
#pragma unroll
  for (int e = 0; e < P; ++e) {
    const uint32_t i = tid + e * kThreads;
    c[e] = i < sh.n_list ? sh.list[i] : 0;
    const uint32_t key = (uint32_t)(c[e] >> 32);
    left[e] = mine[e] = key != 0 && r.bucket(value_of(key)) == b && r.in(key, (uint32_t)~(uint32_t)c[e]);
    w[e] = mine[e] ? r.weight(key) : 0;
  }
  uint64_t n;
  for (;;) {
    uint32_t number = 0;
#pragma unroll
    for (int e = 0; e < P; ++e) number += left[e];
    uint32_t at = (uint32_t)block_scan64(sh, number, n, 0) - number;
    if (n <= 64) {
#pragma unroll
      for (int e = 0; e < P; ++e)
        if (left[e]) sh.sub[at++] = c[e];
      break;
    }
    if (tid == 0) {
      sh.most = 0;
      sh.least = ~0ull;
    }
    sh.sub[tid] = 0;
    __syncthreads();
    uint64_t hi = 0, lo = ~0ull;
#pragma unroll
    for (int e = 0; e < P; ++e)
      if (left[e]) {
        hi = max(hi, c[e]);
        lo = min(lo, c[e]);
      }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      hi = max(hi, (uint64_t)__shfl_xor((unsigned long long)hi, o));
      lo = min(lo, (uint64_t)__shfl_xor((unsigned long long)lo, o));
    }
    if (lane == 0) {
      atomicMax((unsigned long long*)&sh.most, hi);
      atomicMin((unsigned long long*)&sh.least, lo);
    }
    __syncthreads();
    const uint64_t most = sh.most, range = most - sh.least;  // not 0: entries differ
    const int shift = max(0, 54 - __builtin_clzll(range));
#pragma unroll
    for (int e = 0; e < P; ++e)
      if (left[e]) atomicAdd((unsigned long long*)&sh.sub[(most - c[e]) >> shift], BY_MASS ? w[e] : 1ull);
    __syncthreads();
    uint64_t total;
    const uint64_t v = sh.sub[tid], upto = above + block_scan64(sh, v, total, 1);
    if (BY_MASS ? (double)(upto - v) < goal && (double)upto >= goal : upto - v < more && upto >= more) {
      sh.found = tid;
      sh.found_mass = upto - v;
    }
    __syncthreads();
    above = sh.found_mass;
#pragma unroll
    for (int e = 0; e < P; ++e) left[e] = left[e] && (uint32_t)((most - c[e]) >> shift) == sh.found;
    __syncthreads();
  }
  __syncthreads();
  const uint64_t own = lane < n ? sh.sub[lane] : 0, ow = lane < n ? r.weight((uint32_t)(own >> 32)) : 0;
  uint32_t rank;
  const uint64_t before = above + sum_above(sh, own, BY_MASS ? ow : 1, (uint32_t)n, rank);
  const bool stays = lane < n && (BY_MASS ? rank == 0 || (double)before < goal : before < more);
  const uint32_t keep = __popcll(__ballot(stays));
  const uint64_t last = lane64(own, __builtin_ctzll(__ballot(lane < n && rank == keep - 1)));  // the last that stays
  r.cut = (uint32_t)(last >> 32);
  r.cut_at = (uint32_t)~(uint32_t)last;
  uint64_t sum = 0, total;
#pragma unroll
  for (int e = 0; e < P; ++e)
    if (mine[e] && r.in((uint32_t)(c[e] >> 32), (uint32_t)~(uint32_t)c[e])) sum += w[e];
  __syncthreads();
  block_scan64(sh, sum, total, 0);
  __syncthreads();
  return total;
}

// The token, from weights by index: sh.mass holds the sums over 2^shift indices each,
// from index `lo` on.  One wave goes through those of the one that the draw falls in.
// `drawn`: t is the draw, less what lies before `lo`, and `whole` the sum of all; else
// both are formed here.
template <typename T>
__device__ void draw_from_bins(Shared& sh, const Row<T>& r, uint32_t lo, uint32_t hi, uint32_t shift, bool drawn, uint64_t t,
                               uint64_t whole, double u, int32_t* token, float* prob) {
  const uint32_t tid = threadIdx.x, lane = tid & 63;
  uint64_t total;
  const uint64_t v = sh.mass[tid], upto = block_scan64(sh, v, total, 0);
  if (!drawn) {
    whole = total;
    t = draw_at(u, total);
  }
  if (upto - v <= t && upto > t) {
    sh.found = tid;
    sh.found_mass = upto - v;
  }
  __syncthreads();
  if (tid >= 64) return;
  t -= sh.found_mass;
  const uint32_t first = lo + (sh.found << shift);
  for (uint32_t i0 = 0; i0 < (1u << shift); i0 += 64) {
    const uint32_t i = first + i0 + lane;
    const uint64_t w = i < hi && i0 + lane < (1u << shift) ? r.kept((float)r.x[i], i) : 0;
    const uint64_t up = wave_scan64(w), sum = lane64(up, 63);
    if (sum <= t) {
      t -= sum;
      continue;
    }
    if (up - w <= t && up > t) {
      *token = (int32_t)i;
      *prob = (float)((double)w / (double)whole);
    }
    return;
  }
}
// Bins of 2^shift indices for `n` of them.
__device__ __forceinline__ uint32_t bin_shift(uint32_t n) {
  return n <= (uint32_t)kBuckets ? 0 : 32 - __builtin_clz((n - 1) / kBuckets);
}
// The weights of a group's tokens that stay into the bins; a group lies in one or two.
template <typename T>
__device__ __forceinline__ void add_to_bins(Shared& sh, const Row<T>& r, const typename Group<T>::vec& t, uint32_t i0,
                                            uint32_t lo, uint32_t shift) {
  constexpr uint32_t E = Group<T>::kElems;
  uint64_t sum = 0;
  uint32_t at = (i0 - lo) >> shift;
#pragma unroll
  for (uint32_t e = 0; e < E; ++e) {
    const uint32_t bin = (i0 + e - lo) >> shift;
    if (bin != at) {
      if (sum) atomicAdd((unsigned long long*)&sh.mass[at], sum);
      sum = 0;
      at = bin;
    }
    sum += r.kept((float)t[e], i0 + e);
  }
  if (sum) atomicAdd((unsigned long long*)&sh.mass[at], sum);
}

// The chunks that the two passes over a row's logits are spread over: each leaves
// its threads' largest logits, then (without a small top_k) its buckets' counts and
// weights and the sum of its weights that min_p leaves.  Of 64 rows of 128256 in f32 the
// first pass takes 6.7 us (32.8 MB, 4.9 TB/s), the second, bound by the 64-bit
// exponentials and the LDS atomics, 18.6, and the row kernel 45 (below).
constexpr int kChunkThreads = 512;
struct Part {
  uint64_t sum;
  uint64_t mass[kBuckets];
  uint32_t count[kBuckets];
  float top[kChunkThreads];
  float best;
  uint32_t pad;
};

// The largest key of a group's logits so far: fmaxf passes over NaN.
template <typename T>
__device__ __forceinline__ void max_of(float& top, const typename Group<T>::vec& t) {
#pragma unroll
  for (uint32_t e = 0; e < Group<T>::kElems; ++e) top = fmaxf(top, (float)t[e]);
}
__device__ __forceinline__ float wave_maxf(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

// Counts and weights of a group into the histogram; without a cut, the sum of the
// weights that min_p leaves.
template <typename T>
__device__ __forceinline__ void add_to_histogram(const Row<T>& r, const typename Group<T>::vec& t, bool cuts, uint32_t* count,
                                                 uint64_t* mass, uint64_t& sum) {
#pragma unroll
  for (uint32_t e = 0; e < Group<T>::kElems; ++e) {
    const uint32_t b = r.bucket((float)t[e]);
    if (b >= (uint32_t)kBuckets) continue;
    const uint64_t w = r.weight_in((float)t[e]);
    if (!cuts) {
      sum += w >= r.least ? w : 0;
      continue;
    }
    atomicAdd(&count[b], 1u);
    atomicAdd((unsigned long long*)&mass[b], w);
  }
}

template <typename T>
__global__ __launch_bounds__(kChunkThreads) void sample_best_kernel(const T* __restrict__ logits, uint32_t n, uint32_t step,
                                                                    Part* __restrict__ parts) {
  __shared__ float wave_top[kChunkThreads / 64];
  const uint32_t lo = blockIdx.x * step, hi = min(n, lo + step);
  float top = -INFINITY;
  each_group(logits + (uint64_t)blockIdx.y * n, lo, hi,
             [&](const typename Group<T>::vec& t, uint32_t) { max_of<T>(top, t); });
  Part* mine = parts + (uint64_t)blockIdx.y * gridDim.x + blockIdx.x;
  mine->top[threadIdx.x] = top;
  top = wave_maxf(top);
  if ((threadIdx.x & 63) == 0) wave_top[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 0; w < kChunkThreads / 64; ++w) top = fmaxf(top, wave_top[w]);
    mine->best = top;
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
  if (r.greedy || r.small_k()) return;
  Part* mine = parts + (uint64_t)blockIdx.y * gridDim.x;
  float top = -INFINITY;
  for (uint32_t c = 0; c < gridDim.x; ++c) top = fmaxf(top, mine[c].best);
  if (key_of(top) == 0) return;
  r.set_top(key_of(top));
  for (int i = threadIdx.x; i < kBuckets; i += kChunkThreads) {
    mass[i] = 0;
    count[i] = 0;
  }
  __syncthreads();
  const uint32_t lo = blockIdx.x * step, hi = min(n, lo + step);
  uint64_t sum = 0;
  const bool cuts = r.cuts();
  each_group(r.x, lo, hi, [&](const typename Group<T>::vec& t, uint32_t) {
    add_to_histogram(r, t, cuts, count, mass, sum);
  });
  sum = wave_sum64(sum);
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
    mine->mass[i] = mass[i];
  }
}

// A workgroup per row.  Without parts (chunks = 0) it goes over the logits itself.
// A chain of short steps, each waiting for the one before (one row of 32000 with a
// top_k of 40: 12.4 us in all); the longest row of a batch is one with top_p alone,
// whose candidates one CU collects from all of its 0.5 MB (128256 in f32: 12 to 17 of
// about 45 us, then the cut 8, the chunks' sums 4, the draw 9).
template <typename T>
__global__ __launch_bounds__(kThreads) void sample_row_kernel(const T* __restrict__ logits, const float* __restrict__ u,
                                                              const float* __restrict__ params,
                                                              const int32_t* __restrict__ top_k,
                                                              int32_t* __restrict__ token, float* __restrict__ prob,
                                                              uint32_t n, uint32_t chunks, uint32_t step,
                                                              const Part* __restrict__ parts) {
  typedef typename Group<T>::vec vec;
  __shared__ Shared sh;
  const uint32_t row = blockIdx.x, tid = threadIdx.x;
  Row<T> r(logits, row, n, params, top_k);
  const double draw = (double)u[row];
  const Part* mine = parts + (uint64_t)blockIdx.x * chunks;
  token += row;
  prob += row;
  float top = -INFINITY, whole_top;
  if (chunks) {
    for (uint32_t c = tid & 63; c < chunks; c += 64) top = fmaxf(top, mine[c].best);
    whole_top = wave_maxf(top);
  } else {
    each_group(r.x, 0, n, [&](const vec& t, uint32_t) { max_of<T>(top, t); });
    const float w = wave_maxf(top);
    if ((tid & 63) == 0) sh.scan[0][tid >> 6] = __builtin_bit_cast(uint32_t, w);
    __syncthreads();
    whole_top = wave_maxf(__builtin_bit_cast(float, (uint32_t)sh.scan[0][tid & (kWaves - 1)]));
  }
  const uint32_t best = key_of(whole_top);
  if (best == 0) {  // nothing to draw
    if (tid == 0) {
      *token = -1;
      *prob = 0.0f;
    }
    return;
  }
  r.set_top(best);
  uint64_t total;
  if (r.greedy) {
    uint32_t lo = 0, len = n;
    for (uint32_t c = 0; c < chunks; ++c)
      if (key_of(mine[c].best) == best) {
        lo = c * step;
        len = min(step, n - lo);
        break;
      }
    if (tid == 0) sh.found = n;
    __syncthreads();
    uint32_t at = n;
    auto look = [&](const vec& t, uint32_t i0) {
#pragma unroll
      for (uint32_t e = 0; e < Group<T>::kElems; ++e)
        if (key_of((float)t[e]) == best) at = min(at, i0 + e);
    };
    each_group(r.x, lo, lo + len, look);
    if (at < n) atomicMin(&sh.found, at);
    __syncthreads();
    if (tid == 0) {
      *token = (int32_t)sh.found;
      *prob = 1.0f;
    }
    return;
  }
  sh.count[tid] = 0;
  sh.mass[tid] = 0;
  if (!r.cuts()) {
    uint32_t lo = 0, hi = n;
    uint64_t t = 0, sum = 0;
    if (chunks) {  // the chunk that the running sum passes the draw in
      for (uint32_t c = 0; c < chunks; ++c) sum += mine[c].sum;
      t = draw_at(draw, sum);
      uint32_t c = 0;
      for (; c < chunks - 1 && mine[c].sum <= t; ++c) t -= mine[c].sum;
      lo = c * step;
      hi = min(n, lo + step);
    }
    const uint32_t shift = bin_shift(hi - lo);
    __syncthreads();
    auto add = [&](const vec& g, uint32_t i0) { add_to_bins(sh, r, g, i0, lo, shift); };
    each_group(r.x, lo, hi, add);
    __syncthreads();
    draw_from_bins(sh, r, lo, hi, shift, chunks != 0, t, sum, draw, token, prob);
    return;
  }
  uint64_t sum = 0, tokens = 0, all = 0, above = 0;
  uint32_t b;              // the bucket that the first cut ends in
  uint32_t end = kBuckets; // (streamed) tokens of buckets before `end` stay, and of bucket `end` those that the cut leaves
  bool listed, cut = false;
  __syncthreads();
  if (r.small_k()) {
    // The threads' largest logits: where k of them lie, k tokens do.  The candidates
    // up to that bucket are few more than k.
    if (chunks) {
      for (uint32_t i = tid; i < chunks * kChunkThreads; i += kThreads) {
        const uint32_t at = r.bucket(mine[i / kChunkThreads].top[i % kChunkThreads]);
        if (at < (uint32_t)kBuckets) atomicAdd(&sh.count[at], 1u);
      }
    } else {
      const uint32_t at = r.bucket(top);
      if (at < (uint32_t)kBuckets) atomicAdd(&sh.count[at], 1u);
    }
    __syncthreads();
    find_bucket<false>(sh, (double)r.k, tokens);
    collect(sh, r, 0, min(sh.found, (uint32_t)kBuckets - 1));
    listed = sh.n_list <= (uint32_t)kList;
    if (listed && sh.n_list > 64) {  // the exact bucket, among the candidates
      sh.count[tid] = 0;
      __syncthreads();
      for (uint32_t i = tid; i < sh.n_list; i += kThreads)
        atomicAdd(&sh.count[r.bucket(value_of((uint32_t)(sh.list[i] >> 32)))], 1u);
      __syncthreads();
      find_bucket<false>(sh, (double)r.k, tokens);
    }
    b = sh.found;
    above = b < (uint32_t)kBuckets ? sh.found_mass : 0;
  } else {
    if (chunks) {
      uint32_t cnt = 0;
      uint64_t ms = 0;
#pragma unroll 4
      for (uint32_t c = 0; c < chunks; ++c) {
        cnt += mine[c].count[tid];
        ms += mine[c].mass[tid];
      }
      sh.count[tid] = cnt;
      sh.mass[tid] = ms;
    } else {
      uint64_t none = 0;
      each_group(r.x, 0, n, [&](const vec& t, uint32_t) { add_to_histogram(r, t, true, sh.count, sh.mass, none); });
    }
    __syncthreads();
    if (r.k) {
      find_bucket<false>(sh, (double)r.k, tokens);
    } else {
      block_scan64(sh, sh.mass[tid], sum, 1);
      find_bucket<true>(sh, r.top_p * (double)sum, all);
    }
    b = sh.found;  // kBuckets: fewer tokens have a weight than top_k leaves
    above = b < (uint32_t)kBuckets ? sh.found_mass : 0;
    block_scan64(sh, tid <= b ? sh.count[tid] : 0, all, 1);
    listed = all <= (uint64_t)kList;
    cut = b >= (uint32_t)kBuckets && r.top_p >= 1.0;  // nothing is cut
    if (listed) collect(sh, r, 0, min(b, (uint32_t)kBuckets - 1));
    else if (b < (uint32_t)kBuckets && sh.count[b] <= (uint32_t)kList) collect(sh, r, b, b);
  }
  if (listed && sh.n_list <= 64) {
    draw_from_few(sh, r, sh.n_list, sum, draw, token, prob);
    return;
  }
  if (!listed && !cut && (r.small_k() || b >= (uint32_t)kBuckets || sh.count[b] > (uint32_t)kList)) {
    cut_by_passes(sh, r);
    cut = true;
  }
  if (!cut) {
    if (r.k) {
      const uint64_t part = b < (uint32_t)kBuckets ? cut_bucket<false>(sh, r, b, 0, r.k - above, 0) : 0;
      if (r.top_p < 1.0) {
        if (listed) {  // the weights of what top_k leaves, from the list
          sh.mass[tid] = 0;
          __syncthreads();
          for (uint32_t i = tid; i < sh.n_list; i += kThreads) {
            const uint32_t key = (uint32_t)(sh.list[i] >> 32);
            if (r.in(key, (uint32_t)~(uint32_t)sh.list[i]))
              atomicAdd((unsigned long long*)&sh.mass[r.bucket(value_of(key))], r.weight(key));
          }
        } else {
          if (tid == b) sh.mass[tid] = part;
          if (tid > b) sh.mass[tid] = 0;
        }
        __syncthreads();
        block_scan64(sh, sh.mass[tid], sum, 1);
        const double goal = r.top_p * (double)sum;
        find_bucket<true>(sh, goal, all);
        const uint32_t bp = sh.found;
        const uint64_t over = sh.found_mass;
        if (!listed && sh.count[bp] <= (uint32_t)kList) collect(sh, r, bp, bp);
        if (listed || sh.count[bp] <= (uint32_t)kList) cut_bucket<true>(sh, r, bp, over, 0, goal);
        else cut_by_passes(sh, r);
      }
    } else {
      cut_bucket<true>(sh, r, b, above, 0, r.top_p * (double)sum);
      end = b;
    }
  }
  // the draw, from the list, or over the row, or over the chunk that holds the token:
  // its histogram and the tokens of the cut's bucket that stay give each chunk's sum,
  // unless min_p cuts too
  uint32_t lo = 0, hi = n;
  uint64_t t = 0, whole = 0;
  const bool by_chunk = !listed && chunks != 0 && end < (uint32_t)kBuckets && r.least <= 1;
  if (by_chunk) {
    for (uint32_t c = tid; c < chunks; c += kThreads) sh.sub[c] = 0;
    __syncthreads();
    for (uint32_t c = tid >> 6; c < chunks; c += kWaves) {
      uint64_t v = 0;
#pragma unroll 4
      for (uint32_t i = tid & 63; i < end; i += 64) v += mine[c].mass[i];
      v = wave_sum64(v);
      if ((tid & 63) == 0) atomicAdd((unsigned long long*)&sh.sub[c], v);
    }
    for (uint32_t i = tid; i < sh.n_list; i += kThreads) {
      const uint32_t key = (uint32_t)(sh.list[i] >> 32), index = (uint32_t)~(uint32_t)sh.list[i];
      if (r.in(key, index)) atomicAdd((unsigned long long*)&sh.sub[index / step], r.weight(key));
    }
    __syncthreads();
    for (uint32_t c = 0; c < chunks; ++c) whole += sh.sub[c];
    t = draw_at(draw, whole);
    uint32_t c = 0;
    for (; c < chunks - 1 && sh.sub[c] <= t; ++c) t -= sh.sub[c];
    lo = c * step;
    hi = min(n, lo + step);
  }
  const uint32_t shift = bin_shift(hi - lo);
  __syncthreads();
  sh.mass[tid] = 0;
  __syncthreads();
  if (listed) {
    for (uint32_t i = tid; i < sh.n_list; i += kThreads) {
      const uint32_t key = (uint32_t)(sh.list[i] >> 32), index = (uint32_t)~(uint32_t)sh.list[i];
      const uint64_t w = r.in(key, index) ? r.weight(key) : 0;
      if (w && w >= r.least) atomicAdd((unsigned long long*)&sh.mass[index >> shift], w);
    }
  } else {
    auto add = [&](const vec& g, uint32_t i0) { add_to_bins(sh, r, g, i0, lo, shift); };
    each_group(r.x, lo, hi, add);
  }
  __syncthreads();
  draw_from_bins(sh, r, lo, hi, shift, by_chunk, t, whole, draw, token, prob);
}

template <typename T>
hipError_t launch(const T* logits, const float* u, const float* params, const int32_t* top_k, int32_t* token, float* prob,
                  uint32_t rows, uint32_t n, const nfhip::Workspace& ws, hipStream_t s) {
  const uint64_t fits = ws.part ? ws.part_floats * sizeof(float) / sizeof(Part) : 0;
  // Chunks of a row, for two more launches: four workgroups of 512 per CU, at least four
  // chunks a row and 4096 logits a chunk.  Rows of 131072 of every kind: 64 rows 72 us
  // (149 without chunks), 256 rows 142 (180).  Short rows do without, and rows of up to 65536
  // where they are few: a top_k then ends sooner without chunks (one row of 32000: 13 and
  // 17 us), which the other kinds make up for only where a batch waits for its slowest row
  // (by temperature 23 and 18, top_p 29 and 26; 16 rows of every kind 50 and 36).
  uint64_t chunks64 = n > 65536 || (n > 16384 && rows >= 4) ? (1024 + rows - 1) / rows : 0;
  if (chunks64) chunks64 = min(min(max(chunks64, (uint64_t)4), (uint64_t)(n + 4095) / 4096), fits / rows);
  uint32_t chunks = chunks64 > 1 ? (uint32_t)chunks64 : 0;
  const uint32_t step = chunks ? ((n + chunks - 1) / chunks + 7) / 8 * 8 : n;
  if (chunks) chunks = (n + step - 1) / step;
  Part* parts = reinterpret_cast<Part*>(ws.part);
  if (chunks) {
    sample_best_kernel<<<dim3(chunks, rows), kChunkThreads, 0, s>>>(logits, n, step, parts);
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
