// Parts of the sampling kernels: reading a row of logits, its order, integer
// weights, workgroup sums and scans, the selection by a histogram of the
// weights, and the one by radix passes that every row can take.
#pragma once

#include <type_traits>

#include "ikl_common.h"

namespace ikl {

constexpr int SAMPLE_THREADS = 1024;
constexpr int SAMPLE_WAVES = SAMPLE_THREADS / 64;
constexpr int BINS = 2048;  // of a histogram
constexpr int LIST = 2048;  // tokens of the bins where the cuts fall

struct SampleParams {
  const char *logits;
  int64_t stride;  // bytes
  const float *uniform;
  const float *temperature_rows;  // per row where not null, else the value below
  const void *top_k_rows;
  const float *top_p_rows;
  const float *min_p_rows;
  float temperature, top_p, min_p;
  int64_t top_k;
  int64_t *tokens;
  float *policy;    // may be null
  float *sampling;  // may be null
  int32_t vocab;
  int32_t fraction_bits;
  int32_t top_k_wide;
};

// A row's settings, with every value outside its range read as the nearest one
// that has a meaning: a temperature not above 0 (greedy) weighs at 1 and draws
// at 0, a top-k outside 1 .. vocab - 1 is off.
struct RowSettings {
  float temperature, top_p, min_p, uniform;
  int32_t top_k;  // 0: off
};

__device__ inline RowSettings row_settings(const SampleParams &p, int64_t b) {
  RowSettings s;
  const float t = p.temperature_rows ? p.temperature_rows[b] : p.temperature;
  const bool greedy = !(t > 0.f);
  s.temperature = greedy ? 1.f : t;
  const int64_t k = !p.top_k_rows  ? p.top_k
                    : p.top_k_wide ? reinterpret_cast<const int64_t *>(p.top_k_rows)[b]
                                   : reinterpret_cast<const int32_t *>(p.top_k_rows)[b];
  s.top_k = k > 0 && k < p.vocab ? (int32_t)k : 0;
  const float tp = p.top_p_rows ? p.top_p_rows[b] : p.top_p;
  s.top_p = tp >= 1.f ? 1.f : tp > 0.f ? tp : 0.f;
  const float mp = p.min_p_rows ? p.min_p_rows[b] : p.min_p;
  s.min_p = mp >= 1.f ? 1.f : mp > 0.f ? mp : 0.f;
  const float u = p.uniform[b];
  s.uniform = greedy || !(u > 0.f) ? 0.f : u < 1.f ? u : 0x1.fffffep-1f;
  return s;
}

// ------------------------------------------------------------------- order
// Unsigned keys in the order of the floats; both zeros are equal, NaN is -inf.
constexpr uint32_t KEY_NEG_INF = 0x007fffffu;

__device__ inline uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x);
  return (u >> 31) ? ~u : u | 0x80000000u;
}
__device__ inline float key_float(uint32_t k) {
  return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k);
}

// A row in 16-byte vectors from the aligned address at or below its start;
// vectors that the row fills only in part are read by elements.
template <typename Tag>
struct RowReader {
  static constexpr int EB = std::is_same<Tag, f32_tag>::value ? 4 : 2;
  static constexpr int VEC = 16 / EB;
  const char *base;  // aligned
  int vocab, shift, vectors;

  __device__ inline RowReader(const char *row, int n) : vocab(n) {
    const uintptr_t at = (uintptr_t)row;
    base = reinterpret_cast<const char *>(at & ~(uintptr_t)15);
    shift = (int)(at & 15) / EB;
    vectors = (n + shift + VEC - 1) / VEC;
  }
  __device__ inline static float value(const v4u32 &w, int j) {
    float x;
    if constexpr (EB == 4) x = __uint_as_float(w[j]);
    else x = (j & 1) ? elem<Tag>::hi(w[j >> 1]) : elem<Tag>::lo(w[j >> 1]);
    return clean(x);
  }
  __device__ inline static float clean(float x) { return x != x ? -INFINITY : x + 0.f; }
  __device__ inline float one(int i) const {  // element i of the row
    const char *at = base + (int64_t)(i + shift) * EB;
    if constexpr (EB == 4) return clean(*reinterpret_cast<const float *>(at));
    else return clean(elem<Tag>::lo(*reinterpret_cast<const uint16_t *>(at)));
  }
  __device__ inline bool whole(int v) const { return v * VEC >= shift && (v + 1) * VEC <= vocab + shift; }
  __device__ inline v4u32 load(int v) const { return load16v_global(base + (int64_t)v * 16); }
  // f(index, value) for each element of vector v, in order
  template <typename F>
  __device__ inline void each(int v, F f) const {
    const int first = v * VEC - shift;
    if (whole(v)) {
      const v4u32 w = load(v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) f(first + j, value(w, j));
    } else {
      for (int j = 0; j < VEC; ++j)
        if (first + j >= 0 && first + j < vocab) f(first + j, one(first + j));
    }
  }
};

// ------------------------------------------------------------------ weights
// Bits of a weight's fraction: the sum of `vocab` weights stays below 2^63,
// and a weight within the 52 bits that a double rounds to whole numbers.
__host__ __device__ inline int fraction_bits(int64_t vocab) {
  int up = 0;
  while (((int64_t)1 << up) < vocab) ++up;
  return 63 - up < 52 ? 63 - up : 52;
}

// w(x) = 2^((x - m) log2(e) / T) as the nearest integer to w 2^bits, and
// unrounded in units of 2^-bits. 2^f is its Taylor series about 0 up to f^12;
// on |f| <= 1/2 the next term is 2.4e-16 of the value.
struct Weigher {
  float top;
  double m, rate;
  int bits;
  __device__ inline Weigher(uint32_t top_key, float temperature, int fraction)
      : top(key_float(top_key)), m(top), rate(1.4426950408889634 / (double)temperature), bits(fraction) {}
  __device__ inline double scaled(float w) const { return ldexp((double)w, bits); }
  // log2 of the weight; NaN or -inf where x does not count
  __device__ inline double log2w(float x) const { return x == top ? 0.0 : ((double)x - m) * rate; }
  __device__ inline uint64_t of(double y, double &exact) const {
    exact = 0.0;
    if (!(y > -(double)(bits + 2))) return 0;
    const double n = rint(y), f = y - n;
    double p = 2.5678435993488196e-11;  // ln(2)^k / k!
    p = fma(p, f, 4.44553827187081e-10);
    p = fma(p, f, 7.054911620801121e-09);
    p = fma(p, f, 1.0178086009239696e-07);
    p = fma(p, f, 1.3215486790144305e-06);
    p = fma(p, f, 1.5252733804059838e-05);
    p = fma(p, f, 0.00015403530393381606);
    p = fma(p, f, 0.0013333558146428441);
    p = fma(p, f, 0.009618129107628477);
    p = fma(p, f, 0.055504108664821576);
    p = fma(p, f, 0.2402265069591007);
    p = fma(p, f, 0.6931471805599453);
    p = fma(p, f, 1.0);
    exact = ldexp(p, (int)n + bits);
    // rounded to a whole number by the addition: doubles from 2^52 are 1 apart
    return (uint64_t)(__double_as_longlong(exact + 0x1p52) - __double_as_longlong(0x1p52));
  }
  __device__ inline uint64_t operator()(float x, double &exact) const { return of(log2w(x), exact); }
  __device__ inline uint64_t operator()(float x) const {
    double exact;
    return of(log2w(x), exact);
  }
  // ln of the share of token x in `mass`
  __device__ inline float log_share(float x, uint64_t mass) const {
    return (float)(log2w(x) * 0.69314718055994531 - log(ldexp((double)mass, -bits)));
  }
};

// floor(r m) for r in [0, 1): r is a whole number of at most 24 bits over a power of two.
__device__ inline uint64_t scaled_floor(float r, uint64_t m) {
  const uint32_t u = __float_as_uint(r);
  const int e = (int)(u >> 23);
  const uint64_t mant = e ? (u & 0x7fffffu) | 0x800000u : u & 0x7fffffu;
  const int down = 150 - (e ? e : 1);  // r = mant 2^-down, down >= 24
  const uint64_t lo = mant * m, hi = __umul64hi(mant, m);
  if (down >= 128) return 0;
  if (down >= 64) return hi >> (down - 64);
  return (lo >> down) | (hi << (64 - down));
}

// ------------------------------------------------------- workgroup reductions
struct RowShared {
  uint64_t mass[BINS];
  uint32_t count[BINS];
  uint64_t list[LIST];
  uint64_t part[SAMPLE_WAVES];
  uint64_t part2[SAMPLE_WAVES];
  uint64_t found[4];
  uint32_t listed;
};

__device__ inline uint64_t shfl_xor64(uint64_t v, int mask) {
  return ((uint64_t)(uint32_t)__shfl_xor((int)(v >> 32), mask, 64) << 32) | (uint32_t)__shfl_xor((int)v, mask, 64);
}
__device__ inline uint64_t shfl_up64(uint64_t v, int by) {
  return ((uint64_t)(uint32_t)__shfl_up((int)(v >> 32), by, 64) << 32) | (uint32_t)__shfl_up((int)v, by, 64);
}

// Every thread of the workgroup calls these and receives the result.
__device__ inline void block_extremes(uint32_t &top, uint32_t &least, RowShared &sh) {
  for (int d = 32; d; d >>= 1) {
    top = max(top, (uint32_t)__shfl_xor((int)top, d, 64));
    least = min(least, (uint32_t)__shfl_xor((int)least, d, 64));
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    sh.part[threadIdx.x >> 6] = top;
    sh.part2[threadIdx.x >> 6] = least;
  }
  __syncthreads();
  for (int i = 0; i < SAMPLE_WAVES; ++i) {
    top = max(top, (uint32_t)sh.part[i]);
    least = min(least, (uint32_t)sh.part2[i]);
  }
}
__device__ inline uint64_t block_sum(uint64_t v, RowShared &sh) {
  for (int d = 32; d; d >>= 1) v += shfl_xor64(v, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
  for (int i = 0; i < SAMPLE_WAVES; ++i) v += sh.part[i];
  return v;
}
// Sum of the values of the threads before this one; `all` the sum of all.
__device__ inline uint64_t block_before(uint64_t v, uint64_t *part, uint64_t &all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t run = v;
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t up = shfl_up64(run, d);
    if (lane >= d) run += up;
  }
  __syncthreads();
  if (lane == 63) part[wave] = run;
  __syncthreads();
  uint64_t before = 0;
  all = 0;
  for (int i = 0; i < SAMPLE_WAVES; ++i) {
    if (i < wave) before += part[i];
    all += part[i];
  }
  return before + run - v;
}

// The largest key, and the smallest of those that may have a weight.
__device__ inline void extremes(float x, uint32_t &top, uint32_t &least) {
  const uint32_t key = order_key(x);
  top = max(top, key);
  least = min(least, key > KEY_NEG_INF ? key : 0xffffffffu);
}

// ----------------------------------------------------------- radix selection
struct Selected {
  uint32_t key;     // of the group of equal logits
  uint64_t mass;    // of the tokens before the group
  uint64_t count;   // their number
};

// The first group of equal logits, in falling order, through which the
// cumulative count (BY_COUNT) or mass exceeds `bound`, which the row's total
// does. Three passes over the row, each a histogram of the next bits of the
// keys that are left. Tokens without weight do not count.
template <bool BY_COUNT, typename Tag>
__device__ inline Selected radix_select(const RowReader<Tag> &row, const Weigher &weigh, uint64_t bound, RowShared &sh) {
  Selected s = {0, 0, 0};
  for (int level = 0; level < 3; ++level) {
    const int shift = level == 0 ? 21 : level == 1 ? 10 : 0;
    const int bits = level == 2 ? 10 : 11;
    const uint32_t mask = (1u << bits) - 1u;
    __syncthreads();
    for (int i = threadIdx.x; i < BINS; i += SAMPLE_THREADS) {
      sh.mass[i] = 0;
      sh.count[i] = 0;
    }
    __syncthreads();
    for (int v = threadIdx.x; v < row.vectors; v += SAMPLE_THREADS)
      row.each(v, [&](int, float x) {
        const uint32_t key = order_key(x);
        if (level > 0 && (key >> (shift + bits)) != s.key) return;
        const uint64_t w = weigh(x);
        if (w == 0) return;
        const uint32_t bin = mask - ((key >> shift) & mask);  // the largest first
        // equal logits all over a wave: one addition
        const uint64_t here = __ballot(true);
        if (__ballot(key == (uint32_t)__builtin_amdgcn_readfirstlane((int)key)) == here) {
          if (__popcll(here & ((1ull << (threadIdx.x & 63)) - 1ull)) != 0) return;
          const uint64_t n = (uint64_t)__popcll(here);
          atomicAdd((unsigned long long *)&sh.mass[bin], (unsigned long long)(n * w));
          atomicAdd(&sh.count[bin], (uint32_t)n);
          return;
        }
        atomicAdd((unsigned long long *)&sh.mass[bin], (unsigned long long)w);
        atomicAdd(&sh.count[bin], 1u);
      });
    __syncthreads();
    constexpr int PER = BINS / SAMPLE_THREADS;
    const int first = threadIdx.x * PER;
    uint64_t mass = 0, count = 0, all;
    for (int i = 0; i < PER; ++i) {
      mass += sh.mass[first + i];
      count += sh.count[first + i];
    }
    uint64_t mass_before = s.mass + block_before(mass, sh.part, all);
    uint64_t count_before = s.count + block_before(count, sh.part2, all);
    for (int i = 0; i < PER; ++i) {
      const uint64_t before = BY_COUNT ? count_before : mass_before;
      const uint64_t here = BY_COUNT ? sh.count[first + i] : sh.mass[first + i];
      if (before <= bound && bound - before < here) {  // one bin of one thread
        sh.found[0] = (uint64_t)(mask - (uint32_t)(first + i));
        sh.found[1] = mass_before;
        sh.found[2] = count_before;
      }
      mass_before += sh.mass[first + i];
      count_before += sh.count[first + i];
    }
    __syncthreads();
    s.key = (s.key << bits) | (uint32_t)sh.found[0];
    s.mass = sh.found[1];
    s.count = sh.found[2];
  }
  return s;
}

// Index of the `nth` token (from 0) whose key is `key`, in index order.
template <typename Tag>
__device__ inline int nth_of_key(const RowReader<Tag> &row, uint32_t key, uint64_t nth, RowShared &sh) {
  uint64_t passed = 0;
  __syncthreads();
  if (threadIdx.x == 0) sh.found[3] = 0;
  for (int v0 = 0; v0 < row.vectors; v0 += SAMPLE_THREADS) {
    const int v = v0 + threadIdx.x;
    uint64_t mine = 0, all;
    if (v < row.vectors) row.each(v, [&](int, float x) { mine += order_key(x) == key; });
    uint64_t before = passed + block_before(mine, sh.part, all);
    if (mine && nth >= before && nth - before < mine)
      row.each(v, [&](int i, float x) {
        if (order_key(x) == key && before++ == nth) sh.found[3] = (uint64_t)i;
      });
    passed += all;
    if (passed > nth) break;
  }
  __syncthreads();
  return (int)sh.found[3];
}

__device__ inline void store_nothing(const SampleParams &p, int64_t b) {
  p.tokens[b] = -1;
  if (p.policy) p.policy[b] = -INFINITY;
  if (p.sampling) p.sampling[b] = -INFINITY;
}

__device__ inline void store_token(const SampleParams &p, int64_t b, const Weigher &weigh, int token, float x,
                                   uint64_t total, uint64_t kept) {
  p.tokens[b] = token;
  if (p.policy) p.policy[b] = weigh.log_share(x, total);
  if (p.sampling) p.sampling[b] = weigh.log_share(x, kept);
}

// ------------------------------------------------------ selection by a histogram
// One histogram of the weights over their logarithm tells in which bins the
// cuts and the draw fall; only the tokens of those bins are put in order.
//
// Bins are even steps of log2(w) from 0 to the row's smallest weight, at most
// to where weights round to 0: the bin number falls with the logit, in any row.
struct Binner {
  double m, rate;
  float top;
  __device__ inline Binner(const Weigher &weigh, uint32_t least_key) : m(weigh.m), rate(0.0), top(weigh.top) {
    const double range = fmin(((double)key_float(least_key) - weigh.m) * -weigh.rate, (double)(weigh.bits + 2));
    if (range > 0.0) rate = weigh.rate * (-(double)BINS / range);
  }
  __device__ inline int operator()(float x) const {
    const int b = x == top ? 0 : (int)fmin(((double)x - m) * rate, (double)(BINS - 1));
    return b < 0 ? 0 : b;
  }
};

// A thread's share of the row's mass, of what min-p leaves of it, and of the
// tokens with a weight (the last two where the settings need them).
struct Totals {
  uint64_t total = 0, likely = 0, count = 0;
};

__device__ inline void clear_histogram(RowShared &sh) {
  for (int i = threadIdx.x; i < BINS; i += SAMPLE_THREADS) {
    sh.mass[i] = 0;
    sh.count[i] = 0;
  }
}

__device__ inline void add_token(float x, const RowSettings &set, const Weigher &weigh, const Binner &bin_of,
                                 Totals &sums, RowShared &sh) {
  double exact;
  const uint64_t w = weigh(x, exact);
  if (w == 0) return;
  sums.total += w;
  sums.likely += exact >= weigh.scaled(set.min_p) ? w : 0;
  ++sums.count;
  const int bin = bin_of(x);
  atomicAdd((unsigned long long *)&sh.mass[bin], (unsigned long long)w);
  if (set.top_k > 0) atomicAdd(&sh.count[bin], 1u);
}

// The bins whose tokens have to be known one by one: first and last of up to
// three runs (where top-k, top-p and the draw may fall).
struct Cuts {
  int first[3], last[3];
  __device__ inline bool has(int bin) const {
    bool in = false;
#pragma unroll
    for (int i = 0; i < 3; ++i) in |= bin >= first[i] && bin <= last[i];
    return in;
  }
};

// Turns the histogram in shared memory into the masses and counts before each
// bin (counts only where top-k needs them) and finds the cuts' bins. A cut
// that depends on an earlier one's exact place is bracketed by that one's bin.
__device__ inline Cuts find_cuts(const RowSettings &set, uint64_t total, uint64_t likely, uint64_t count,
                                 RowShared &sh) {
  constexpr int PER = BINS / SAMPLE_THREADS;
  const bool by_rank = set.top_k > 0 && (uint64_t)set.top_k < count;
  const int first = threadIdx.x * PER;
  uint64_t mass[PER + 1], rank[PER + 1], all, sum = 0, num = 0;
  for (int i = 0; i < PER; ++i) {
    mass[i + 1] = sh.mass[first + i];
    rank[i + 1] = sh.count[first + i];
    sum += mass[i + 1];
    num += rank[i + 1];
  }
  mass[0] = block_before(sum, sh.part, all);
  rank[0] = by_rank ? block_before(num, sh.part2, all) : 0;
  for (int i = 0; i < PER; ++i) {
    sh.mass[first + i] = mass[i];
    sh.count[first + i] = (uint32_t)rank[i];
    mass[i + 1] += mass[i];
    rank[i + 1] += rank[i];
  }
  Cuts c;
  uint64_t low = total, high = total;  // the kept mass lies between
  for (int i = 0; i < 3; ++i) {
    c.first[i] = 1;
    c.last[i] = 0;
  }
  // the bin through which the cumulative mass exceeds `bound`, for two bounds
  const auto bins_of = [&](uint64_t a, uint64_t b, int which) {
    __syncthreads();
    for (int i = 0; i < PER; ++i) {
      if (mass[i] <= a && a < mass[i + 1]) {
        sh.found[0] = (uint64_t)(first + i);
        sh.found[1] = mass[i];
      }
      if (mass[i] <= b && b < mass[i + 1]) {
        sh.found[2] = (uint64_t)(first + i);
        sh.found[3] = mass[i + 1];
      }
    }
    __syncthreads();
    c.first[which] = (int)sh.found[0];
    c.last[which] = (int)sh.found[2];
  };
  if (by_rank) {
    __syncthreads();
    for (int i = 0; i < PER; ++i)
      if (rank[i] < (uint64_t)set.top_k && (uint64_t)set.top_k <= rank[i + 1]) {
        sh.found[0] = (uint64_t)(first + i);
        sh.found[1] = mass[i];
        sh.found[3] = mass[i + 1];
      }
    __syncthreads();
    c.first[0] = c.last[0] = (int)sh.found[0];
    low = sh.found[1] + 1;
    high = sh.found[3];
  }
  if (set.top_p < 1.f) {
    bins_of(scaled_floor(set.top_p, low), scaled_floor(set.top_p, high), 1);
    low = min(low, sh.found[1] + 1);
    high = min(high, sh.found[3]);
  }
  if (set.min_p > 0.f) {
    low = min(low, likely);
    high = min(high, likely);
  }
  bins_of(scaled_floor(set.uniform, low), scaled_floor(set.uniform, high), 2);
  return c;
}

// A listed token: its key above its index, so that falling order of the word
// is the order of the tokens.
__device__ inline uint64_t token_word(uint32_t key, int index) { return ((uint64_t)key << 32) | (uint32_t)~index; }

// Puts the `n` words in sh.list in falling order, in place (n <= LIST; words behind them are overwritten).
__device__ inline void sort_list(int n, RowShared &sh) {
  int size = 64;
  while (size < n) size <<= 1;
  for (int i = n + threadIdx.x; i < size; i += SAMPLE_THREADS) sh.list[i] = 0;
  for (int run = 2; run <= size; run <<= 1)
    for (int d = run >> 1; d; d >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < size / 2; i += SAMPLE_THREADS) {
        const int a = ((i & ~(d - 1)) << 1) | (i & (d - 1)), b = a | d;
        const uint64_t x = sh.list[a], y = sh.list[b];
        if ((x < y) == ((a & run) == 0)) {
          sh.list[a] = y;
          sh.list[b] = x;
        }
      }
    }
  __syncthreads();
}

// The draw from the `n` tokens in sh.list, all those of the cuts' bins, with
// sh.mass and sh.count as find_cuts left them.
__device__ inline void sample_from_list(const SampleParams &p, int64_t b, const RowSettings &set, const Weigher &weigh,
                                        const Binner &bin_of, uint64_t total, uint64_t likely, uint64_t count, int n,
                                        RowShared &sh) {
  constexpr int PER = LIST / SAMPLE_THREADS;
  sort_list(n, sh);
  const int first = threadIdx.x * PER;
  uint64_t before[PER], w[PER], sum = 0, all;
  int bin[PER];
  for (int i = 0; i < PER; ++i) {
    const bool on = first + i < n;
    const float x = on ? key_float((uint32_t)(sh.list[first + i] >> 32)) : 0.f;
    w[i] = on ? weigh(x) : 0;
    bin[i] = on ? bin_of(x) : -1;
    before[i] = sum;
    sum += w[i];
  }
  const uint64_t ahead = block_before(sum, sh.part, all);
  // where a bin's tokens begin in the list: what stands before the bin less
  // what stands before them here (modulo 2^64)
  for (int i = 0; i < PER; ++i) {
    before[i] += ahead;
    const int at = first + i;
    if (bin[i] < 0 || (at > 0 && bin_of(key_float((uint32_t)(sh.list[at - 1] >> 32))) == bin[i])) continue;
    sh.mass[bin[i]] -= before[i];
    sh.count[bin[i]] -= (uint32_t)at;
  }
  if (threadIdx.x == 0) sh.found[0] = sh.found[1] = 0;
  __syncthreads();
  const bool by_rank = set.top_k > 0 && (uint64_t)set.top_k < count;
  for (int i = 0; i < PER; ++i) {
    if (bin[i] < 0) continue;
    before[i] += sh.mass[bin[i]];
    if (by_rank && sh.count[bin[i]] + (uint32_t)(first + i) == (uint32_t)set.top_k - 1) sh.found[0] = before[i] + w[i];
  }
  __syncthreads();
  uint64_t kept = by_rank ? sh.found[0] : total;
  if (set.top_p < 1.f) {
    const uint64_t most = scaled_floor(set.top_p, kept);
    for (int i = 0; i < PER; ++i)
      if (bin[i] >= 0 && before[i] <= most)
        atomicMax((unsigned long long *)&sh.found[1], (unsigned long long)(before[i] + w[i]));
    __syncthreads();
    kept = min(kept, sh.found[1]);
  }
  if (set.min_p > 0.f) kept = min(kept, likely);
  const uint64_t aim = scaled_floor(set.uniform, kept);
  for (int i = 0; i < PER; ++i)
    if (bin[i] >= 0 && before[i] <= aim && aim - before[i] < w[i]) {  // one token
      const uint64_t word = sh.list[first + i];
      store_token(p, b, weigh, (int)~(uint32_t)word, key_float((uint32_t)(word >> 32)), total, kept);
    }
}

// The whole draw by radix selections, for rows whose cuts fall in bins of more
// than LIST tokens: `total` the row's mass, `likely` what
// min-p leaves of it, `count` the tokens with weight.
template <typename Tag>
__device__ inline void sample_by_radix(const SampleParams &p, int64_t b, const RowReader<Tag> &row,
                                       const RowSettings &set, const Weigher &weigh, uint64_t total, uint64_t likely,
                                       uint64_t count, RowShared &sh) {
  uint64_t kept = total;
  if (set.top_k > 0 && (uint64_t)set.top_k < count) {
    const Selected s = radix_select<true>(row, weigh, (uint64_t)set.top_k - 1, sh);
    kept = s.mass + ((uint64_t)set.top_k - s.count) * weigh(key_float(s.key));
  }
  if (set.top_p < 1.f) {  // the tokens with at most `most` before them
    const uint64_t most = scaled_floor(set.top_p, kept);
    const Selected s = radix_select<false>(row, weigh, most, sh);
    const uint64_t w = weigh(key_float(s.key));
    kept = min(kept, s.mass + ((most - s.mass) / w + 1) * w);
  }
  if (set.min_p > 0.f) kept = min(kept, likely);
  const uint64_t aim = scaled_floor(set.uniform, kept);
  const Selected s = radix_select<false>(row, weigh, aim, sh);
  const float x = key_float(s.key);
  const int token = nth_of_key(row, s.key, (aim - s.mass) / weigh(x), sh);
  if (threadIdx.x == 0) store_token(p, b, weigh, token, x, total, kept);
}

}  // namespace ikl
