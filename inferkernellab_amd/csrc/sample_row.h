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

// NaN as -inf, and one zero.
__device__ inline float clean(float x) { return x != x ? -INFINITY : x + 0.f; }

// A row in 16-byte vectors from the aligned address at or below its start.
// Elements of the first and last vector that are not the row's read as -inf.
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
    if constexpr (EB == 4) return __uint_as_float(w[j]);
    else return (j & 1) ? elem<Tag>::hi(w[j >> 1]) : elem<Tag>::lo(w[j >> 1]);
  }
  static constexpr uint32_t NONE = std::is_same<Tag, f32_tag>::value   ? 0xff800000u
                                   : std::is_same<Tag, f16_tag>::value ? 0xfc00u
                                                                       : 0xff80u;  // -inf
  __device__ inline v4u32 load(int v) const {
    const char *at = base + (int64_t)v * 16;
    if (v * VEC >= shift && (v + 1) * VEC <= vocab + shift) return load16v_global(at);
    v4u32 w = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int i = v * VEC + j - shift;
      uint32_t e = NONE;
      if (i >= 0 && i < vocab) {
        if constexpr (EB == 4) e = reinterpret_cast<const uint32_t *>(at)[j];
        else e = reinterpret_cast<const uint16_t *>(at)[j];
      }
      if constexpr (EB == 4) w[j] = e;
      else w[j >> 1] |= e << (16 * (j & 1));
    }
    return w;
  }
  // A vector that is the row's whole: all but the first and the last are.
  __device__ inline v4u32 load_whole(int v) const { return load16v_global(base + (int64_t)v * 16); }
  // `to`, or the last vector before it if other elements share that one
  __device__ inline int whole_end(int to) const { return to == vectors && (vocab + shift) % VEC ? to - 1 : to; }

  // f(index of the first, values) for the vectors [from, to), by vectors, so that
  // what is done to its elements can overlap; a thread's next one is on its way
  // meanwhile. Vectors that are not the row's whole are loaded by begin() alone:
  // the thread that has a last one behind the first round begins with it. (With
  // loads of either kind in the loop, the wait for them stands before the work: 256
  // x 131072 fp32 64 us, else 59.)
  template <typename F>
  __device__ inline void each(int from, int to, F f) const {
    each(from, to, begin(from, to), f);
  }
  // the same, with the thread's first vector loaded some time before by begin()
  __device__ inline bool begins_at_end(int from, int to) const {
    const int last = to - 1 - from, its = last % SAMPLE_THREADS;  // the first thread may begin with the first vector
    return (int)threadIdx.x == (its ? its : SAMPLE_THREADS - 1) && last >= SAMPLE_THREADS && whole_end(to) != to;
  }
  __device__ inline v4u32 begin(int from, int to) const {
    const int v = begins_at_end(from, to) ? to - 1 : from + (int)threadIdx.x;
    return v < to ? load(v) : v4u32{0, 0, 0, 0};
  }
  template <typename F>
  __device__ inline void each(int from, int to, v4u32 w, F f) const {
    int v = from + threadIdx.x, ahead = v + SAMPLE_THREADS;
    if (v >= to) return;
    if (begins_at_end(from, to)) {
      ahead = v;
      v = to - 1;
    }
    const int end = whole_end(to);
    while (true) {
      v4u32 next = w;
      if (ahead < end) next = load_whole(ahead);
      float x[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[j] = value(w, j);
      f(v * VEC - shift, x);
      if (ahead >= end) return;
      v = ahead;
      ahead += SAMPLE_THREADS;
      w = next;
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
// unrounded in units of 2^-bits. 2^(k/32 + r/32) for whole k and |r| <= 1/2 is
// a power of two, one of 32 roots in shared memory (64 banks: no two entries
// collide; they hold the 2^bits too) and the Taylor series of 2^(r/32) up to r^5,
// whose next term is 2.2e-15 of the value. m is finite; NaN, -inf and whatever
// else weighs under half a unit come to 0. The products and sums are fused where
// it says so and nowhere else: a token weighs the same in every kernel.
struct Weigher {
  double m, rate, floor;  // rate: 32 log2(e) / T; floor: of x - m, a quarter of a unit
  const double *roots;
  int bits;
  __device__ inline Weigher(float top, float temperature, int fraction, const double *table)
      : m(top), roots(table), bits(fraction) {
    const double t = fmin((double)temperature, 1e300);  // its reciprocal by Newton's steps: a division costs thrice
    double r = __builtin_amdgcn_rcp(t);
    r = fma(fma(-t, r, 1.0), r, r);
    r = fma(fma(-t, r, 1.0), r, r);
    rate = 32.0 * 1.4426950408889634 * r;
    floor = -(fraction + 2) * 0.69314718055994531 * t;
  }
  __device__ inline double scaled(float w) const { return ldexp((double)w, bits); }
  // Whether a token may weigh something: false for what is masked, NaN or -inf.
  __device__ inline bool counts(float x) const { return (double)x - m > floor; }
  // Unrounded weights of N tokens; step by step for all of them, as their chains
  // of 15 operations and a load are to overlap.
  template <int N>
  __device__ inline void of(const float (&x)[N], double (&exact)[N]) const {
#pragma clang fp contract(off)
    double r[N], root[N], q[N];
    int k[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const double d = fmax((double)x[j] - m, floor);
      const double z = fma(d, rate, 0x1.8p52);  // its low word: the nearest whole number
      k[j] = (int)(uint32_t)__double_as_longlong(z);
      root[j] = roots[k[j] & 31];
      r[j] = fma(d, rate, -(z - 0x1.8p52));
    }
#pragma unroll
    for (int j = 0; j < N; ++j) q[j] = fma(3.9737099845494154e-11, r[j], 9.172562701824643e-09);
#pragma unroll
    for (int j = 0; j < N; ++j) q[j] = fma(q[j], r[j], 1.6938509724371819e-06);  // (ln(2) / 32)^i / i!
#pragma unroll
    for (int j = 0; j < N; ++j) q[j] = fma(q[j], r[j], 0.00023459619820224677);
#pragma unroll
    for (int j = 0; j < N; ++j) q[j] = fma(q[j], r[j], 0.02166084939249829);
#pragma unroll
    for (int j = 0; j < N; ++j) q[j] = fma(q[j], r[j], 1.0);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const double v = root[j] * q[j];
      exact[j] = __hiloint2double(__double2hiint(v) + ((k[j] & ~31) << 15), __double2loint(v));
    }
  }
  // Rounded to a whole number by the addition: doubles from 2^52 are 1 apart.
  __device__ inline static uint64_t rounded(double exact) {
    return (uint64_t)(__double_as_longlong(exact + 0x1p52) - __double_as_longlong(0x1p52));
  }
  __device__ inline uint64_t operator()(float x) const {
    const float one[1] = {x};
    double exact[1];
    of(one, exact);
    return rounded(exact[0]);
  }
  // ln of the share of token x in `mass`
  __device__ inline float log_share(float x, uint64_t mass) const {
    return (float)(((double)x - m) * rate * (0.69314718055994531 / 32.0) - log(ldexp((double)mass, -bits)));
  }
};

// The weights of a row whose largest logit is +inf: those tokens share all mass.
struct InfiniteWeigher {
  int bits;
  __device__ inline uint64_t operator()(float x) const { return x == INFINITY ? (uint64_t)1 << bits : 0; }
  __device__ inline float log_share(float, uint64_t mass) const { return (float)-log(ldexp((double)mass, -bits)); }
};

__device__ inline void fill_roots(double *table, int bits) {
  if (threadIdx.x < 32) table[threadIdx.x] = ldexp(exp2((double)threadIdx.x / 32.0), bits);
}

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
// The bins whose tokens have to be known one by one: up to three runs (where
// top-k, top-p and the draw may fall), as first bin and length less one.
struct Cuts {
  uint32_t first[3], span[3];
  __device__ inline bool has(int bin) const {
    bool in = false;
#pragma unroll
    for (int i = 0; i < 3; ++i) in |= (uint32_t)bin - first[i] <= span[i];
    return in;
  }
};

struct RowShared {
  uint64_t mass[BINS];
  uint32_t count[BINS];
  double list[LIST];
  uint64_t part[SAMPLE_WAVES];
  uint64_t part2[SAMPLE_WAVES];
  uint64_t found[4];
  double roots[32];
  Cuts cuts;
  uint64_t total, likely, binned;  // mass of the row, of what min-p leaves of it, in the histogram
  uint64_t others;                 // mass of what min-p takes; of all where candidates are alone
  uint32_t weighted, listed;       // tokens in the histogram (where top-k asks), in the list
};

// Where one workgroup has the whole row, its second pass lists up to this many
// candidates, the first LIST of them in sh.list. A row with more of them needs the
// third pass, and the slowest row counts (256 x 131072 fp32, one row of some above
// 2048: 65.5 -> 63.0 us, without such a row 0.2 more). A compute unit has the
// registers for one workgroup, so its 89 KB of LDS keep none out.
constexpr int CANDIDATES = 4 * LIST;
struct WholeRowShared : RowShared {
  double more[CANDIDATES - LIST];
};

// Lane permutations inside rows of 16 lanes without the LDS round trip.
template <int CTRL>
__device__ inline uint64_t dpp64(uint64_t v) {  // lanes without a source get 0
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, 0xf, 0xf, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, 0xf, 0xf, true);
  return ((uint64_t)hi << 32) | lo;
}
__device__ inline uint64_t lane64(uint64_t v, int lane) {
  return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32) |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}
// Sum over the lanes of a row of 16 up to this one.
__device__ inline uint64_t row_scan(uint64_t v) {
  v += dpp64<0x111>(v);  // row_shr 1, 2, 4, 8
  v += dpp64<0x112>(v);
  v += dpp64<0x114>(v);
  v += dpp64<0x118>(v);
  return v;
}
__device__ inline uint64_t wave_scan(uint64_t v) {
  v = row_scan(v);
  const uint64_t a = lane64(v, 15), b = a + lane64(v, 31), c = b + lane64(v, 47);
  const int row = (threadIdx.x & 63) >> 4;
  return v + (row == 0 ? 0 : row == 1 ? a : row == 2 ? b : c);
}
__device__ inline float row_max(float v) {
  v = fmaxf(v, dpp_mov<DPP_QUAD_XOR1>(v));
  v = fmaxf(v, dpp_mov<DPP_QUAD_XOR2>(v));
  v = fmaxf(v, dpp_mov<DPP_ROW_HALF_MIRROR>(v));
  return fmaxf(v, dpp_mov<DPP_ROW_MIRROR>(v));
}
__device__ inline float wave_max(float v) { return max_xor32(max_xor16(row_max(v))); }

// Every thread of the workgroup calls these and receives the result. The waves'
// values are joined in the lanes of each wave, not in a loop: these run once or
// twice a row, and code that runs once is paid for by fetching it.
static_assert(SAMPLE_WAVES == 16, "a row of lanes holds the waves' values");
__device__ inline void block_extremes(float &top, float &least, RowShared &sh) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  top = wave_max(top);
  least = wave_max(-least);
  float *part = reinterpret_cast<float *>(sh.part);
  __syncthreads();
  if (lane == 0) {
    part[wave] = top;
    part[SAMPLE_WAVES + wave] = least;
  }
  __syncthreads();
  const int both = __float_as_int(row_max(part[lane & 31]));
  top = __int_as_float(__builtin_amdgcn_readlane(both, 0));
  least = -__int_as_float(__builtin_amdgcn_readlane(both, 16));
}
// Sum of the values of the threads before this one; `all` the sum of all.
__device__ inline uint64_t block_before(uint64_t v, uint64_t *part, uint64_t &all) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint64_t run = wave_scan(v);
  __syncthreads();
  if (lane == 63) part[wave] = run;
  __syncthreads();
  const uint64_t sums = row_scan(part[lane & 15]);
  all = lane64(sums, 15);
  return (wave ? lane64(sums, wave - 1) : 0) + run - v;
}
__device__ inline uint64_t block_sum(uint64_t v, RowShared &sh) {
  uint64_t all;
  block_before(v, sh.part, all);
  return all;
}

// The largest logit, and the smallest above -inf.
template <int N>
__device__ inline void extremes(const float (&x)[N], float &top, float &least) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    top = fmaxf(top, x[j]);
    least = fminf(least, x[j] > -INFINITY ? x[j] : INFINITY);
  }
}

// Those of the row's vectors [from, to), four of a thread's on their way at a time
// where there are so many: nothing but memory bounds this pass (256 x 131072
// fp32: 72 -> 65 us in all).
template <typename Tag>
__device__ inline void row_extremes(const RowReader<Tag> &row, int from, int to, float &top, float &least) {
  constexpr int AHEAD = 4;
  const auto take = [&](const v4u32 &w) {
    float x[RowReader<Tag>::VEC];
#pragma unroll
    for (int j = 0; j < RowReader<Tag>::VEC; ++j) x[j] = row.value(w, j);
    extremes(x, top, least);
  };
  int v = from + threadIdx.x;
  for (; v + (AHEAD - 1) * SAMPLE_THREADS < to; v += AHEAD * SAMPLE_THREADS) {
    v4u32 w[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) w[u] = row.load(v + u * SAMPLE_THREADS);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) take(w[u]);
  }
  for (; v < to; v += SAMPLE_THREADS) take(row.load(v));
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
template <bool BY_COUNT, typename Tag, typename W>
__device__ inline Selected radix_select(const RowReader<Tag> &row, const W &weigh, uint64_t bound, RowShared &sh) {
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
    row.each(0, row.vectors, [&](int, const float(&raw)[RowReader<Tag>::VEC]) {
      for (int j = 0; j < RowReader<Tag>::VEC; ++j) {
        const float x = clean(raw[j]);
        const uint32_t key = order_key(x);
        if (level > 0 && (key >> (shift + bits)) != s.key) continue;
        const uint64_t w = weigh(x);
        if (w == 0) continue;
        const uint32_t bin = mask - ((key >> shift) & mask);  // the largest first
        // equal logits all over a wave: one addition
        const uint64_t here = __ballot(true);
        if (__ballot(key == (uint32_t)__builtin_amdgcn_readfirstlane((int)key)) == here) {
          if (__popcll(here & ((1ull << (threadIdx.x & 63)) - 1ull)) != 0) continue;
          const uint64_t n = (uint64_t)__popcll(here);
          atomicAdd((unsigned long long *)&sh.mass[bin], (unsigned long long)(n * w));
          atomicAdd(&sh.count[bin], (uint32_t)n);
          continue;
        }
        atomicAdd((unsigned long long *)&sh.mass[bin], (unsigned long long)w);
        atomicAdd(&sh.count[bin], 1u);
      }
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
    v4u32 w = {0, 0, 0, 0};
    if (v < row.vectors) {
      w = row.load(v);
#pragma unroll
      for (int j = 0; j < RowReader<Tag>::VEC; ++j) mine += order_key(clean(row.value(w, j))) == key;
    }
    uint64_t before = passed + block_before(mine, sh.part, all);
    if (mine && nth >= before && nth - before < mine) {
#pragma unroll
      for (int j = 0; j < RowReader<Tag>::VEC; ++j)
        if (order_key(clean(row.value(w, j))) == key && before++ == nth)
          sh.found[3] = (uint64_t)(v * RowReader<Tag>::VEC + j - row.shift);
    }
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

template <typename W>
__device__ inline void store_token(const SampleParams &p, int64_t b, const W &weigh, int token, float x,
                                   uint64_t total, uint64_t kept) {
  p.tokens[b] = token;
  if (p.policy) p.policy[b] = weigh.log_share(x, total);
  if (p.sampling) p.sampling[b] = weigh.log_share(x, kept);
}

// ------------------------------------------------------ selection by a histogram
// One histogram of the weights over their logarithm tells in which bins the
// cuts and the draw fall; only the tokens of those bins are put in order.
__device__ inline void clear_histogram(RowShared &sh) {
  for (int i = threadIdx.x; i < BINS; i += SAMPLE_THREADS) {
    sh.mass[i] = 0;
    sh.count[i] = 0;
  }
}

// A listed token: its key above its index, so that falling order of the word
// is the order of the tokens. Held as the double of these bits (positive,
// finite and normal): doubles are put in order by one instruction each way.
constexpr int INDEX_BITS = 22;
static_assert((1 << INDEX_BITS) >= IKL_SAMPLE_MAX_VOCAB, "an index fits");
__device__ inline double token_word(uint32_t key, int index) {
  return __longlong_as_double((1ll << 62) | ((int64_t)key << INDEX_BITS) | ((1 << INDEX_BITS) - 1 - index));
}
__device__ inline float word_logit(double word) {
  return key_float((uint32_t)((uint64_t)__double_as_longlong(word) >> INDEX_BITS));
}
__device__ inline int word_index(double word) {
  const int mask = (1 << INDEX_BITS) - 1;
  return mask - ((int)__double_as_longlong(word) & mask);
}

// What min-p makes of the tokens it leaves out. They are no candidates, and
// where the first k need not be weighed without them, only their mass counts
// (top-p's share is of it too): they stay out of the histogram.
struct Candidates {
  double least;  // weight of a candidate: more than half a unit, which rounds to 1
  bool alone;    // in the histogram
  __device__ inline Candidates(const RowSettings &set, const Weigher &weigh)
      : least(fmax(weigh.scaled(set.min_p), 0x1.0000000000001p-1)),
        alone(set.min_p > 0.f && !(set.top_k > 0 && set.top_p < 1.f)) {}
};

// Bins are even steps of the logit from the largest down to the smallest, at
// most to where weights round to 0 or candidates end: the bin number falls with
// the logit, in any row, which is all that is asked of it.
struct Binner {
  float top, rate;
  __device__ inline Binner(const RowSettings &set, const Weigher &weigh, const Candidates &cand, float most, float least)
      : top(most) {
    float range = fminf(most - least, (float)-weigh.floor);
    if (cand.alone) range = fminf(range, set.temperature * -0.69314718f * __log2f(set.min_p));
    // a row whose tokens share a bin has no rate
    rate = range > 0.f ? fminf((float)BINS * __builtin_amdgcn_rcpf(range), 0x1.fffffep+127f) : 0.f;
  }
  __device__ inline int operator()(float x) const {  // any value: 0 .. BINS - 1
    return (int)fminf(fmaxf((top - x) * rate, 0.f), (float)(BINS - 1));
  }
};

// Adds a token to the histogram and, where a workgroup has the whole row, a
// candidate to the list as well.
template <bool LISTED, typename Shared>
__device__ inline void add_token(int index, float x, uint64_t w, const RowSettings &set, const Binner &bin_of,
                                 Shared &sh) {
  const int bin = bin_of(x);
  atomicAdd((unsigned long long *)&sh.mass[bin], (unsigned long long)w);
  if (set.top_k > 0) atomicAdd(&sh.count[bin], 1u);
  if constexpr (LISTED) {
    const uint32_t at = atomicAdd(&sh.listed, 1u);
    const double word = token_word(order_key(clean(x)), index);
    if (at < LIST) sh.list[at] = word;
    else if (at < CANDIDATES) sh.more[at - LIST] = word;
  }
}

// Adds tokens to the histogram, and to `others` what min-p asks for: the mass of
// all tokens where candidates are alone in the histogram (there most waves have
// none and are done with a sum), else that of the tokens that are none.
template <int N, typename Shared>
__device__ inline void add_tokens(int index, const float (&x)[N], const RowSettings &set, const Weigher &weigh,
                                  const Candidates &cand, const Binner &bin_of, uint64_t &others, Shared &sh) {
  constexpr bool LISTED = std::is_same<Shared, WholeRowShared>::value;
  double exact[N];
  weigh.of(x, exact);
  uint64_t w[N];
#pragma unroll
  for (int j = 0; j < N; ++j) w[j] = weigh.rounded(exact[j]);
  if (cand.alone) {
    uint32_t hits = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      others += w[j];
      hits |= (uint32_t)(exact[j] >= cand.least) << j;
    }
    if (hits) {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (hits >> j & 1) add_token<LISTED>(index + j, x[j], w[j], set, bin_of, sh);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (w[j]) add_token<false>(index + j, x[j], w[j], set, bin_of, sh);
  if (set.min_p > 0.f) {
#pragma unroll
    for (int j = 0; j < N; ++j) others += exact[j] < cand.least ? w[j] : 0;
  }
}

// The last bin whose `before` is at most `bound`: with less than the row's total
// for a bound, the one that the cumulative count or mass exceeds it in. By the
// lanes of half a wave, in two looks; the halves have a bound each.
template <typename T>
__device__ inline int bin_at(const T *before, uint64_t bound) {
  constexpr int STEP = BINS / 32;
  static_assert(STEP == 64, "two looks");
  const int lane = threadIdx.x & 31;
  const auto lanes = [](bool in) {  // of this half
    const uint64_t all = __ballot(in);
    return __popc((threadIdx.x & 32) ? (uint32_t)(all >> 32) : (uint32_t)all);
  };
  const int part = (lanes((uint64_t)before[lane * STEP] <= bound) - 1) * STEP, at = part + 2 * lane;
  return part + lanes((uint64_t)before[at] <= bound) + lanes((uint64_t)before[at + 1] <= bound) - 1;
}

// Turns the histogram in shared memory into the masses and counts before each
// bin (counts only where top-k needs them), with the row's sums, and finds the
// cuts' bins, into sh.cuts. A cut that depends on an earlier one's exact place
// is bracketed by that one's bin; one behind all candidates has none.
__device__ inline void find_cuts(const RowSettings &set, const Candidates &cand, RowShared &sh) {
  constexpr int PER = BINS / SAMPLE_THREADS;
  const int at = threadIdx.x * PER;
  uint64_t mass[PER], binned, sum = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    mass[i] = sum;
    sum += sh.mass[at + i];
  }
  const uint64_t before = block_before(sum, sh.part, binned);
#pragma unroll
  for (int i = 0; i < PER; ++i) sh.mass[at + i] = before + mass[i];
  uint64_t weighted = 0;
  if (set.top_k > 0) {
    uint64_t rank[PER];
    sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      rank[i] = sum;
      sum += sh.count[at + i];
    }
    const uint64_t ahead = block_before(sum, sh.part2, weighted);
#pragma unroll
    for (int i = 0; i < PER; ++i) sh.count[at + i] = (uint32_t)(ahead + rank[i]);
  }
  const uint64_t total = cand.alone ? sh.others : binned, likely = cand.alone ? binned : total - sh.others;
  __syncthreads();
  if (threadIdx.x < 64) {
    // What is kept lies between two masses: one half of the wave goes by the lower
    // one, the other by the upper. One loop for the cuts: code that runs once is
    // paid for by fetching it.
    uint64_t kept = total;
    const auto run = [&](int i, int bin) {
      const int first = __builtin_amdgcn_readlane(bin, 0);
      const uint64_t past = bin + 1 < BINS ? sh.mass[bin + 1] : binned;
      kept = min(kept, threadIdx.x >= 32 ? past : sh.mass[bin] + 1);
      sh.cuts.first[i] = (uint32_t)first;
      sh.cuts.span[i] = (uint32_t)(__builtin_amdgcn_readlane(bin, 32) - first);
    };
    if (threadIdx.x < 2) {  // no bin
      sh.cuts.first[threadIdx.x] = 2 * BINS;
      sh.cuts.span[threadIdx.x] = 0;
    }
    if (set.top_k > 0 && (uint64_t)set.top_k < weighted) run(0, bin_at(sh.count, (uint64_t)set.top_k - 1));
#pragma unroll 1
    for (int i = set.top_p < 1.f ? 1 : 2; i < 3; ++i) {
      if (i == 2) kept = min(kept, likely);
      const uint64_t bound = scaled_floor(i == 1 ? set.top_p : set.uniform, kept);
      if (lane64(bound, 0) < binned) run(i, bin_at(sh.mass, bound));
    }
    if (threadIdx.x == 0) {
      sh.total = total;
      sh.likely = likely;
      sh.binned = binned;
      sh.weighted = (uint32_t)weighted;
    }
  }
  __syncthreads();
}

// The word of the lane whose number differs in bit D.
template <int D>
__device__ inline double across(double v) {
  const int lo = (int)__double_as_longlong(v), hi = __double2hiint(v);
  if constexpr (D == 1 || D == 2 || D == 8) {  // quad permutations, a row turned by 8
    constexpr int CTRL = D == 1 ? DPP_QUAD_XOR1 : D == 2 ? DPP_QUAD_XOR2 : 0x128;
    return __hiloint2double(__builtin_amdgcn_mov_dpp(hi, CTRL, 0xf, 0xf, false),
                            __builtin_amdgcn_mov_dpp(lo, CTRL, 0xf, 0xf, false));
  } else {
    return __hiloint2double(__shfl_xor(hi, D, 64), __shfl_xor(lo, D, 64));
  }
}

// One step of the sorting network between lanes D apart: the lower lane of a
// pair keeps the larger word where its run falls.
template <int D>
__device__ inline void step_across(double (&w)[2], bool falls) {
  const bool larger = falls == ((threadIdx.x & D) == 0);
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const double other = across<D>(w[e]);
    w[e] = larger ? fmax(w[e], other) : fmin(w[e], other);
  }
}

// Puts the `n` words in sh.list in falling order, n <= 256: four threads count the
// words above each. (By a bitonic network in one wave's registers 92 words took
// 1.1 us more, 256 as long.)
__device__ inline void rank_list(int n, RowShared &sh) {
  constexpr int LANES = 4;
  const int at = threadIdx.x / LANES;
  double word = 0.0;
  int rank = 0;
  if (at < n) {
    word = sh.list[at];
#pragma unroll 4
    for (int j = threadIdx.x % LANES; j < n; j += LANES) rank += sh.list[j] > word;
  }
  rank += __builtin_amdgcn_mov_dpp(rank, DPP_QUAD_XOR1, 0xf, 0xf, false);
  rank += __builtin_amdgcn_mov_dpp(rank, DPP_QUAD_XOR2, 0xf, 0xf, false);
  __syncthreads();
  if (at < n && threadIdx.x % LANES == 0) sh.list[rank] = word;
  __syncthreads();
}

// Puts the `n` words in sh.list in falling order (n <= LIST; the words behind
// them are overwritten up to a power of two). A bitonic network over pairs in
// registers: steps inside a wave need no barrier, and of the 45 steps of 512
// words only 3 cross waves. (With the words in shared memory, 259 words took
// 12 us.)
static_assert(LIST == 2 * SAMPLE_THREADS, "two words a thread");
__device__ inline void sort_list(int n, RowShared &sh) {
  int size = 128;
  while (size < n) size <<= 1;
  const int at = 2 * threadIdx.x;
  const bool on = at < size;  // whole waves
  double w[2] = {0.0, 0.0};
  if (on) {
    w[0] = at < n ? sh.list[at] : 0.0;
    w[1] = at + 1 < n ? sh.list[at + 1] : 0.0;
  }
  for (int run = 2; run <= size; run <<= 1) {
    const bool falls = (at & run) == 0;
    for (int d = run >> 1; d >= 128; d >>= 1) {  // between waves
      __syncthreads();
      if (on) {
        sh.list[at] = w[0];
        sh.list[at + 1] = w[1];
      }
      __syncthreads();
      if (on) {
        const bool larger = falls == ((at & d) == 0);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const double other = sh.list[(at ^ d) + e];
          w[e] = larger ? fmax(w[e], other) : fmin(w[e], other);
        }
      }
    }
    if (on) {
      if (run >= 128) step_across<32>(w, falls);
      if (run >= 64) step_across<16>(w, falls);
      if (run >= 32) step_across<8>(w, falls);
      if (run >= 16) step_across<4>(w, falls);
      if (run >= 8) step_across<2>(w, falls);
      if (run >= 4) step_across<1>(w, falls);
      const double hi = fmax(w[0], w[1]), lo = fmin(w[0], w[1]);
      w[0] = falls ? hi : lo;
      w[1] = falls ? lo : hi;
    }
  }
  __syncthreads();
  if (on) {
    sh.list[at] = w[0];
    sh.list[at + 1] = w[1];
  }
  __syncthreads();
}

// By the first wave: the token of a word and its log probabilities, each by a lane.
__device__ inline void store_drawn(const SampleParams &p, int64_t b, const Weigher &weigh, double word, uint64_t total,
                                   uint64_t kept) {
  const int lane = threadIdx.x;
  const float share = weigh.log_share(word_logit(word), lane == 0 ? total : kept);
  if (lane == 0) {
    p.tokens[b] = word_index(word);
    if (p.policy) p.policy[b] = share;
  }
  if (lane == 1 && p.sampling) p.sampling[b] = share;
}

// The draw from up to 64 E tokens, by the first wave: what sample_from_list does,
// E tokens a lane and without a barrier (3 tokens 4.7 -> 1.3 us). Up to 64 words
// take their place by counting the larger ones, more are in order already.
template <int E>
__device__ inline void sample_from_few(const SampleParams &p, int64_t b, const RowSettings &set, const Weigher &weigh,
                                       const Binner &bin_of, int n, RowShared &sh) {
  const int lane = threadIdx.x, at = lane * E;  // this lane's tokens: at .. at + E - 1 of the order
  double word[E];
#pragma unroll
  for (int e = 0; e < E; ++e) word[e] = at + e < n ? sh.list[at + e] : 0.0;
  if constexpr (E == 1) {
    int rank = 0;
    for (int j = 0; j < n; ++j)
      rank += __longlong_as_double((int64_t)lane64((uint64_t)__double_as_longlong(word[0]), j)) > word[0];
    const int to = 4 * (lane < n ? rank : lane);
    word[0] = __hiloint2double(__builtin_amdgcn_ds_permute(to, __double2hiint(word[0])),
                               __builtin_amdgcn_ds_permute(to, __double2loint(word[0])));
  }
  uint64_t w[E], before[E], sum = 0;
  int bin[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float x = word_logit(word[e]);
    w[e] = at + e < n ? weigh(x) : 0;
    bin[e] = at + e < n ? bin_of(x) : BINS;  // a bin of their own behind the others
    before[e] = sum;
    sum += w[e];
  }
  const uint64_t ahead = wave_scan(sum) - sum;
  // Where a bin's tokens begin here: what stands before that place is taken off
  // what stands before the bin in the row.
  const int left = __shfl_up(bin[E - 1], 1, 64);  // with every lane active
  bool starts[E];
  uint64_t begins = 0, offset[E];  // of the last bin that begins in this lane, then of each token's
  int first = 0, head[E];
  bool any = false;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    before[e] += ahead;
    starts[e] = e == 0 ? lane == 0 || left != bin[0] : bin[e - 1] != bin[e];
    begins = starts[e] ? before[e] : begins;
    first = starts[e] ? at + e : first;
    any = any || starts[e];
  }
  const uint64_t lower = __ballot(any) & ((1ull << lane) - 1ull);  // lane 0 begins one
  const int from = lower ? 63 - __clzll(lower) : 0;
  uint64_t run = ((uint64_t)(uint32_t)__shfl((int)(begins >> 32), from, 64) << 32) |
                 (uint32_t)__shfl((int)(uint32_t)begins, from, 64);
  int run_head = __shfl(first, from, 64);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    run = starts[e] ? before[e] : run;
    run_head = starts[e] ? at + e : run_head;
    offset[e] = run;
    head[e] = run_head;
  }
  uint64_t kept = sh.total;
  const bool by_rank = set.top_k > 0 && (uint32_t)set.top_k < sh.weighted;
#pragma unroll
  for (int e = 0; e < E; ++e) before[e] += sh.mass[min(bin[e], BINS - 1)] - offset[e];  // of the whole row
  if (by_rank) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint64_t kth = __ballot(at + e < n && sh.count[min(bin[e], BINS - 1)] + (uint32_t)(at + e - head[e]) ==
                                                      (uint32_t)set.top_k - 1);
      if (kth) kept = lane64(before[e] + w[e], __ffsll((unsigned long long)kth) - 1);
    }
  }
  // The masses before the tokens rise, so the tokens up to a bound are the first
  // ones; the last of them is the one the bound falls in.
  const auto last_up_to = [&](uint64_t bound, uint64_t &end, double &which) {
    int count = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) count += __popcll(__ballot(at + e < n && before[e] <= bound));
    const int place = count - 1;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (place % E == e) {
        end = lane64(before[e] + w[e], place / E);
        which = __longlong_as_double((int64_t)lane64((uint64_t)__double_as_longlong(word[e]), place / E));
      }
  };
  uint64_t end = 0;
  double drawn = 0.0;
  const uint64_t most = scaled_floor(set.top_p, kept);
  if (set.top_p < 1.f && most < sh.binned) {
    last_up_to(most, end, drawn);
    kept = min(kept, end);
  }
  kept = min(kept, sh.likely);
  last_up_to(scaled_floor(set.uniform, kept), end, drawn);
  store_drawn(p, b, weigh, drawn, sh.total, kept);
}

// The draw from the `n` tokens in sh.list, all those of the cuts' bins, with
// sh.mass and sh.count as find_cuts left them.
__device__ inline void sample_from_list(const SampleParams &p, int64_t b, const RowSettings &set, const Weigher &weigh,
                                        const Binner &bin_of, int n, RowShared &sh) {
  constexpr int PER = LIST / SAMPLE_THREADS;
  sort_list(n, sh);
  const int first = threadIdx.x * PER;
  uint64_t before[PER], w[PER], sum = 0, all;
  int bin[PER];
  for (int i = 0; i < PER; ++i) {
    const bool on = first + i < n;
    const float x = on ? word_logit(sh.list[first + i]) : 0.f;
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
    if (bin[i] < 0 || (at > 0 && bin_of(word_logit(sh.list[at - 1])) == bin[i])) continue;
    sh.mass[bin[i]] -= before[i];
    sh.count[bin[i]] -= (uint32_t)at;
  }
  if (threadIdx.x == 0) sh.found[0] = sh.found[1] = 0;
  __syncthreads();
  const bool by_rank = set.top_k > 0 && (uint32_t)set.top_k < sh.weighted;
  for (int i = 0; i < PER; ++i) {
    if (bin[i] < 0) continue;
    before[i] += sh.mass[bin[i]];
    if (by_rank && sh.count[bin[i]] + (uint32_t)(first + i) == (uint32_t)set.top_k - 1) sh.found[0] = before[i] + w[i];
  }
  __syncthreads();
  uint64_t kept = by_rank ? sh.found[0] : sh.total;
  const uint64_t most = scaled_floor(set.top_p, kept);
  if (set.top_p < 1.f && most < sh.binned) {
    for (int i = 0; i < PER; ++i)
      if (bin[i] >= 0 && before[i] <= most && most - before[i] < w[i]) sh.found[1] = before[i] + w[i];  // one token
    __syncthreads();
    kept = min(kept, sh.found[1]);
  }
  kept = min(kept, sh.likely);
  const uint64_t aim = scaled_floor(set.uniform, kept);
  for (int i = 0; i < PER; ++i)
    if (bin[i] >= 0 && before[i] <= aim && aim - before[i] < w[i]) sh.found[2] = (uint64_t)(first + i);  // one token
  __syncthreads();
  if (threadIdx.x < 64) store_drawn(p, b, weigh, sh.list[sh.found[2]], sh.total, kept);
}

// The whole draw by radix selections, for rows whose cuts fall in bins of more
// than LIST tokens; sh.total, sh.likely and sh.weighted hold the row's.
template <typename Tag, typename W>
__device__ inline void sample_by_radix(const SampleParams &p, int64_t b, const RowReader<Tag> &row,
                                       const RowSettings &set, const W &weigh, RowShared &sh) {
  const uint64_t total = sh.total;
  uint64_t kept = total;
  if (set.top_k > 0 && (uint32_t)set.top_k < sh.weighted) {
    const Selected s = radix_select<true>(row, weigh, (uint64_t)set.top_k - 1, sh);
    kept = s.mass + ((uint64_t)set.top_k - s.count) * weigh(key_float(s.key));
  }
  if (set.top_p < 1.f) {  // the tokens with at most `most` before them
    const uint64_t most = scaled_floor(set.top_p, kept);
    const Selected s = radix_select<false>(row, weigh, most, sh);
    const uint64_t w = weigh(key_float(s.key));
    kept = min(kept, s.mass + ((most - s.mass) / w + 1) * w);
  }
  kept = min(kept, sh.likely);
  const uint64_t aim = scaled_floor(set.uniform, kept);
  const Selected s = radix_select<false>(row, weigh, aim, sh);
  const float x = key_float(s.key);
  const int token = nth_of_key(row, s.key, (aim - s.mass) / weigh(x), sh);
  if (threadIdx.x == 0) store_token(p, b, weigh, token, x, total, kept);
}

// A row whose largest logit is +inf: one group of equal tokens.
template <typename Tag>
__device__ inline void sample_infinite(const SampleParams &p, int64_t b, const RowReader<Tag> &row,
                                       const RowSettings &set, RowShared &sh) {
  const InfiniteWeigher weigh = {p.fraction_bits};
  uint64_t count = 0;
  row.each(0, row.vectors, [&](int, const float(&x)[RowReader<Tag>::VEC]) {
#pragma unroll
    for (int j = 0; j < RowReader<Tag>::VEC; ++j) count += x[j] == INFINITY;
  });
  count = block_sum(count, sh);
  if (threadIdx.x == 0) {
    sh.total = sh.likely = count << p.fraction_bits;
    sh.weighted = (uint32_t)count;
  }
  __syncthreads();
  sample_by_radix<Tag>(p, b, row, set, weigh, sh);
}

}  // namespace ikl
