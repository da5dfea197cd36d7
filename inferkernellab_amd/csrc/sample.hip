// One token per row of logits, drawn with given uniform numbers under
// temperature, top-k, top-p and min-p (the runner's sampling step,
// hf_benchmark.py:578-606, with top-k and min-p beside it).
//
// Row: w_i = e^((x_i - m) / T) with m the largest logit. Tokens stand in the
// order of falling logit, equal ones by index. All three filters keep a prefix
// of that order: top-k its first k; top-p those whose mass before them is at
// most p times the mass of the first k; min-p those with w >= min_p. The
// shortest prefix stays, with mass S, and the token is the first whose
// cumulative mass exceeds u S.
//
// A weight is held as the integer nearest to w 2^s, s so that a row's sum fits
// 63 bits (46 at 131072 tokens): sums of integers have no rounding and no
// order, so atomics and any split of a row give the same token, and p M and
// u S are compared exactly. A mass is off by half a unit a token, 2^-47 of the
// likeliest token's weight at 131072 tokens, and by 2.4e-15 of itself from the
// exponential (11 units of a weight at s = 52, the most); fp32 sums would move
// the border of a token by more than what a rare token weighs. The exponential is
// a double polynomial: fp64 multiply-adds issue at the rate of unpacked fp32 ones
// here.
#include "ikl_common.h"
#include "sample_row.h"

namespace ikl {
namespace {

// Leaves the tokens of the cuts' bins among the `n` candidates in sh.list, as far as
// it holds them, and returns their number.
__device__ inline uint32_t drop_uncut(const Binner &bin_of, uint32_t n, WholeRowShared &sh) {
  constexpr int PER = CANDIDATES / SAMPLE_THREADS, FEW = LIST / SAMPLE_THREADS;
  const Cuts cuts = sh.cuts;
  double word[PER];
  const auto fetch = [&](int i) {
    const int at = threadIdx.x + i * SAMPLE_THREADS;
    word[i] = i < FEW ? sh.list[at] : sh.more[at - LIST];
  };
  const auto keep = [&](int i) {
    if (threadIdx.x + i * SAMPLE_THREADS < n && cuts.has(bin_of(word_logit(word[i])))) {
      const uint32_t at = atomicAdd(&sh.listed, 1u);
      if (at < LIST) sh.list[at] = word[i];
    }
  };
#pragma unroll
  for (int i = 0; i < FEW; ++i) fetch(i);
  __syncthreads();
  if (threadIdx.x == 0) sh.listed = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < FEW; ++i) keep(i);
  if (n > LIST) {
#pragma unroll
    for (int i = FEW; i < PER; ++i) fetch(i);
#pragma unroll
    for (int i = FEW; i < PER; ++i) keep(i);
  }
  __syncthreads();
  return sh.listed;
}

// The draw of a row whose cuts' bins hold `n` tokens, listed if they are at most LIST.
template <typename Tag>
__device__ inline void draw(const SampleParams &p, int64_t b, const RowReader<Tag> &row, const RowSettings &set,
                            const Weigher &weigh, const Binner &bin_of, uint32_t n, RowShared &sh) {
  if (n > LIST) return sample_by_radix<Tag>(p, b, row, set, weigh, sh);
  if (n > 256) return sample_from_list(p, b, set, weigh, bin_of, (int)n, sh);
  if (n > 64) rank_list((int)n, sh);
  if (threadIdx.x >= 64) return;
  if (n > 64) sample_from_few<4>(p, b, set, weigh, bin_of, (int)n, sh);
  else sample_from_few<1>(p, b, set, weigh, bin_of, (int)n, sh);
}

constexpr int MAX_PARTS = 64;

// The tokens of the cuts' bins among the vectors [from, to) of the row.
template <typename Tag>
__device__ inline void list_tokens(const RowReader<Tag> &row, int from, int to, const Weigher &weigh,
                                   const Candidates &cand, const Binner &bin_of, const v4u32 &begin, RowShared &sh) {
  const Cuts cuts = sh.cuts;
  row.each(from, to, begin, [&](int first, const float(&x)[RowReader<Tag>::VEC]) {
    uint32_t hits = 0;
#pragma unroll
    for (int j = 0; j < RowReader<Tag>::VEC; ++j) hits |= (uint32_t)cuts.has(bin_of(x[j])) << j;
    while (hits) {
      const int j = __ffs(hits) - 1;
      hits &= hits - 1;
      float y = x[0];
#pragma unroll
      for (int k = 1; k < RowReader<Tag>::VEC; ++k) y = j == k ? x[k] : y;
      if (!weigh.counts(y)) continue;  // those that come to 0 all the same stand behind all others
      if (cand.alone) {
        const float one[1] = {y};
        double exact[1];
        weigh.of(one, exact);
        if (exact[0] < cand.least) continue;
      }
      const uint32_t at = atomicAdd(&sh.listed, 1u);
      if (at < LIST) sh.list[at] = token_word(order_key(clean(y)), first + j);
    }
  });
}

// One workgroup per row and three passes over it: the largest logit; the
// histogram of the weights, in shared memory; the tokens of the bins where the
// cuts fall, unless min-p left so few candidates that the second pass has listed
// them all.
template <typename Tag>
__global__ __launch_bounds__(SAMPLE_THREADS) void sample_row_kernel(const SampleParams p) {
  __shared__ WholeRowShared sh;
  const int64_t b = blockIdx.x;
  const RowReader<Tag> row(p.logits + b * p.stride, p.vocab);
  const RowSettings set = row_settings(p, b);
  fill_roots(sh.roots, p.fraction_bits);
  clear_histogram(sh);
  if (threadIdx.x == 0) sh.listed = 0;
  float top = -INFINITY, least = INFINITY;
  row_extremes(row, 0, row.vectors, top, least);
  block_extremes(top, least, sh);
  if (top == -INFINITY) {
    if (threadIdx.x == 0) store_nothing(p, b);
    return;
  }
  if (top == INFINITY) {
    sample_infinite(p, b, row, set, sh);
    return;
  }
  const Weigher weigh(top, set.temperature, p.fraction_bits, sh.roots);
  const Candidates cand(set, weigh);
  const Binner bin_of(set, weigh, cand, top, least);
  uint64_t others = 0;
  row.each(0, row.vectors, [&](int first, const float(&x)[RowReader<Tag>::VEC]) {
    add_tokens(first, x, set, weigh, cand, bin_of, others, sh);
  });
  if (set.min_p > 0.f) others = block_sum(others, sh);
  if (threadIdx.x == 0) sh.others = others;
  __syncthreads();
  find_cuts(set, cand, sh);
  uint32_t n = sh.listed;
  if (!cand.alone || n > CANDIDATES) {
    __syncthreads();
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    list_tokens(row, 0, row.vectors, weigh, cand, bin_of, row.begin(0, row.vectors), sh);
    __syncthreads();
    n = sh.listed;
  } else if (n > 64) {
    n = drop_uncut(bin_of, n, sh);
  }
  draw(p, b, row, set, weigh, bin_of, n, sh);
}

// A row split over the launch's workgroups, `parts` to a row: three launches
// for the three passes. The parts' histograms and lists meet in memory, and the
// last part of a row to finish its list draws the token. Sums of integers: the
// order of arrival leaves no trace.
struct SplitRow {  // of the workspace
  uint64_t mass[BINS];
  double list[LIST];
  uint32_t count[BINS];
  uint64_t others;
  uint32_t listed, arrived;
  float top[MAX_PARTS], least[MAX_PARTS];
};

// What a row's parts hand over inside a launch is written and read by atomic
// operations of device scope only: they take effect in memory, past the caches
// of the 8 dies, so no cache has to be written back. (With a device-wide fence
// in each wave instead, 32 rows of 131072 tokens took 155 us a launch.)
template <typename T>
__device__ inline T shared_load(const T *p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T>
__device__ inline void shared_store(T *p, T v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Whether this workgroup is the row's last to come here. Each wave waits for its
// own operations to be complete before the workgroup's arrival is counted; the
// fence keeps the compiler from moving any of them behind the wait.
__device__ inline bool last_to_arrive(uint32_t *arrived, int parts, RowShared &sh) {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0) sh.found[0] = atomicAdd(arrived, 1u) == (uint32_t)(parts - 1);
  __syncthreads();
  const bool last = sh.found[0] != 0;
  __syncthreads();
  return last;
}

// This workgroup's row and its vectors of it.
template <typename Tag>
struct Part {
  int64_t b;
  RowReader<Tag> row;
  int part, from, to;
  __device__ inline Part(const SampleParams &p, int parts)
      : b(blockIdx.x / parts), row(p.logits + b * p.stride, p.vocab), part((int)(blockIdx.x - b * parts)) {
    const int per = (row.vectors + parts - 1) / parts;
    from = min(part * per, row.vectors);
    to = min(from + per, row.vectors);
  }
};

template <typename Tag>
__global__ __launch_bounds__(SAMPLE_THREADS) void sample_extremes_kernel(const SampleParams p, SplitRow *rows, int parts) {
  __shared__ RowShared sh;
  const Part<Tag> at(p, parts);
  SplitRow &r = rows[at.b];
  for (int i = at.part * SAMPLE_THREADS + threadIdx.x; i < BINS; i += parts * SAMPLE_THREADS) {
    r.mass[i] = 0;
    r.count[i] = 0;
  }
  float top = -INFINITY, least = INFINITY;
  row_extremes(at.row, at.from, at.to, top, least);
  block_extremes(top, least, sh);
  if (threadIdx.x == 0) {
    r.top[at.part] = top;
    r.least[at.part] = least;
    if (at.part == 0) {
      r.others = 0;
      r.listed = r.arrived = 0;
    }
  }
}

__device__ inline void joined_extremes(const SplitRow &r, int parts, float &top, float &least) {
  const int lane = threadIdx.x & 63;  // MAX_PARTS lanes
  top = wave_max(lane < parts ? r.top[lane] : -INFINITY);
  least = -wave_max(lane < parts ? -r.least[lane] : -INFINITY);
}

template <typename Tag>
__global__ __launch_bounds__(SAMPLE_THREADS) void sample_histogram_kernel(const SampleParams p, SplitRow *rows, int parts) {
  __shared__ RowShared sh;
  const Part<Tag> at(p, parts);
  SplitRow &r = rows[at.b];
  const v4u32 begin = at.row.begin(at.from, at.to);  // on its way meanwhile
  fill_roots(sh.roots, p.fraction_bits);
  clear_histogram(sh);
  const RowSettings set = row_settings(p, at.b);
  float top, least;
  joined_extremes(r, parts, top, least);
  if (top == -INFINITY || top == INFINITY) return;
  const Weigher weigh(top, set.temperature, p.fraction_bits, sh.roots);
  const Candidates cand(set, weigh);
  const Binner bin_of(set, weigh, cand, top, least);
  uint64_t others = 0;
  __syncthreads();
  at.row.each(at.from, at.to, begin, [&](int first, const float(&x)[RowReader<Tag>::VEC]) {
    add_tokens(first, x, set, weigh, cand, bin_of, others, sh);
  });
  if (set.min_p > 0.f) {
    others = block_sum(others, sh);
    if (threadIdx.x == 0) atomicAdd((unsigned long long *)&r.others, (unsigned long long)others);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += SAMPLE_THREADS) {
    if (sh.mass[i]) atomicAdd((unsigned long long *)&r.mass[i], (unsigned long long)sh.mass[i]);
    if (sh.count[i]) atomicAdd(&r.count[i], sh.count[i]);
  }
}

template <typename Tag>
__global__ __launch_bounds__(SAMPLE_THREADS, 8) void sample_pick_kernel(const SampleParams p, SplitRow *rows, int parts) {
  __shared__ RowShared sh;
  const Part<Tag> at(p, parts);
  SplitRow &r = rows[at.b];
  const v4u32 begin = at.row.begin(at.from, at.to);  // these are on their way meanwhile
  uint64_t mass[BINS / SAMPLE_THREADS];
  uint32_t count[BINS / SAMPLE_THREADS];
#pragma unroll
  for (int i = 0; i < BINS / SAMPLE_THREADS; ++i) {
    mass[i] = r.mass[threadIdx.x + i * SAMPLE_THREADS];
    count[i] = r.count[threadIdx.x + i * SAMPLE_THREADS];
  }
  const RowSettings set = row_settings(p, at.b);
  float top, least;
  joined_extremes(r, parts, top, least);
  if (top == -INFINITY || top == INFINITY) {  // nothing to weigh
    if (at.part != 0) return;
    if (top == INFINITY) sample_infinite(p, at.b, at.row, set, sh);
    else if (threadIdx.x == 0) store_nothing(p, at.b);
    return;
  }
  fill_roots(sh.roots, p.fraction_bits);
#pragma unroll
  for (int i = 0; i < BINS / SAMPLE_THREADS; ++i) {
    sh.mass[threadIdx.x + i * SAMPLE_THREADS] = mass[i];
    sh.count[threadIdx.x + i * SAMPLE_THREADS] = count[i];
  }
  if (threadIdx.x == 0) {
    sh.listed = 0;
    sh.others = r.others;
  }
  const Weigher weigh(top, set.temperature, p.fraction_bits, sh.roots);
  const Candidates cand(set, weigh);
  const Binner bin_of(set, weigh, cand, top, least);
  __syncthreads();
  find_cuts(set, cand, sh);
  list_tokens(at.row, at.from, at.to, weigh, cand, bin_of, begin, sh);
  __syncthreads();
  const uint32_t mine = sh.listed;
  if (threadIdx.x == 0) sh.found[1] = mine ? atomicAdd(&r.listed, mine) : 0;
  __syncthreads();
  const uint32_t start = (uint32_t)sh.found[1];  // past LIST in all, no list is read
  for (uint32_t i = threadIdx.x; i < mine && i < LIST && start + i < LIST; i += SAMPLE_THREADS)
    shared_store(&r.list[start + i], sh.list[i]);
  if (!last_to_arrive(&r.arrived, parts, sh)) return;
  const uint32_t n = shared_load(&r.listed);
  for (uint32_t i = threadIdx.x; i < n && i < LIST; i += SAMPLE_THREADS) sh.list[i] = shared_load(&r.list[i]);
  __syncthreads();
  draw(p, at.b, at.row, set, weigh, bin_of, n, sh);
}

// Workgroups of a row. One is one launch, three where a row is split, which pays
// from 24 tokens a thread (us with top-p 0.95, one / split by 4: 1 x 24000 bf16 17.2
// / 18.4, 1 x 16000 fp32 13.4 / 16.4, 1 x 32000 bf16 20.6 / 19.4; not for 48 x 32000,
// 21.7 / 23.0): into as many parts as have a vector a thread, as long as there is a
// compute unit for each (bf16 x 131072, in 1, 4, 8 and 16: 1 row 59, 32, 27, 24; 32
// rows 63, 37, 33, 40; 128 rows 64, 60, 76, in 2 54; in 1 and 2: 129 rows 64, 75, 192
// rows 66, 83, 257 rows 115, 105; 256 rows fp32 in 1 and 4: 84, 108). Two parts do not
// pay for rows under 64 tokens a thread (100 x 50257 30.3 / 33.1).
int parts_of(int64_t rows, int64_t vocab, int64_t dtype) {
  if (vocab <= 24 * SAMPLE_THREADS) return 1;
  const int64_t per = dtype == IKL_F32 ? 4 : 8, vectors = (vocab + per - 1) / per;
  const int64_t most = (vectors + SAMPLE_THREADS - 1) / SAMPLE_THREADS, want = 256 / rows;
  const int64_t n = most < want ? most : want;
  if (n < (vocab < 64 * SAMPLE_THREADS ? 3 : 2)) return 1;
  return (int)(n < MAX_PARTS ? n : MAX_PARTS);
}

template <typename Tag>
void launch(const SampleParams &p, int64_t rows, int parts, SplitRow *split, hipStream_t s) {
  if (parts == 1) {
    sample_row_kernel<Tag><<<dim3((unsigned)rows), SAMPLE_THREADS, 0, s>>>(p);
    return;
  }
  const dim3 grid((unsigned)(rows * parts));
  sample_extremes_kernel<Tag><<<grid, SAMPLE_THREADS, 0, s>>>(p, split, parts);
  sample_histogram_kernel<Tag><<<grid, SAMPLE_THREADS, 0, s>>>(p, split, parts);
  sample_pick_kernel<Tag><<<grid, SAMPLE_THREADS, 0, s>>>(p, split, parts);
}

}  // namespace
}  // namespace ikl

using namespace ikl;

extern "C" int ikl_sample_tokens(const ikl_sample_args *a, void *stream) {
  if (!a) return fail(IKL_EINVAL, "sample: null argument struct");
  if (a->rows < 0) return fail(IKL_EINVAL, "sample: rows must be non-negative");
  if (a->vocab <= 0) return fail(IKL_EINVAL, "sample: vocab must be positive");
  if (a->vocab > IKL_SAMPLE_MAX_VOCAB) return fail(IKL_EUNSUPPORTED, "sample: vocab above IKL_SAMPLE_MAX_VOCAB");
  int eb;
  switch (a->dtype) {
    case IKL_F16:
    case IKL_BF16: eb = 2; break;
    case IKL_F32: eb = 4; break;
    default: return fail(IKL_EINVAL, "sample: unsupported dtype");
  }
  if (a->rows == 0) return IKL_OK;
  if (a->rows > max_grid(SAMPLE_THREADS)) return fail(IKL_EINVAL, "sample: too many rows for one launch");
  if (!a->logits || !a->uniform || !a->tokens) return fail(IKL_EINVAL, "sample: null tensor pointer");
  if (a->top_k_rows && a->top_k_type != IKL_I32 && a->top_k_type != IKL_I64)
    return fail(IKL_EINVAL, "sample: top_k must use int32 or int64");
  if ((uintptr_t)a->logits % eb || (uintptr_t)a->uniform % 4 || (uintptr_t)a->tokens % 8)
    return fail(IKL_EINVAL, "sample: misaligned tensor");
  SampleParams p;
  p.logits = (const char *)a->logits;
  p.stride = a->logits_stride * eb;
  p.uniform = (const float *)a->uniform;
  p.temperature_rows = (const float *)a->temperature_rows;
  p.top_k_rows = a->top_k_rows;
  p.top_k_wide = a->top_k_type == IKL_I64;
  p.top_p_rows = (const float *)a->top_p_rows;
  p.min_p_rows = (const float *)a->min_p_rows;
  p.temperature = a->temperature;
  p.top_k = a->top_k;
  p.top_p = a->top_p;
  p.min_p = a->min_p;
  p.tokens = (int64_t *)a->tokens;
  p.policy = (float *)a->policy_logprobs;
  p.sampling = (float *)a->sampling_logprobs;
  p.vocab = (int32_t)a->vocab;
  p.fraction_bits = fraction_bits(a->vocab);
  const int parts = parts_of(a->rows, a->vocab, a->dtype);
  if (parts > 1 && (!a->workspace || (uintptr_t)a->workspace % 16 ||
                    a->workspace_bytes < a->rows * (int64_t)sizeof(SplitRow)))
    return fail(IKL_EWORKSPACE, "sample: workspace missing, misaligned or too small");
  SplitRow *split = (SplitRow *)a->workspace;
  hipStream_t s = (hipStream_t)stream;
  switch (a->dtype) {
    case IKL_F16: launch<f16_tag>(p, a->rows, parts, split, s); break;
    case IKL_BF16: launch<bf16_tag>(p, a->rows, parts, split, s); break;
    default: launch<f32_tag>(p, a->rows, parts, split, s); break;
  }
  return check_launch("sample launch");
}

extern "C" int64_t ikl_sample_workspace_size(const ikl_sample_args *a) {
  if (!a || a->rows < 0 || a->vocab <= 0 || a->vocab > IKL_SAMPLE_MAX_VOCAB)
    return fail(IKL_EINVAL, "sample: invalid sizes");
  if (a->rows == 0 || parts_of(a->rows, a->vocab, a->dtype) == 1) return 0;
  return a->rows * (int64_t)sizeof(SplitRow);
}
