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
// u S are compared exactly. The error of a mass is at most half a unit a token,
// 2^-47 of the likeliest token's weight; fp32 sums would move the border of a
// token by more than what a rare token weighs. The exponential is a double
// polynomial: fp64 multiply-adds issue at the rate of unpacked fp32 ones here.
#include "ikl_common.h"
#include "sample_row.h"

namespace ikl {
namespace {

// One workgroup per row and three passes over it: the largest logit; the
// histogram of the weights, in shared memory; the tokens of the bins where the
// cuts fall.
template <typename Tag>
__global__ __launch_bounds__(SAMPLE_THREADS) void sample_row_kernel(const SampleParams p) {
  __shared__ RowShared sh;
  const int64_t b = blockIdx.x;
  const RowReader<Tag> row(p.logits + b * p.stride, p.vocab);
  const RowSettings set = row_settings(p, b);
  uint32_t top = 0, least = 0xffffffffu;
  for (int v = threadIdx.x; v < row.vectors; v += SAMPLE_THREADS)
    row.each(v, [&](int, float x) { extremes(x, top, least); });
  block_extremes(top, least, sh);
  if (top <= KEY_NEG_INF) {
    if (threadIdx.x == 0) store_nothing(p, b);
    return;
  }
  const Weigher weigh(top, set.temperature, p.fraction_bits);
  const Binner bin_of(weigh, least);
  Totals sums;
  clear_histogram(sh);
  __syncthreads();
  for (int v = threadIdx.x; v < row.vectors; v += SAMPLE_THREADS)
    row.each(v, [&](int, float x) { add_token(x, set, weigh, bin_of, sums, sh); });
  const uint64_t total = block_sum(sums.total, sh);
  const uint64_t likely = set.min_p > 0.f ? block_sum(sums.likely, sh) : total;
  const uint64_t count = set.top_k > 0 ? block_sum(sums.count, sh) : 0;
  const Cuts cuts = find_cuts(set, total, likely, count, sh);
  if (threadIdx.x == 0) sh.listed = 0;
  __syncthreads();
  for (int v = threadIdx.x; v < row.vectors; v += SAMPLE_THREADS)
    row.each(v, [&](int i, float x) {
      if (!cuts.has(bin_of(x)) || weigh(x) == 0) return;
      const uint32_t at = atomicAdd(&sh.listed, 1u);
      if (at < LIST) sh.list[at] = token_word(order_key(x), i);
    });
  __syncthreads();
  const uint32_t n = sh.listed;
  if (n <= LIST) sample_from_list(p, b, set, weigh, bin_of, total, likely, count, (int)n, sh);
  else sample_by_radix<Tag>(p, b, row, set, weigh, total, likely, count, sh);
}

template <typename Tag>
void launch(const SampleParams &p, int64_t rows, hipStream_t s) {
  sample_row_kernel<Tag><<<dim3((unsigned)rows), SAMPLE_THREADS, 0, s>>>(p);
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
  if (a->rows > 0x7fffffffLL) return fail(IKL_EINVAL, "sample: too many rows for one launch");
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
  hipStream_t s = (hipStream_t)stream;
  switch (a->dtype) {
    case IKL_F16: launch<f16_tag>(p, a->rows, s); break;
    case IKL_BF16: launch<bf16_tag>(p, a->rows, s); break;
    default: launch<f32_tag>(p, a->rows, s); break;
  }
  return check_launch("sample launch");
}

extern "C" int64_t ikl_sample_workspace_size(const ikl_sample_args *a) {
  if (!a || a->rows < 0 || a->vocab <= 0 || a->vocab > IKL_SAMPLE_MAX_VOCAB)
    return fail(IKL_EINVAL, "sample: invalid sizes");
  return 0;
}
