// RMSNorm of each query and key head, rotate-half RoPE and the KV append in
// one launch, for models that normalise their heads before attention (beside
// rope_append.hip, which rotates and appends them as they are).
//
// y = x r w with r = (mean(x^2) + eps)^-1/2 over a head's row; out = y cos +
// rotate_half(y) sin, in fp32 from the loads to the one rounding of the store
// (as separate modules the row would be rounded after the norm, after the
// weight and three times in the rotation); an FP8 cache quantises the fp32
// row.
//
// LPR lanes hold a row, each a 16-byte piece of the first half and the piece
// D/2 later that rotate-half pairs with it, so the sum of squares crosses
// log2(LPR) lanes and nothing is loaded twice. v rows go through the same
// lanes unchanged. Lane groups are numbered over the rows of all tokens: few
// heads fill a wave as well as many. Bound: memory; 8192 tokens of 32/8 heads of
// 128, bf16, take 44.6 us or 4.6 TB/s (a copy: 5.2), back to back. In a graph, the
// forms in turn: 45.7 us, 45.9 with the row's token by a 64-bit division, 48.8 with
// stores that stay in the caches; 32 tokens 2.92, 3.04 and 2.96. Three rows a group
// with their loads ahead were no faster and cost few tokens dearly (32: 5.1 us).
#include "fp8_row.h"
#include "ikl_common.h"
#include "rope_args.h"

namespace ikl {
namespace {

struct NormRopeParams {
  RopeParams r;
  const char *q_w;
  const char *k_w;
  int64_t qw_sh, kw_sh;  // bytes
  float *k_scale;        // FP8 cache
  float *v_scale;
  int64_t s_sb, s_sh;    // elements
  int64_t tokens;
  float inv_dim, eps;
};

template <typename Tag>
struct piece {  // 16 bytes of a row as floats
  static constexpr int N = 8;
  __device__ static inline void get(const u32x4 &w, float *x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = elem<Tag>::lo(u32x4_at(w, i));
      x[2 * i + 1] = elem<Tag>::hi(u32x4_at(w, i));
    }
  }
  __device__ static inline u32x4 put(const float *x) {
    return u32x4{elem<Tag>::pack2(x[0], x[1]), elem<Tag>::pack2(x[2], x[3]), elem<Tag>::pack2(x[4], x[5]),
                 elem<Tag>::pack2(x[6], x[7])};
  }
};
template <>
struct piece<f32_tag> {
  static constexpr int N = 4;
  __device__ static inline void get(const u32x4 &w, float *x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(u32x4_at(w, i));
  }
  __device__ static inline u32x4 put(const float *x) {
    return u32x4{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
  }
};

template <int N>
__device__ inline float lanes_sum(float v) {
  v = group_sum<N < 16 ? N : 16>(v);
  if constexpr (N >= 32) v = sum_xor16(v);
  if constexpr (N >= 64) v = sum_xor32(v);
  return v;
}

// N codes of a row's piece
template <int N>
__device__ inline void store_codes(char *p, const float *x, float scale) {
#pragma unroll
  for (int i = 0; i < N; i += 4) *reinterpret_cast<int *>(p + i) = fp8x4(x + i, scale);
}

__device__ inline void store_out(char *p, const u32x4 &v) {
  __builtin_nontemporal_store((v4u32){v.x, v.y, v.z, v.w}, reinterpret_cast<v4u32 *>(p));
}

template <typename Tag, typename IdxT, int LPR, bool FP8>
__global__ __launch_bounds__(256) void norm_rope_kernel(const NormRopeParams f) {
  using P = piece<Tag>;
  constexpr int N = P::N;
  const RopeParams &p = f.r;
  const int lane = threadIdx.x % LPR;
  const int rows = p.num_heads + 2 * p.num_kv_heads;  // of a token: q, then k, then v
  const uint32_t group = blockIdx.x * (256 / LPR) + threadIdx.x / LPR, all = (uint32_t)f.tokens * (uint32_t)rows;
  const bool has = group < all;  // groups past the last row read it again
  const uint32_t index = has ? group : all - 1, token = index / (uint32_t)rows;
  const int64_t t = token;
  const int row = (int)(index - token * (uint32_t)rows);
  const int kv_row = row - p.num_heads;
  const bool is_q = kv_row < 0, is_v = kv_row >= p.num_kv_heads;
  const int h = is_q ? row : is_v ? kv_row - p.num_kv_heads : kv_row;
  const int hc = p.half_chunks;
  const bool on = lane < hc;
  const int lo = on ? lane * 16 : 0, hi = on ? (lane + hc) * 16 : 0;  // bytes; idle lanes read along
  const int64_t slot = (int64_t)reinterpret_cast<const IdxT *>(p.slots)[t];
  const bool slot_ok = slot >= 0 && slot < p.num_slots;
  const int64_t blk = slot_ok ? slot / p.block_size : 0;
  const int64_t off = slot_ok ? slot - blk * p.block_size : 0;
  const char *src = is_q ? p.q_in + t * p.qi_st + h * p.qi_sh
                         : is_v ? p.value + t * p.v_st + h * p.v_sh : p.key + t * p.k_st + h * p.k_sh;
  const u32x4 xl = load16(src + lo), xh = load16(src + hi);
  float a[N], b[N];
  P::get(xl, a);
  P::get(xh, b);
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) ss = fmaf(a[i], a[i], fmaf(b[i], b[i], ss));
  const float r = rsqrtf(lanes_sum<LPR>(on ? ss : 0.f) * f.inv_dim + f.eps);
  if (!is_v) {
    const char *w = is_q ? f.q_w + h * f.qw_sh : f.k_w + h * f.kw_sh;
    const char *c = p.cos + t * p.cos_st, *s = p.sin + t * p.sin_st;
    float w1[N], w2[N], c1[N], c2[N], s1[N], s2[N];
    P::get(load16(w + lo), w1);
    P::get(load16(w + hi), w2);
    P::get(load16(c + lo), c1);
    P::get(load16(c + hi), c2);
    P::get(load16(s + lo), s1);
    P::get(load16(s + hi), s2);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float y1 = a[i] * r * w1[i], y2 = b[i] * r * w2[i];
      a[i] = y1 * c1[i] - y2 * s1[i];
      b[i] = y2 * c2[i] + y1 * s2[i];
    }
  }
  if (is_q) {
    if (has && on) {
      char *dst = p.q_out + t * p.qo_st + h * p.qo_sh;
      store_out(dst + lo, P::put(a));
      store_out(dst + hi, P::put(b));
    }
    if constexpr (!FP8) return;
  }
  char *dst = is_v ? p.vc + blk * p.vc_sb + off * p.vc_st + h * p.vc_sh
                   : p.kc + blk * p.kc_sb + off * p.kc_st + h * p.kc_sh;
  if constexpr (!FP8) {
    if (!has || !on || !slot_ok) return;
    store_out(dst + lo, is_v ? xl : P::put(a));
    store_out(dst + hi, is_v ? xh : P::put(b));
  } else {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, fmaxf(fabsf(a[i]), fabsf(b[i])));
    const float scale = e4m3_row_scale(group_max<LPR>(on ? m : 0.f));  // every lane of the wave takes part
    if (is_q || !has || !slot_ok) return;
    if (on) {
      store_codes<N>(dst + lane * N, a, scale);
      store_codes<N>(dst + (lane + hc) * N, b, scale);
    }
    if (lane == 0) (is_v ? f.v_scale : f.k_scale)[blk * f.s_sb + h * f.s_sh + off] = scale;
  }
}

template <typename Tag, int LPR, bool FP8>
int launch(const NormRopeParams &f, bool i64, hipStream_t s) {
  const int64_t rows = f.tokens * (f.r.num_heads + 2 * (int64_t)f.r.num_kv_heads), per = 256 / LPR;
  const int64_t grid = (rows + per - 1) / per;
  if (grid > max_grid(256)) return fail(IKL_EINVAL, "norm rope append: too many rows for one launch");
  if (i64) norm_rope_kernel<Tag, int64_t, LPR, FP8><<<dim3((unsigned)grid), 256, 0, s>>>(f);
  else norm_rope_kernel<Tag, int32_t, LPR, FP8><<<dim3((unsigned)grid), 256, 0, s>>>(f);
  return check_launch("norm rope append launch");
}

template <typename Tag, bool FP8>
int launch(const NormRopeParams &f, bool i64, hipStream_t s) {
  const int hc = f.r.half_chunks;
  if (hc <= 4) return launch<Tag, 4, FP8>(f, i64, s);
  if (hc <= 8) return launch<Tag, 8, FP8>(f, i64, s);
  if (hc <= 16) return launch<Tag, 16, FP8>(f, i64, s);
  if (hc <= 32) return launch<Tag, 32, FP8>(f, i64, s);
  return launch<Tag, 64, FP8>(f, i64, s);
}

template <typename Tag>
int launch(const NormRopeParams &f, bool fp8, bool i64, hipStream_t s) {
  return fp8 ? launch<Tag, true>(f, i64, s) : launch<Tag, false>(f, i64, s);
}

}  // namespace
}  // namespace ikl

using namespace ikl;

extern "C" int ikl_qk_norm_rope_append_kv(const ikl_qk_norm_rope_args *args, void *stream) {
  if (!args) return fail(IKL_EINVAL, "norm rope append: null argument struct");
  const ikl_rope_append_args *a = &args->rope;
  NormRopeParams f;
  if (const int bad = rope_params(a, "norm rope append", &f.r); bad != IKL_OK) return bad;
  if (a->num_tokens == 0) return IKL_OK;
  const int eb = a->dtype == IKL_F32 ? 4 : 2;
  if ((int64_t)a->head_dim * eb > 2048)
    return fail(IKL_EUNSUPPORTED, "norm rope append: head_dim * element size above 2048 bytes");
  if (!args->k_weight || (a->num_heads > 0 && !args->q_weight))
    return fail(IKL_EINVAL, "norm rope append: null weight");
  if (!(args->eps >= 0.f)) return fail(IKL_EINVAL, "norm rope append: eps must be non-negative");
  if ((int64_t)a->num_heads + 2 * (int64_t)a->num_kv_heads > 0x7fffffffLL)
    return fail(IKL_EINVAL, "norm rope append: too many heads");
  f.q_w = (const char *)args->q_weight;
  f.k_w = (const char *)args->k_weight;
  f.qw_sh = args->q_weight_stride_h * eb;
  f.kw_sh = args->k_weight_stride_h * eb;
  if (!al16(f.k_w) || f.kw_sh % 16 != 0 || (a->num_heads > 0 && (!al16(f.q_w) || f.qw_sh % 16 != 0)))
    return fail(IKL_EINVAL, "norm rope append: rows must be 16-byte aligned");
  f.k_scale = (float *)a->k_scale;
  f.v_scale = (float *)a->v_scale;
  f.s_sb = a->scale_stride_block;
  f.s_sh = a->scale_stride_head;
  f.tokens = a->num_tokens;
  f.inv_dim = 1.f / (float)a->head_dim;
  f.eps = args->eps;
  const bool fp8 = a->cache_dtype == IKL_FP8_E4M3, i64 = a->slot_type == IKL_I64;
  hipStream_t s = (hipStream_t)stream;
  switch (a->dtype) {
    case IKL_F16: return launch<f16_tag>(f, fp8, i64, s);
    case IKL_BF16: return launch<bf16_tag>(f, fp8, i64, s);
    default: return launch<f32_tag>(f, fp8, i64, s);
  }
}
