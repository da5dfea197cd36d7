// Rows in 8 bits with a scale for each row and group of 32, 64 or 128 columns:
// of a tensor's rows, of SiLU(gate) * up, and of RMSNorm after the residual
// add; and back to 16 bits or fp32.
//
// A group's scale is a = max(amax, 2^-100) / 127 and its codes are the whole
// numbers nearest to v / a. The values v of the norm and the activation are
// fp32 and rounded nowhere but in their codes: half a step, amax / 254, is far
// more than fp32's arithmetic adds. amax is taken as an unsigned maximum of
// the bits of |v|, in which a NaN or an infinity is the largest: its group's
// scale is then not finite and the whole group stands for NaN.
#include "ikl_common.h"
#include "mfma_ops.h"

namespace ikl {
namespace {

constexpr float LEAST_AMAX = 0x1p-100f;  // 127 / amax stays finite

// The 16-byte piece of a row that a lane holds, widened.
template <typename Tag>
struct piece {
  static constexpr int N = 8;
  __device__ static inline void get(const v4u32 &w, float *x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = mfma_ops<Tag>::lo(w[i]);
      x[2 * i + 1] = mfma_ops<Tag>::hi(w[i]);
    }
  }
  __device__ static inline v4u32 put(const float *x) {
    v4u32 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = mfma_ops<Tag>::pack(x[2 * i], x[2 * i + 1]);
    return w;
  }
};
template <>
struct piece<f32_tag> {
  static constexpr int N = 4;
  __device__ static inline void get(const v4u32 &w, float *x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]);
  }
  __device__ static inline v4u32 put(const float *x) {
    return v4u32{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
  }
};

template <int CTRL>
__device__ inline uint32_t dpp_max(uint32_t v) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, false);
  return v > o ? v : o;
}

// Maximum over aligned groups of LANES (4 .. 32) lanes, in every lane of them.
template <int LANES>
__device__ inline uint32_t group_max(uint32_t v) {
  v = dpp_max<DPP_QUAD_XOR1>(v);
  v = dpp_max<DPP_QUAD_XOR2>(v);
  if constexpr (LANES >= 8) v = dpp_max<DPP_ROW_HALF_MIRROR>(v);
  if constexpr (LANES >= 16) v = dpp_max<DPP_ROW_MIRROR>(v);
  if constexpr (LANES >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = r[0] > r[1] ? r[0] : r[1];
  }
  return v;
}

// Largest magnitude of the group that this lane holds N values of.
template <int N, int LANES>
__device__ inline float group_amax(const float *v) {
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
    amax = amax > b ? amax : b;
  }
  return __uint_as_float(group_max<LANES>(amax));
}

// Codes of this lane's N values, whose group's largest magnitude is `most`.
// Adding 1.5 * 2^23 rounds to the nearest whole number, ties to even, and
// leaves it in the low bits. 16-bit values meet ties often (a value and the
// largest one have few bits, so 127 v / amax is a half exactly): EXACT takes
// the quotient to its correct rounding, by its remainder, where one
// multiplication would put them on either side. (A norm's products of two fp16
// numbers have 22 bits, and 127 / 128 of them round: to 2^-16 of a step.)
template <int N, bool EXACT>
__device__ inline void codes_of(const float *v, float most, uint32_t *codes) {
  const float part = most * 0x1p-7f, inv = EXACT ? 1.f / part : 127.f / most;
#pragma unroll
  for (int j = 0; j < N / 4; ++j) {
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (EXACT) {
        const float x = v[4 * j + i] * (127.f / 128.f), t = x * inv;
        b[i] = __float_as_uint(fmaf(fmaf(-t, part, x), inv, t) + 12582912.f);
      } else {
        b[i] = __float_as_uint(fmaf(v[4 * j + i], inv, 12582912.f));
      }
    }
    const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
    codes[j] = lo | hi;
  }
}

// max(most, 2^-100), a NaN kept.
__device__ inline float at_least(float most) { return most < LEAST_AMAX ? LEAST_AMAX : most; }

template <int N>
__device__ inline void store_codes(char *p, const uint32_t *codes) {
  if constexpr (N == 8) *reinterpret_cast<u32x2_t *>(p) = u32x2_t{codes[0], codes[1]};
  else *reinterpret_cast<uint32_t *>(p) = codes[0];
}

struct RowsParams {
  const char *x;
  const char *up;  // nullptr: the rows of x
  char *codes;
  float *scales;
  int64_t x_st, up_st;  // bytes
  uint32_t pieces;      // of all rows
  uint32_t row_pieces;
};

// A lane a piece, the pieces of all rows numbered through: a group's lanes
// stand side by side in a wave, since a row is whole groups. Bound: memory.
// 4099 x 2048 fp16 6.4 us (3.9 TB/s), SiLU * up of 4096 x 14336 bf16 61 us
// (4.8 TB/s).
template <typename Tag, int G, bool SILU>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const RowsParams p) {
  constexpr int N = piece<Tag>::N, LANES = G / N;
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i >= p.pieces) return;
  const uint32_t row = i / p.row_pieces, c = i - row * p.row_pieces;
  float v[N];
  piece<Tag>::get(load16v_global(p.x + row * p.x_st + 16 * (int64_t)c), v);
  if constexpr (SILU) {
    float u[N];
    piece<Tag>::get(load16v_global(p.up + row * p.up_st + 16 * (int64_t)c), u);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = silu_fast(v[e]) * u[e];
  }
  uint32_t codes[N / 4];
  const float most = at_least(group_amax<N, LANES>(v));
  codes_of<N, !SILU>(v, most, codes);
  store_codes<N>(p.codes + (int64_t)N * i, codes);
  if (i % LANES == 0) p.scales[i / LANES] = most / 127.f;
}

struct NormParams {
  const char *x;
  const char *delta;
  const char *weight;
  char *sum;
  char *codes;
  float *scales;
  int64_t x_st, d_st, s_st;  // bytes
  int32_t pieces;            // of a row
  float inv_cols, eps;
};

// One workgroup a row, the row in registers between the sum of squares and
// the codes: each tensor crosses memory once. 8192 x 4096 bf16 with the add
// 48.9 us (4.8 TB/s).
template <typename Tag, int G, int NV>
__global__ __launch_bounds__(256) void norm_int8_kernel(const NormParams p) {
  constexpr int N = piece<Tag>::N, LANES = G / N;
  __shared__ float part[4];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  v4u32 v[NV];
  float ss = 0.f;
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const int c = tid + 256 * u;
    if (c >= p.pieces) continue;
    v[u] = load16v_global(p.x + row * p.x_st + 16 * (int64_t)c);
    float a[N];
    piece<Tag>::get(v[u], a);
    if (p.delta) {
      float b[N];
      piece<Tag>::get(load16v_global(p.delta + row * p.d_st + 16 * (int64_t)c), b);
#pragma unroll
      for (int e = 0; e < N; ++e) a[e] += b[e];
      v[u] = piece<Tag>::put(a);
      *reinterpret_cast<v4u32 *>(p.sum + row * p.s_st + 16 * (int64_t)c) = v[u];
      piece<Tag>::get(v[u], a);
    }
#pragma unroll
    for (int e = 0; e < N; ++e) ss = fmaf(a[e], a[e], ss);
  }
  ss = sum_xor32(sum_xor16(group_sum<16>(ss)));
  if ((tid & 63) == 0) part[tid >> 6] = ss;
  __syncthreads();
  ss = (part[0] + part[1]) + (part[2] + part[3]);
  const float r = rsqrtf(ss * p.inv_cols + p.eps);
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const int c = tid + 256 * u;
    if (c >= p.pieces) continue;
    float a[N], w[N];
    piece<Tag>::get(v[u], a);
    piece<Tag>::get(load16v_global(p.weight + 16 * (int64_t)c), w);
#pragma unroll
    for (int e = 0; e < N; ++e) a[e] *= w[e];
    // The codes do not depend on r: they are those of x * weight, exact where
    // both have 16 bits. Where that, or its largest value by r, is near the
    // least or past fp32, they are those of x * r * weight.
    float most = group_amax<N, LANES>(a);
    const bool first = !(most >= LEAST_AMAX && most * r >= LEAST_AMAX && most < INFINITY && most * r < INFINITY);
    if (first) {
      piece<Tag>::get(v[u], a);
#pragma unroll
      for (int e = 0; e < N; ++e) a[e] = a[e] * r * w[e];
      most = at_least(group_amax<N, LANES>(a));
    }
    uint32_t codes[N / 4];
    codes_of<N, true>(a, most, codes);
    const float scale = (first ? most : most * r) / 127.f;
    const int64_t at = row * p.pieces + c;
    store_codes<N>(p.codes + N * at, codes);
    if (c % LANES == 0) p.scales[at / LANES] = scale;
  }
}

// 8192 x 4096 to bf16 19.5 us (5.2 TB/s).
template <typename Tag>
__global__ __launch_bounds__(256) void dequantize_rows_kernel(const char *codes, const float *scales, char *out,
                                                              uint32_t pieces, int shift) {
  constexpr int N = piece<Tag>::N;
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;  // 16 codes
  if (i >= pieces) return;
  const v4u32 w = load16v_global(codes + 16 * (int64_t)i);
  const float s = scales[i >> shift];
#pragma unroll
  for (int j = 0; j < 16 / N; ++j) {
    float v[N];
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = (float)(int8_t)(w[(N * j + e) / 4] >> (8 * (e & 3))) * s;
    *reinterpret_cast<v4u32 *>(out + 16 * ((int64_t)i * (16 / N) + j)) = piece<Tag>::put(v);
  }
}

bool off16(const void *ptr) { return ((uintptr_t)ptr & 15u) != 0; }

// The checks that the three forms share; `what` names the call.
int check_rows(const char *what, int64_t rows, int64_t cols, int32_t group, int32_t dtype) {
  if (rows < 0 || cols <= 0) return fail(IKL_EINVAL, std::string(what) + ": sizes must be positive");
  if (dtype != IKL_F16 && dtype != IKL_BF16 && dtype != IKL_F32)
    return fail(IKL_EINVAL, std::string(what) + ": unknown dtype");
  if (group != 32 && group != 64 && group != 128)
    return fail(IKL_EUNSUPPORTED, std::string(what) + ": groups of 32, 64 or 128 columns only");
  if (cols % group != 0) return fail(IKL_EUNSUPPORTED, std::string(what) + ": cols must be whole groups");
  return IKL_OK;
}

template <typename Tag, bool SILU>
void launch_rows(const RowsParams &p, int group, unsigned grid, hipStream_t s) {
  if (group == 128) quantize_rows_kernel<Tag, 128, SILU><<<dim3(grid), 256, 0, s>>>(p);
  else if (group == 64) quantize_rows_kernel<Tag, 64, SILU><<<dim3(grid), 256, 0, s>>>(p);
  else quantize_rows_kernel<Tag, 32, SILU><<<dim3(grid), 256, 0, s>>>(p);
}

template <typename Tag, int G>
void launch_norm_of(const NormParams &p, unsigned rows, hipStream_t s) {
  const int vecs = (p.pieces + 255) / 256;
  if (vecs <= 1) norm_int8_kernel<Tag, G, 1><<<dim3(rows), 256, 0, s>>>(p);
  else if (vecs <= 2) norm_int8_kernel<Tag, G, 2><<<dim3(rows), 256, 0, s>>>(p);
  else if (vecs <= 4) norm_int8_kernel<Tag, G, 4><<<dim3(rows), 256, 0, s>>>(p);
  else norm_int8_kernel<Tag, G, 16><<<dim3(rows), 256, 0, s>>>(p);
}

template <typename Tag>
void launch_norm(const NormParams &p, int group, unsigned rows, hipStream_t s) {
  if (group == 128) launch_norm_of<Tag, 128>(p, rows, s);
  else if (group == 64) launch_norm_of<Tag, 64>(p, rows, s);
  else launch_norm_of<Tag, 32>(p, rows, s);
}

}  // namespace
}  // namespace ikl

using namespace ikl;

extern "C" int ikl_quantize_rows_int8(const ikl_int8_rows_args *a, void *stream) {
  if (!a) return fail(IKL_EINVAL, "int8 rows: args is NULL");
  if (const int bad = check_rows("int8 rows", a->rows, a->cols, a->group, a->dtype)) return bad;
  if (a->rows == 0) return IKL_OK;
  const int64_t eb = a->dtype == IKL_F32 ? 4 : 2;
  if (!a->x || !a->codes || !a->scales) return fail(IKL_EINVAL, "int8 rows: NULL tensor pointer");
  if (off16(a->x) || off16(a->up) || off16(a->codes) || ((uintptr_t)a->scales & 3u) ||
      (a->rows > 1 && (a->x_stride * eb | (a->up ? a->up_stride * eb : 0)) % 16 != 0))
    return fail(IKL_EINVAL, "int8 rows: rows must be 16-byte aligned");
  const int64_t row_pieces = a->cols * eb / 16;
  if (a->rows > max_grid(1) / row_pieces) return fail(IKL_EINVAL, "int8 rows: too many rows for a launch");
  const int64_t pieces = a->rows * row_pieces, grid = (pieces + 255) / 256;
  if (grid > max_grid(256)) return fail(IKL_EINVAL, "int8 rows: too many rows for a launch");
  RowsParams p;
  p.x = (const char *)a->x;
  p.up = (const char *)a->up;
  p.codes = (char *)a->codes;
  p.scales = a->scales;
  p.x_st = a->rows > 1 ? a->x_stride * eb : 0;
  p.up_st = a->rows > 1 ? a->up_stride * eb : 0;
  p.pieces = (uint32_t)pieces;
  p.row_pieces = (uint32_t)row_pieces;
  hipStream_t s = (hipStream_t)stream;
  const unsigned g = (unsigned)grid;
  if (a->dtype == IKL_BF16) a->up ? launch_rows<bf16_tag, true>(p, a->group, g, s) : launch_rows<bf16_tag, false>(p, a->group, g, s);
  else if (a->dtype == IKL_F16) a->up ? launch_rows<f16_tag, true>(p, a->group, g, s) : launch_rows<f16_tag, false>(p, a->group, g, s);
  else a->up ? launch_rows<f32_tag, true>(p, a->group, g, s) : launch_rows<f32_tag, false>(p, a->group, g, s);
  return check_launch("int8 rows");
}

extern "C" int ikl_dequantize_rows_int8(const void *codes, const float *scales, void *out, int64_t rows, int64_t cols,
                                        int32_t group, int32_t dtype, void *stream) {
  if (const int bad = check_rows("dequantize rows", rows, cols, group, dtype)) return bad;
  if (rows == 0) return IKL_OK;
  if (!codes || !scales || !out) return fail(IKL_EINVAL, "dequantize rows: NULL tensor pointer");
  if (off16(codes) || off16(out) || ((uintptr_t)scales & 3u))
    return fail(IKL_EINVAL, "dequantize rows: tensors must be 16-byte aligned");
  if (rows > max_grid(1) / (cols / 16)) return fail(IKL_EINVAL, "dequantize rows: too many rows for a launch");
  const int64_t pieces = rows * (cols / 16), grid = (pieces + 255) / 256;
  if (grid > max_grid(256)) return fail(IKL_EINVAL, "dequantize rows: too many rows for a launch");
  const int shift = group == 128 ? 3 : group == 64 ? 2 : 1;
  hipStream_t s = (hipStream_t)stream;
  const dim3 g((unsigned)grid);
  const char *c = (const char *)codes;
  const uint32_t n = (uint32_t)pieces;
  if (dtype == IKL_BF16) dequantize_rows_kernel<bf16_tag><<<g, 256, 0, s>>>(c, scales, (char *)out, n, shift);
  else if (dtype == IKL_F16) dequantize_rows_kernel<f16_tag><<<g, 256, 0, s>>>(c, scales, (char *)out, n, shift);
  else dequantize_rows_kernel<f32_tag><<<g, 256, 0, s>>>(c, scales, (char *)out, n, shift);
  return check_launch("dequantize rows");
}

extern "C" int ikl_add_rms_norm_int8(const ikl_norm_int8_args *a, void *stream) {
  if (!a) return fail(IKL_EINVAL, "rms norm int8: args is NULL");
  if (const int bad = check_rows("rms norm int8", a->rows, a->cols, a->group, a->dtype)) return bad;
  if (!(a->eps >= 0.f)) return fail(IKL_EINVAL, "rms norm int8: eps must be non-negative");
  if (a->rows == 0) return IKL_OK;
  const int64_t eb = a->dtype == IKL_F32 ? 4 : 2;
  if (!a->x || !a->weight || !a->codes || !a->scales || (a->delta && !a->sum))
    return fail(IKL_EINVAL, "rms norm int8: NULL tensor pointer");
  if (off16(a->x) || off16(a->delta) || off16(a->sum) || off16(a->weight) || off16(a->codes) ||
      ((uintptr_t)a->scales & 3u) ||
      (a->rows > 1 && (a->x_stride * eb | (a->delta ? (a->delta_stride | a->sum_stride) * eb : 0)) % 16 != 0))
    return fail(IKL_EINVAL, "rms norm int8: rows must be 16-byte aligned");
  if (a->cols * eb > 65536) return fail(IKL_EUNSUPPORTED, "rms norm int8: rows of at most 64 KB");
  if (a->rows > max_grid(256)) return fail(IKL_EINVAL, "rms norm int8: too many rows for a launch");
  NormParams p;
  p.x = (const char *)a->x;
  p.delta = (const char *)a->delta;
  p.weight = (const char *)a->weight;
  p.sum = (char *)a->sum;
  p.codes = (char *)a->codes;
  p.scales = a->scales;
  const bool many = a->rows > 1;
  p.x_st = many ? a->x_stride * eb : 0;
  p.d_st = many ? a->delta_stride * eb : 0;
  p.s_st = many ? a->sum_stride * eb : 0;
  p.pieces = (int32_t)(a->cols * eb / 16);
  p.inv_cols = 1.f / (float)a->cols;
  p.eps = a->eps;
  hipStream_t s = (hipStream_t)stream;
  const unsigned rows = (unsigned)a->rows;
  if (a->dtype == IKL_BF16) launch_norm<bf16_tag>(p, a->group, rows, s);
  else if (a->dtype == IKL_F16) launch_norm<f16_tag>(p, a->group, rows, s);
  else launch_norm<f32_tag>(p, a->group, rows, s);
  return check_launch("rms norm int8");
}
