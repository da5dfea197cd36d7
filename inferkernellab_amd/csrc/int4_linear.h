// Parts that the kernels over 4-bit weights share: the parameters, the
// unpacking of codes into matrix operands, the products of a group and the
// stores of y.
//
// W[n][k] = s[n][g] (c[n][k] - z[n][g]), so with P = sum over a group of x c
// and X = sum over it of x,  y = sum_g s (P - z X).  Codes are whole numbers
// up to 15, exact in every operand type: what is rounded is the fp32 sums.
// Over 16-bit rows a code reaches its operand through the E4M3 form of its
// byte: 0 .. 15 read as E4M3 are code * 2^-9 (subnormals, then the first
// binade, whose step is the same), so one conversion with a scale turns two of
// them into 16-bit numbers: beside fp16 rows the codes themselves (scale 2^9),
// beside bf16 ones, which reach fp32's largest values, codes * 2^-11 (scale
// 2^-2), so that a group's sums, 128 * 15 * 2^-11 of the largest value at most,
// stay finite. s carries what is missing. Over 8-bit rows z is taken off the
// bytes themselves.
#pragma once

#include "ikl_common.h"
#include "mfma_ops.h"

namespace ikl {

struct Int4Params {
  const char *x;
  int64_t x_st;     // bytes
  const float *xs;  // 8-bit rows: [rows][groups]
  const char *codes;
  const float *scales;
  const uint8_t *zeros;  // nullptr: 8
  const char *res;       // nullptr: none
  int64_t res_st;        // bytes
  char *y;
  int64_t y_st;  // bytes
  float *part;   // split contraction: [split][rows][16 * tiles]; else nullptr
  int64_t rows;
  int32_t outs;    // columns of y
  int32_t tiles;   // 16-row tiles of W
  int32_t steps;   // of 128 along the contraction
  int32_t groups;  // of the contraction
  int32_t gated;
  int32_t dtype;  // of y
  int32_t wide;   // y and residual take four columns in one access
};

// How a launch is cut: `few`: the few rows' kernel, else the many rows'; mt
// tiles of 16 rows and nt of 16 columns a workgroup, `split` workgroups along
// the contraction; `blocks`: workgroups of a part of it, columns first.
struct Int4Plan {
  bool few;
  int mt, nt, split;
  int64_t blocks;
};

// One for each type of x, in a source file of its own.
void launch_int4_bf16(const Int4Params &p, int group, const Int4Plan &plan, hipStream_t s);
void launch_int4_f16(const Int4Params &p, int group, const Int4Plan &plan, hipStream_t s);
void launch_int4_i8(const Int4Params &p, int group, const Int4Plan &plan, hipStream_t s);

namespace {

struct i8_tag {};
typedef int i32x4_t __attribute__((ext_vector_type(4)));

// 8-bit rows: each sum of a group leaves the matrix core as a whole number
// below 2^22 (of codes times 16 without zero points: below 2^21) on top of
// MAGIC, the bits of 1.5 * 2^23 as a float: the number as a float, without a
// conversion. What turns it into its share of y are two multiply-adds: first
// times a of its row less MAGIC times a, which is exact because a is rounded to
// 22 significant bits (to the nearest: 2^-22 of it at most, as in two fp32
// operations), then times s of its column. a carries 2^-17 and s 2^17
// (without zero points 2^13), so that MAGIC * a stays finite up to fp32's
// largest value over 127.
constexpr int MAGIC = 0x4b400000;
template <bool Z>
constexpr float S_CARRIES = Z ? 0x1p17f : 0x1p13f;
__device__ inline f32x2_t row_scale(float a) {
#pragma clang fp contract(off)
  a *= 0x1p-17f;
  // Dekker's split: the sum and difference with 4 times more round a to 24 - 2 bits
  const float more = a * 5.f, less = a - more;
  a = more + less;
  return f32x2_t{a, a * -12582912.f};
}

// ------------------------------------------------------------- operands
// HELD: what a code is held at in an operand; ONES: two 16-bit numbers of it.
template <typename XT>
struct codes_as;
template <>
struct codes_as<bf16_tag> {
  static constexpr float HELD = 0x1p-11f;
  static constexpr uint32_t ONES = 0x3a003a00u;
  __device__ static inline uint32_t two(uint32_t w, bool high) {
    return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 512.f * HELD, true))
                : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 512.f * HELD, false));
  }
};
template <>
struct codes_as<f16_tag> {
  static constexpr float HELD = 1.f;
  static constexpr uint32_t ONES = 0x3c003c00u;
  __device__ static inline uint32_t two(uint32_t w, bool high) {
    return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 512.f * HELD, true))
                : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 512.f * HELD, false));
  }
};

// The 8 codes of a dword, times HELD, as an operand.
template <typename XT>
__device__ inline v4u32 unpack16(uint32_t w) {
  const uint32_t lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;
  return v4u32{codes_as<XT>::two(lo, false), codes_as<XT>::two(lo, true), codes_as<XT>::two(hi, false),
               codes_as<XT>::two(hi, true)};
}

// The 8 codes of a dword less the zero point (its byte in all four bytes of
// z4), as signed bytes: the high bit keeps a byte's borrow inside it.
__device__ inline u32x2_t unpack8(uint32_t w, uint32_t z4) {
  const uint32_t lo = (w & 0x0f0f0f0fu) | 0x80808080u, hi = ((w >> 4) & 0x0f0f0f0fu) | 0x80808080u;
  return u32x2_t{(lo - z4) ^ 0x80808080u, (hi - z4) ^ 0x80808080u};
}

// The 8 codes less 8, times 16, as signed bytes: a code in the high half of its
// byte, the byte's sign turned. Less than half of unpack8's instructions.
__device__ inline u32x2_t unpack8_sixteenfold(uint32_t w) {
  return u32x2_t{((w << 4) & 0xf0f0f0f0u) ^ 0x80808080u, (w & 0xf0f0f0f0u) ^ 0x80808080u};
}

// The 8 codes less z as 16-bit numbers, all exact, at 2^-11 (bf16) or 2^-9
// (fp16, which has no normal numbers below 2^-14): zh is z at the same.
template <typename XT>
constexpr float LESS_HELD = __is_same(XT, bf16_tag) ? 0x1p-11f : 0x1p-9f;
template <typename XT>
__device__ inline v4u32 unpack16_less(uint32_t w, float zh) {
  const uint32_t lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;
  f32x2_t f[4];
  if constexpr (__is_same(XT, bf16_tag)) {
    f[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(lo, 0.25f, false);
    f[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(lo, 0.25f, true);
    f[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, 0.25f, false);
    f[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, 0.25f, true);
  } else {
    f[0] = __builtin_amdgcn_cvt_pk_f32_fp8((int)lo, false);
    f[1] = __builtin_amdgcn_cvt_pk_f32_fp8((int)lo, true);
    f[2] = __builtin_amdgcn_cvt_pk_f32_fp8((int)hi, false);
    f[3] = __builtin_amdgcn_cvt_pk_f32_fp8((int)hi, true);
  }
  v4u32 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = mfma_ops<XT>::pack(f[i][0] - zh, f[i][1] - zh);
  return v;
}

// First k of a lane's dword i within a step; q = lane / 16.
template <int G>
__device__ inline int dword_k(int i, int q) {
  return G == 32 ? 32 * i + 8 * q : 64 * (i >> 1) + 16 * q + 8 * (i & 1);
}

// ------------------------------------------------------------- the result
template <typename Tag>
__device__ inline float load_one(const char *p) {
  if constexpr (__is_same(Tag, f32_tag)) return *reinterpret_cast<const float *>(p);
  else if constexpr (__is_same(Tag, f16_tag)) return (float)*reinterpret_cast<const _Float16 *>(p);
  else return __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t *>(p) << 16);
}

template <typename Tag>
__device__ inline void finish_as(const Int4Params &p, int64_t row, int col, f32x4_t v) {
  constexpr int EB = __is_same(Tag, f32_tag) ? 4 : 2;
  char *y = p.y + row * p.y_st + (int64_t)EB * col;
  const char *r = p.res ? p.res + row * p.res_st + (int64_t)EB * col : nullptr;
  if (p.wide && col + 4 <= p.outs) {
    if constexpr (EB == 4) {
      if (r) v += *reinterpret_cast<const f32x4_t *>(r);
      *reinterpret_cast<f32x4_t *>(y) = v;
    } else {
      if (r) {
        const u32x2_t w = *reinterpret_cast<const u32x2_t *>(r);
        v += f32x4_t{mfma_ops<Tag>::lo(w[0]), mfma_ops<Tag>::hi(w[0]), mfma_ops<Tag>::lo(w[1]), mfma_ops<Tag>::hi(w[1])};
      }
      *reinterpret_cast<u32x2_t *>(y) = u32x2_t{mfma_ops<Tag>::pack(v[0], v[1]), mfma_ops<Tag>::pack(v[2], v[3])};
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (col + i >= p.outs) break;
    float x = v[i];
    if (r) x += load_one<Tag>(r + EB * i);
    if constexpr (EB == 4) *reinterpret_cast<float *>(y + EB * i) = x;
    else *reinterpret_cast<uint16_t *>(y + EB * i) = (uint16_t)mfma_ops<Tag>::pack(x, x);
  }
}

// Four columns of y from `col` on, of sums v, over rows of XT: y is of 16-bit
// rows' own type.
template <typename XT>
__device__ inline void finish(const Int4Params &p, int64_t row, int col, f32x4_t v) {
  if constexpr (!__is_same(XT, i8_tag)) finish_as<XT>(p, row, col, v);
  else if (p.dtype == IKL_BF16) finish_as<bf16_tag>(p, row, col, v);
  else if (p.dtype == IKL_F16) finish_as<f16_tag>(p, row, col, v);
  else finish_as<f32_tag>(p, row, col, v);
}

__device__ inline f32x4_t gate_up(f32x4_t gate, f32x4_t up) {
  f32x4_t v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = silu_fast(gate[i]) * up[i];
  return v;
}

// Columns of y that lane group q holds of a tile (of a pair's first tile
// where the weight is gated).
__device__ inline int tile_col(const Int4Params &p, int tile, int q) {
  return (p.gated ? tile >> 1 : tile) * 16 + 4 * q;
}

}  // namespace
}  // namespace ikl
