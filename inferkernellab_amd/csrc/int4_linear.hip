// y = x W^T over 4-bit weights with a scale (and a zero point) for each output
// column and group of the contraction, for rows in 16 or in 8 bits.
#include "int4_linear.h"

namespace ikl {
namespace {

// --------------------------------------------------------------- few rows
constexpr int ROW_WAVES = 8;

// A workgroup owns NT tiles of 16 columns and MT tiles of 16 rows; its waves
// split the contraction in steps of 128 and meet in LDS.
template <typename XT, int G, int MT, int NT>
__global__ __launch_bounds__(64 * ROW_WAVES) void int4_rows_kernel(const Int4Params p) {
  constexpr bool I8 = __is_same(XT, i8_tag);
  constexpr int GPS = 128 / G, DPG = 4 / GPS;  // groups a step, dwords a group
  __shared__ __attribute__((aligned(16))) float red[ROW_WAVES][NT * MT][64][4];
  const int tid = threadIdx.x, lane = tid & 63, hl = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tile0 = blockIdx.x * NT;
  const int64_t row0 = (int64_t)blockIdx.y * (16 * MT);
  const char *xrow[MT];
  const float *xs[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {  // rows past the last read it again and are not stored
    int64_t r = row0 + 16 * m + hl;
    r = r < p.rows ? r : p.rows - 1;
    xrow[m] = p.x + r * p.x_st;
    xs[m] = p.xs + (I8 ? r * p.groups : 0);
  }
  f32x4_t acc[NT][MT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[n][m] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  for (int s = wave; s < p.steps; s += ROW_WAVES) {
    v4u32 w[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int t = tile0 + n < p.tiles ? tile0 + n : p.tiles - 1;
      w[n] = load16v_global(p.codes + (((int64_t)t * p.steps + s) * 64 + lane) * 16);
    }
#pragma unroll
    for (int g = 0; g < GPS; ++g) {
      const int gk = s * GPS + g;
      if (gk >= p.groups) continue;  // the contraction ends inside the step
      v4u32 xv[MT][DPG];
      float sx[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if constexpr (!I8) {
#pragma unroll
          for (int i = 0; i < DPG; ++i)
            xv[m][i] = load16v_global(xrow[m] + 2 * ((int64_t)s * 128 + dword_k<G>(g * DPG + i, q)));
        } else if constexpr (G >= 64) {
#pragma unroll
          for (int i = 0; i < DPG / 2; ++i)
            xv[m][i] = load16v_global(xrow[m] + (int64_t)s * 128 + dword_k<G>(g * DPG + 2 * i, q));
          sx[m] = xs[m][gk];
        } else {
          const u32x2_t h = *reinterpret_cast<const u32x2_t *>(xrow[m] + (int64_t)s * 128 + dword_k<G>(g, q));
          xv[m][0] = v4u32{h[0], h[1], 0u, 0u};
          sx[m] = xs[m][gk];
        }
      }
      f32x4_t X[MT];
      if constexpr (!I8) {
        const v4u32 ones = {mfma_ops<XT>::ONE2, mfma_ops<XT>::ONE2, mfma_ops<XT>::ONE2, mfma_ops<XT>::ONE2};
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          X[m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < DPG; ++i) X[m] = mfma_ops<XT>::mma_k32(ones, xv[m][i], X[m]);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int t = tile0 + n < p.tiles ? tile0 + n : p.tiles - 1;
        const int64_t at = ((int64_t)t * p.steps * GPS + gk) * 16;
        const f32x4_t sc = *reinterpret_cast<const f32x4_t *>(p.scales + at + 4 * q);
        if constexpr (!I8) {
          f32x4_t z = {8.f, 8.f, 8.f, 8.f};
          if (p.zeros) {
            const uint32_t zw = *reinterpret_cast<const uint32_t *>(p.zeros + at + 4 * q);
#pragma unroll
            for (int i = 0; i < 4; ++i) z[i] = (float)((zw >> (8 * i)) & 0xffu);
          }
          v4u32 a[DPG];
#pragma unroll
          for (int i = 0; i < DPG; ++i) a[i] = unpack16<XT>(w[n][g * DPG + i]);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            f32x4_t P = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < DPG; ++i) P = mfma_ops<XT>::mma_k32(a[i], xv[m][i], P);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[n][m][i] = fmaf(sc[i], fmaf(-z[i], X[m][i], P[i]), acc[n][m][i]);
          }
        } else {
          const uint32_t z4 = (p.zeros ? (uint32_t)p.zeros[at + hl] : 8u) * 0x01010101u;
          u32x2_t a[DPG];
#pragma unroll
          for (int i = 0; i < DPG; ++i) a[i] = unpack8(w[n][g * DPG + i], z4);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            i32x4_t P = {0, 0, 0, 0};
            if constexpr (G >= 64) {
#pragma unroll
              for (int i = 0; i < DPG / 2; ++i)
                P = __builtin_amdgcn_mfma_i32_16x16x64_i8(
                    i32x4_t{(int)a[2 * i][0], (int)a[2 * i][1], (int)a[2 * i + 1][0], (int)a[2 * i + 1][1]},
                    __builtin_bit_cast(i32x4_t, xv[m][i]), P, 0, 0, 0);
            } else {
              P = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, a[0]),
                                                        __builtin_bit_cast(long, u32x2_t{xv[m][0][0], xv[m][0][1]}), P, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[n][m][i] = fmaf(sc[i] * sx[m], (float)P[i], acc[n][m][i]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) *reinterpret_cast<f32x4_t *>(red[wave][n * MT + m][lane]) = acc[n][m];
  __syncthreads();
  // lane l of an accumulator: columns 4 (l / 16) + i, row l % 16
  const int per = p.gated ? 2 : 1;
  for (int u = tid; u < NT * MT * 64 / per; u += 64 * ROW_WAVES) {
    const int l = u & 63, tm = u >> 6, n = tm / MT * per, m = tm % MT;
    f32x4_t v[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      v[k] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      if (k >= per) continue;
#pragma unroll
      for (int h = 0; h < ROW_WAVES; ++h) v[k] += *reinterpret_cast<const f32x4_t *>(red[h][(n + k) * MT + m][l]);
    }
    const int64_t row = row0 + 16 * m + (l & 15);
    const int col = tile_col(p, tile0 + n, l >> 4);
    if (row < p.rows && col < p.outs) finish(p, row, col, p.gated ? gate_up(v[0], v[1]) : v[0]);
  }
}

// --------------------------------------------------------------- many rows
constexpr int BM = 128, MTILES = BM / 16, WTILES = 4;  // rows of a workgroup; 16-column tiles of a wave

template <typename XT, int G>
__global__ __launch_bounds__(256) void int4_tiles_kernel(const Int4Params p) {
  constexpr bool I8 = __is_same(XT, i8_tag);
  constexpr int GPS = 128 / G, DPG = 4 / GPS;
  constexpr int RB = I8 ? 128 : 256, RC = RB / 16;  // bytes and 16-byte chunks of a row's step
  constexpr int LOADS = BM * RC / 256;
  __shared__ __attribute__((aligned(16))) char xt[2][BM * RB];
  __shared__ float xsc[2][I8 ? BM * GPS : 1];
  const int tid = threadIdx.x, lane = tid & 63, hl = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tile0 = (blockIdx.x * 4 + wave) * WTILES;
  const int64_t row0 = (int64_t)blockIdx.y * BM;
  const int row_bytes = p.groups * G * (I8 ? 1 : 2);

  v4u32 held[LOADS];
  float held_s[GPS];
  auto fetch = [&](int s) {
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int c = (tid + 256 * u) % RC, r = (tid + 256 * u) / RC;
      int64_t row = row0 + r;
      row = row < p.rows ? row : p.rows - 1;
      held[u] = zero4();
      if (s * RB + 16 * c < row_bytes) held[u] = load16v_global(p.x + row * p.x_st + (int64_t)s * RB + 16 * c);
    }
    if constexpr (I8) {
      int64_t row = row0 + (tid & (BM - 1));
      row = row < p.rows ? row : p.rows - 1;
#pragma unroll
      for (int g = 0; g < GPS; ++g) {
        held_s[g] = 0.f;
        if (s * GPS + g < p.groups) held_s[g] = p.xs[row * p.groups + s * GPS + g];
      }
    }
  };
  auto put = [&](int b) {
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int c = (tid + 256 * u) % RC, r = (tid + 256 * u) / RC;
      *reinterpret_cast<v4u32 *>(xt[b] + r * RB + 16 * (c ^ (r & 7))) = held[u];
    }
    if constexpr (I8) {
      if (tid < BM) {
#pragma unroll
        for (int g = 0; g < GPS; ++g) xsc[b][g * BM + tid] = held_s[g];
      }
    }
  };

  f32x4_t acc[WTILES][MTILES];
#pragma unroll
  for (int n = 0; n < WTILES; ++n)
#pragma unroll
    for (int m = 0; m < MTILES; ++m) acc[n][m] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  fetch(0);
  put(0);
  __syncthreads();
  for (int s = 0; s < p.steps; ++s) {
    const int b = s & 1;
    if (s + 1 < p.steps) fetch(s + 1);
    v4u32 w[WTILES];
#pragma unroll
    for (int n = 0; n < WTILES; ++n) {
      const int t = tile0 + n < p.tiles ? tile0 + n : p.tiles - 1;
      w[n] = load16v_global(p.codes + (((int64_t)t * p.steps + s) * 64 + lane) * 16);
    }
#pragma unroll
    for (int g = 0; g < GPS; ++g) {
      const int gk = s * GPS + g;
      if (gk >= p.groups) continue;
      f32x4_t sc[WTILES];
      v4u32 a[WTILES][DPG];  // I8: two dwords of a step's code dword in one
#pragma unroll
      for (int n = 0; n < WTILES; ++n) {
        const int t = tile0 + n < p.tiles ? tile0 + n : p.tiles - 1;
        const int64_t at = ((int64_t)t * p.steps * GPS + gk) * 16;
        sc[n] = *reinterpret_cast<const f32x4_t *>(p.scales + at + 4 * q);
        const uint32_t z = p.zeros ? (uint32_t)p.zeros[at + hl] : 8u;  // this lane's row of W
#pragma unroll
        for (int i = 0; i < DPG; ++i) {
          const u32x2_t d = unpack8(w[n][g * DPG + i], z * 0x01010101u);
          if constexpr (I8) {
            a[n][i] = v4u32{d[0], d[1], 0u, 0u};
          } else {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = (float)(int8_t)(d[e >> 2] >> (8 * (e & 3)));
            a[n][i] = v4u32{mfma_ops<XT>::pack(f[0], f[1]), mfma_ops<XT>::pack(f[2], f[3]), mfma_ops<XT>::pack(f[4], f[5]),
                            mfma_ops<XT>::pack(f[6], f[7])};
          }
        }
      }
#pragma unroll
      for (int m = 0; m < MTILES; ++m) {
        const int r = 16 * m + hl;
        const char *xr = xt[b] + r * RB;
        if constexpr (!I8) {
          v4u32 xv[DPG];
#pragma unroll
          for (int i = 0; i < DPG; ++i)
            xv[i] = *reinterpret_cast<const v4u32 *>(xr + 16 * ((dword_k<G>(g * DPG + i, q) / 8) ^ (r & 7)));
#pragma unroll
          for (int n = 0; n < WTILES; ++n) {
            f32x4_t P = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < DPG; ++i) P = mfma_ops<XT>::mma_k32(a[n][i], xv[i], P);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[n][m][i] = fmaf(sc[n][i], P[i], acc[n][m][i]);
          }
        } else {
          const float sx = xsc[b][g * BM + r];
          if constexpr (G >= 64) {
            v4u32 xv[DPG / 2];
#pragma unroll
            for (int i = 0; i < DPG / 2; ++i)
              xv[i] = *reinterpret_cast<const v4u32 *>(xr + 16 * ((dword_k<G>(g * DPG + 2 * i, q) / 16) ^ (r & 7)));
#pragma unroll
            for (int n = 0; n < WTILES; ++n) {
              i32x4_t P = {0, 0, 0, 0};
#pragma unroll
              for (int i = 0; i < DPG / 2; ++i)
                P = __builtin_amdgcn_mfma_i32_16x16x64_i8(
                    i32x4_t{(int)a[n][2 * i][0], (int)a[n][2 * i][1], (int)a[n][2 * i + 1][0], (int)a[n][2 * i + 1][1]},
                    __builtin_bit_cast(i32x4_t, xv[i]), P, 0, 0, 0);
#pragma unroll
              for (int i = 0; i < 4; ++i) acc[n][m][i] = fmaf(sc[n][i] * sx, (float)P[i], acc[n][m][i]);
            }
          } else {
            const int k = dword_k<G>(g, q);
            const u32x2_t xv = *reinterpret_cast<const u32x2_t *>(xr + 16 * ((k / 16) ^ (r & 7)) + (k & 8));
#pragma unroll
            for (int n = 0; n < WTILES; ++n) {
              i32x4_t P = {0, 0, 0, 0};
              P = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, u32x2_t{a[n][0][0], a[n][0][1]}),
                                                        __builtin_bit_cast(long, xv), P, 0, 0, 0);
#pragma unroll
              for (int i = 0; i < 4; ++i) acc[n][m][i] = fmaf(sc[n][i] * sx, (float)P[i], acc[n][m][i]);
            }
          }
        }
      }
    }
    // the other buffer was last read before the barrier that ended step s - 1
    if (s + 1 < p.steps) put(b ^ 1);
    __syncthreads();
  }
  const int per = p.gated ? 2 : 1;
#pragma unroll
  for (int n = 0; n < WTILES; ++n) {
    if (p.gated && (n & 1)) continue;
    if (tile0 + n >= p.tiles) continue;
    const int col = tile_col(p, tile0 + n, q);
    if (col >= p.outs) continue;
#pragma unroll
    for (int m = 0; m < MTILES; ++m) {
      const int64_t row = row0 + 16 * m + hl;
      if (row < p.rows) finish(p, row, col, per == 2 ? gate_up(acc[n][m], acc[n + 1 < WTILES ? n + 1 : n][m]) : acc[n][m]);
    }
  }
}

template <typename XT, int G>
void launch(const Int4Params &p, hipStream_t s) {
  if (p.rows <= 64) {
    const int tiles = p.gated ? p.tiles / 2 : p.tiles;
    const dim3 wg(64 * ROW_WAVES);
    const unsigned n = (unsigned)tiles;
    if (p.rows <= 16) {
      if (p.gated) int4_rows_kernel<XT, G, 1, 2><<<dim3(n), wg, 0, s>>>(p);
      else int4_rows_kernel<XT, G, 1, 1><<<dim3(n), wg, 0, s>>>(p);
    } else {
      const unsigned m = (unsigned)((p.rows + 31) / 32);
      if (p.gated) int4_rows_kernel<XT, G, 2, 2><<<dim3(n, m), wg, 0, s>>>(p);
      else int4_rows_kernel<XT, G, 2, 1><<<dim3(n, m), wg, 0, s>>>(p);
    }
    return;
  }
  const dim3 grid((unsigned)((p.tiles + 4 * WTILES - 1) / (4 * WTILES)), (unsigned)((p.rows + BM - 1) / BM));
  int4_tiles_kernel<XT, G><<<grid, 256, 0, s>>>(p);
}

template <typename XT>
void launch_group(const Int4Params &p, int group, hipStream_t s) {
  if (group == 128) launch<XT, 128>(p, s);
  else if (group == 64) launch<XT, 64>(p, s);
  else launch<XT, 32>(p, s);
}

bool off16(const void *ptr) { return ((uintptr_t)ptr & 15u) != 0; }

int check_args(const ikl_int4_linear_args *a) {
  if (!a) return fail(IKL_EINVAL, "int4 linear: args is NULL");
  if (a->rows < 0 || a->cols <= 0 || a->out_cols <= 0) return fail(IKL_EINVAL, "int4 linear: sizes must be positive");
  if (a->dtype != IKL_F16 && a->dtype != IKL_BF16 && a->dtype != IKL_F32)
    return fail(IKL_EINVAL, "int4 linear: unknown dtype");
  if (a->dtype == IKL_F32 && !a->x_scales) return fail(IKL_EUNSUPPORTED, "int4 linear: rows of fp16, bf16 or 8 bits only");
  if (a->group != 32 && a->group != 64 && a->group != 128)
    return fail(IKL_EUNSUPPORTED, "int4 linear: groups of 32, 64 or 128 only");
  if (a->cols % a->group != 0 || a->cols > (1 << 24) || a->out_cols > (1 << 24))
    return fail(IKL_EUNSUPPORTED, "int4 linear: cols must be whole groups; cols and out_cols at most 2^24");
  if (a->gated && a->residual) return fail(IKL_EUNSUPPORTED, "int4 linear: a gated weight takes no residual");
  if (a->rows > 128LL * 65535) return fail(IKL_EINVAL, "int4 linear: too many rows for a launch");
  return IKL_OK;
}

}  // namespace
}  // namespace ikl

using namespace ikl;

extern "C" int64_t ikl_int4_linear_workspace_size(const ikl_int4_linear_args *a) {
  if (const int bad = check_args(a)) return bad;
  return 0;
}

extern "C" int ikl_int4_linear(const ikl_int4_linear_args *a, void *stream) {
  if (const int bad = check_args(a)) return bad;
  if (a->rows == 0) return IKL_OK;
  const int64_t eb = a->dtype == IKL_F32 ? 4 : 2;
  if (!a->x || !a->codes || !a->scales || !a->y) return fail(IKL_EINVAL, "int4 linear: NULL tensor pointer");
  if (off16(a->x) || (!a->x_scales && a->rows > 1 && a->x_stride % 8 != 0) || ((uintptr_t)a->x_scales & 3u))
    return fail(IKL_EINVAL, "int4 linear: x rows must be 16-byte aligned");
  if (off16(a->codes) || off16(a->scales) || ((uintptr_t)a->zeros & 3u))
    return fail(IKL_EINVAL, "int4 linear: the weight must be 16-byte aligned");
  if (((uintptr_t)a->y | (uintptr_t)a->residual) & (uintptr_t)(eb - 1))
    return fail(IKL_EINVAL, "int4 linear: y and residual must be aligned to their elements");
  Int4Params p{};
  p.x = (const char *)a->x;
  p.x_st = a->rows > 1 ? (a->x_scales ? a->cols : a->x_stride * 2) : 0;
  p.xs = a->x_scales;
  p.codes = (const char *)a->codes;
  p.scales = a->scales;
  p.zeros = (const uint8_t *)a->zeros;
  p.res = (const char *)a->residual;
  p.res_st = a->rows > 1 ? a->residual_stride * eb : 0;
  p.y = (char *)a->y;
  p.y_st = a->rows > 1 ? a->y_stride * eb : 0;
  p.rows = a->rows;
  p.outs = (int32_t)a->out_cols;
  p.tiles = (int32_t)((a->out_cols + 15) / 16) * (a->gated ? 2 : 1);
  p.steps = (int32_t)((a->cols + 127) / 128);
  p.groups = (int32_t)(a->cols / a->group);
  p.gated = a->gated != 0;
  p.dtype = a->dtype;
  p.wide = (((uintptr_t)p.y | (uintptr_t)p.y_st | (uintptr_t)p.res | (p.res ? (uintptr_t)p.res_st : 0)) & (uintptr_t)(4 * eb - 1)) == 0;
  hipStream_t s = (hipStream_t)stream;
  if (a->x_scales) launch_group<i8_tag>(p, a->group, s);
  else if (a->dtype == IKL_BF16) launch_group<bf16_tag>(p, a->group, s);
  else launch_group<f16_tag>(p, a->group, s);
  return check_launch("int4 linear");
}
