// The kernels of y = x W^T over 4-bit weights for one type of x: for few rows
// and for many. Compiled once for each type.
#pragma once

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
// A workgroup owns MT tiles of 16 rows and 4 WT tiles of 16 columns, WT for
// each of its four waves. Rows go to LDS in steps of 128 of the contraction,
// by loads that write LDS themselves, one step ahead; 16-byte chunks are
// exchanged by row there (chunk ^ row % 8), so that the 16 rows of a matrix
// operand lie in different banks. Codes go from memory to the wave that
// unpacks them: no other wave reads them.
//
// 8-bit rows: each sum of a group leaves the matrix core as a whole number
// below 2^22 (of codes times 16 without zero points: below 2^21) on top of
// MAGIC, the bits of 1.5 * 2^23 as a float: the number as a float, without a
// conversion. What turns it into its share of y are two multiply-adds: first
// times a of its row less MAGIC times a, which is exact because a is held to
// 22 significant bits (less than 2^-21 of it lost, as in four fp32 operations),
// then times s of its column. a carries 2^-16 and s 2^16, so that
// MAGIC * a stays finite for rows up to 2^127.
constexpr int MAGIC = 0x4b400000;

typedef const __attribute__((address_space(1))) void *global_ptr;
typedef __attribute__((address_space(3))) void *lds_ptr;

template <bool FIRST, typename A, typename B>
struct pick {
  using type = A;
};
template <typename A, typename B>
struct pick<false, A, B> {
  using type = B;
};
__device__ inline f32x2_t with_offset(f32x2_t a) { return a; }
__device__ inline f32x2_t with_offset(float a) { return f32x2_t{a, a * -12582912.f}; }

template <typename XT, int G, int MT, int WT, bool Z>
__global__ __launch_bounds__(256, 2) void int4_tiles_kernel(const Int4Params p, const int split) {
  constexpr bool I8 = __is_same(XT, i8_tag);
  constexpr int GPS = 128 / G, DPG = 4 / GPS;
  constexpr int BM = 16 * MT;
  constexpr int RB = I8 ? 128 : 256, RC = RB / 16;  // bytes and 16-byte chunks of a row's step
  constexpr int LOADS = BM * RC / 256;
  static_assert(LOADS >= 1, "every wave loads");
  // what s carries beside the column's scale
  constexpr float SCALE = !I8 ? 512.f : Z ? 65536.f : 4096.f;
  // At most 80 KB, for two workgroups on a CU: the rows' two steps (at the end
  // each wave's accumulators of two row tiles), a of the rows and less MAGIC
  // times it (groups of 32: a alone), the columns' scales and zero points, the
  // codes.
  constexpr int TAIL = 4 * 32 * 16 * WT * 4;
  using scale_t = typename pick<(G >= 64), f32x2_t, float>::type;
  __shared__ __attribute__((aligned(16))) char mem[2 * BM * RB > TAIL ? 2 * BM * RB : TAIL];
  __shared__ __attribute__((aligned(16))) scale_t xsc[2][I8 ? BM * GPS : 4];
  __shared__ __attribute__((aligned(16))) float wsc[2][4][GPS][16 * WT];
  __shared__ uint8_t wz[2][Z ? 4 * GPS * 16 * WT : 1];
  __shared__ __attribute__((aligned(16))) char codes[2][I8 ? 4 * WT * 1024 : 16];
  const int tid = threadIdx.x, lane = tid & 63, hl = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tile0 = (blockIdx.x * 4 + wave) * WT;
  const int64_t row0 = (int64_t)blockIdx.y * BM;
  const int chunks = p.groups * (G * (I8 ? 1 : 2) / 16);  // of a row
  const int s0 = split > 1 ? (int)((int64_t)blockIdx.z * p.steps / split) : 0;
  const int s1 = split > 1 ? (int)((int64_t)(blockIdx.z + 1) * p.steps / split) : p.steps;

  // This thread's chunk of its first row; its others are 256 / RC rows apart.
  // Rows past the last: the last again.
  const int r0 = tid / RC, chunk = (tid % RC) ^ (r0 & 7);
  const int left = (int)(p.rows - 1 - row0 < BM ? p.rows - 1 - row0 : BM);  // rows behind the block's first
  // 8-bit rows are contiguous: a block's offsets have 31 bits
  const char *xthread = p.x + row0 * p.x_st;
  if constexpr (!I8) xthread += (int64_t)(r0 < left ? r0 : left) * p.x_st + 16 * chunk;
  auto rows_to_lds = [&](int s, int b) {
    // past the contraction: the row's last chunk, for groups that are skipped
    int over = 0;
    if (GPS > 1 && (s + 1) * RC > chunks) {
      over = s * RC + chunk - (chunks - 1);
      over = 16 * (over > 0 ? over : 0);
    }
    const char *from = xthread + (int64_t)s * RB;
    // The rows' offsets are computed anew each step: kept, they take registers
    // that the accumulators need.
    int r = r0;
    asm volatile("" : "+v"(r));
    const int most = left > r ? left - r : 0;
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const char *at;
      if constexpr (I8) {
        const int row = r + u * (256 / RC) < left ? r + u * (256 / RC) : left;
        at = from + (uint32_t)(__umul24((uint32_t)row, (uint32_t)p.x_st) + 16u * chunk - over);
      } else {
        const int64_t down = u * (256 / RC) < most ? u * (256 / RC) : most;
        at = from + down * p.x_st - over;
      }
      __builtin_amdgcn_global_load_lds((global_ptr)at, (lds_ptr)(mem + b * (BM * RB) + 4096 * u + 1024 * wave), 16, 0, 0);
    }
  };
  // Scales (and zero points) of a step: a lane each, on their way in registers
  const float *xs = I8 ? p.xs + row0 * p.groups : nullptr;
  const uint32_t xs_at = (uint32_t)(tid % BM < left ? tid % BM : left) * (uint32_t)p.groups;
  const int live = p.tiles - tile0 < 1 ? 1 : p.tiles - tile0;  // tiles that this wave has, or would read
  const int64_t first = p.tiles - tile0 < 1 ? p.tiles - 1 : tile0;
  const int64_t wbase = first * p.steps * GPS * 16;
  const uint32_t wat = (uint32_t)((lane / 16 < WT && lane / 16 < live ? lane / 16 : 0) * p.steps * GPS * 16 + hl);
  float held_x[GPS], held_w[GPS];
  uint32_t held_z[GPS];
  auto fetch = [&](int s) {
#pragma unroll
    for (int g = 0; g < GPS; ++g) {
      const int gk = s * GPS + g;
      if constexpr (I8) held_x[g] = (xs + (gk < p.groups ? gk : p.groups - 1))[xs_at];
      held_w[g] = (p.scales + wbase + (int64_t)gk * 16)[wat];
      if constexpr (Z) held_z[g] = (p.zeros + wbase + (int64_t)gk * 16)[wat];
    }
  };
  auto put = [&](int b) {
#pragma unroll
    for (int g = 0; g < GPS; ++g) {
      if constexpr (I8) {
        const float a = __uint_as_float(__float_as_uint(held_x[g]) & ~3u) * 0x1p-16f;
        if constexpr (G >= 64) xsc[b][g * BM + tid % BM] = f32x2_t{a, a * -12582912.f};
        else xsc[b][g * BM + tid % BM] = a;  // by every thread of the row, the same
      }
      if (lane < 16 * WT) {
        wsc[b][wave][g][lane] = held_w[g] * SCALE;
        if constexpr (Z) {
          wz[b][(wave * GPS + g) * 16 * WT + lane] = (uint8_t)held_z[g];
        }
      }
    }
  };
  // Codes: of 8-bit rows by way of LDS too, of 16-bit ones, whose rows fill
  // it, in registers.
  const char *code_at = p.codes + first * p.steps * 1024;
  v4u32 w[WT];
  auto codes_ahead = [&](int s, int b) {
#pragma unroll
    for (int n = 0; n < WT; ++n) {
      const char *from = code_at + ((int64_t)(n < live ? n : 0) * p.steps + s) * 1024 + (uint32_t)(16 * lane);
      if constexpr (I8)
        __builtin_amdgcn_global_load_lds((global_ptr)from, (lds_ptr)(codes[b] + 1024 * (WT * wave + n)), 16, 0, 0);
      else w[n] = load16v_global(from);
    }
  };

  f32x4_t acc[WT][MT];
#pragma unroll
  for (int n = 0; n < WT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[n][m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  rows_to_lds(s0, 0);
  codes_ahead(s0, 0);
  fetch(s0);
  put(0);
  __syncthreads();
  for (int s = s0; s < s1; ++s) {
    const int b = (s - s0) & 1;
    const int next = s + 1 < s1 ? s + 1 : s;
    // the other buffers were last read before the barrier that ended step s - 1
    if (s + 1 < s1) {
      rows_to_lds(s + 1, b ^ 1);
      if constexpr (I8) codes_ahead(s + 1, b ^ 1);
    }
    fetch(next);
    if constexpr (I8) {
#pragma unroll
      for (int n = 0; n < WT; ++n) w[n] = *reinterpret_cast<const v4u32 *>(codes[b] + 1024 * (WT * wave + n) + 16 * lane);
    }
#pragma unroll
    for (int g = 0; g < GPS; ++g) {
      if (GPS > 1 && s * GPS + g >= p.groups) continue;  // the contraction ends inside the step
      v4u32 a[WT][I8 ? (DPG + 1) / 2 : DPG];
#pragma unroll
      for (int n = 0; n < WT; ++n) {
        uint32_t z = 0;
        if constexpr (Z) {  // of this lane's row of W
          z = wz[b][(wave * GPS + g) * 16 * WT + 16 * n + hl];
          z = I8 ? z * 0x01010101u : __float_as_uint((float)z * 0x1p-9f);
        }
#pragma unroll
        for (int i = 0; i < DPG; ++i) {
          const uint32_t d = w[n][g * DPG + i];
          if constexpr (I8) {
            const u32x2_t v = Z ? unpack8(d, z) : unpack8_sixteenfold(d);
            a[n][i / 2][2 * (i & 1)] = v[0];
            a[n][i / 2][2 * (i & 1) + 1] = v[1];
          } else {
            a[n][i] = unpack16_less<XT>(d, Z ? __uint_as_float(z) : 8.f * 0x1p-9f);
          }
        }
      }
      if (!I8 && g == GPS - 1) codes_ahead(next, 0);
      f32x4_t sc[WT];
#pragma unroll
      for (int n = 0; n < WT; ++n) sc[n] = *reinterpret_cast<const f32x4_t *>(&wsc[b][wave][g][16 * n + 4 * q]);
      const char *xrow = mem + b * (BM * RB) + hl * RB;
      if constexpr (!I8) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          v4u32 xv[DPG];
#pragma unroll
          for (int i = 0; i < DPG; ++i)
            xv[i] = *reinterpret_cast<const v4u32 *>(xrow + 16 * m * RB + 16 * ((dword_k<G>(g * DPG + i, q) / 8) ^ (hl & 7)));
#pragma unroll
          for (int n = 0; n < WT; ++n) {
            f32x4_t P = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < DPG; ++i) P = mfma_ops<XT>::mma_k32(a[n][i], xv[i], P);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[n][m][i] = fmaf(sc[n][i], P[i], acc[n][m][i]);
          }
          __builtin_amdgcn_sched_barrier(0);  // or all tiles' rows are read at once, into registers that are not there
        }
      } else {
        // Tile m's sums are scaled while the matrix core works on m + 1, whose
        // rows were read an iteration before.
        constexpr int XV = (DPG + 1) / 2;
        v4u32 xv[XV];
        f32x2_t sx[3];  // a of the row, and less MAGIC times it
        i32x4_t P[2][WT];
        auto read = [&](int m) {
          sx[m % 3] = with_offset(xsc[b][g * BM + 16 * m + hl]);
          const char *xr = xrow + 16 * m * RB;
          if constexpr (G == 32) {
            const int k = dword_k<G>(g, q);
            const u32x2_t h = *reinterpret_cast<const u32x2_t *>(xr + 16 * ((k / 16) ^ (hl & 7)) + (k & 8));
            xv[0] = v4u32{h[0], h[1], 0u, 0u};
          } else {
#pragma unroll
            for (int i = 0; i < XV; ++i)
              xv[i] = *reinterpret_cast<const v4u32 *>(xr + 16 * ((dword_k<G>(g * DPG + 2 * i, q) / 16) ^ (hl & 7)));
          }
        };
        auto multiply = [&](int m, int n) {
          i32x4_t v = {MAGIC, MAGIC, MAGIC, MAGIC};
          if constexpr (G >= 64) {
#pragma unroll
            for (int i = 0; i < XV; ++i)
              v = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, a[n][i]),
                                                        __builtin_bit_cast(i32x4_t, xv[i]), v, 0, 0, 0);
          } else {
            v = __builtin_amdgcn_mfma_i32_16x16x32_i8(__builtin_bit_cast(long, u32x2_t{a[n][0][0], a[n][0][1]}),
                                                      __builtin_bit_cast(long, u32x2_t{xv[0][0], xv[0][1]}), v, 0, 0, 0);
          }
          P[m & 1][n] = v;
        };
        read(0);
#pragma unroll
        for (int n = 0; n < WT; ++n) multiply(0, n);
        if (MT > 1) read(1);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
          for (int n = 0; n < WT; ++n) {
            if (m + 1 < MT) multiply(m + 1, n);
            if (n == WT - 1 && m + 2 < MT) read(m + 2);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              acc[n][m][i] = fmaf(sc[n][i], fmaf(__int_as_float(P[m & 1][n][i]), sx[m % 3][0], sx[m % 3][1]), acc[n][m][i]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    put(b ^ 1);
    __syncthreads();
  }
  // Through LDS, so that a row's columns leave side by side
  float *mine = reinterpret_cast<float *>(mem) + wave * 32 * 16 * WT;
  constexpr int CHUNKS = 4 * WT;  // of four columns, exchanged by row as the rows' are
  const int tiles = p.tiles - tile0;  // that this wave has
#pragma unroll
  for (int m0 = 0; m0 < MT; m0 += 2) {
#pragma unroll
    for (int m = m0; m < m0 + 2 && m < MT; ++m)
#pragma unroll
      for (int n = 0; n < WT; ++n)
        *reinterpret_cast<f32x4_t *>(mine + (16 * (m - m0) + hl) * 16 * WT + 4 * ((4 * n + q) ^ (hl % CHUNKS))) = acc[n][m];
    wave_lds_sync();
    const int units = (p.gated && !p.part) ? WT / 2 : WT;  // results of 16 columns
#pragma unroll 1
    for (int i = lane; i < 32 * 4 * units; i += 64) {
      const int r = i / (4 * units), c = i % (4 * units), n = c / 4 * (WT / units);
      const int64_t row = row0 + 16 * m0 + r;
      if (row >= p.rows || n >= tiles || 16 * m0 + r >= BM) continue;
      const float *at = mine + r * 16 * WT;
      const f32x4_t v = *reinterpret_cast<const f32x4_t *>(at + 4 * ((4 * n + (c & 3)) ^ (r % CHUNKS)));
      if (p.part) {
        float *to = p.part + ((int64_t)blockIdx.z * p.rows + row) * 16 * p.tiles + 16 * (tile0 + n) + 4 * (c & 3);
        *reinterpret_cast<f32x4_t *>(to) = v;
        continue;
      }
      const int col = tile_col(p, tile0 + n, c & 3);
      if (col < p.outs) finish(p, row, col, p.gated ? gate_up(v, *reinterpret_cast<const f32x4_t *>(at + 4 * ((4 * n + 4 + (c & 3)) ^ (r % CHUNKS)))) : v);
    }
    wave_lds_sync();
  }
}

template <typename XT, int G, bool Z>
void launch_tiles(const Int4Params &p, const Int4Plan &plan, hipStream_t s) {
  const dim3 grid((unsigned)((p.tiles + 4 * plan.wt - 1) / (4 * plan.wt)),
                  (unsigned)((p.rows + 16 * plan.mt - 1) / (16 * plan.mt)), (unsigned)plan.split);
  if (plan.mt == 4) int4_tiles_kernel<XT, G, 4, 4, Z><<<grid, 256, 0, s>>>(p, plan.split);
  else int4_tiles_kernel<XT, G, 8, 4, Z><<<grid, 256, 0, s>>>(p, plan.split);
}

template <typename XT, int G>
void launch(const Int4Params &p, const Int4Plan &plan, hipStream_t s) {
  if (plan.mt == 0) {
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
  if (p.zeros) launch_tiles<XT, G, true>(p, plan, s);
  else launch_tiles<XT, G, false>(p, plan, s);
}

template <typename XT>
void launch_group(const Int4Params &p, int group, const Int4Plan &plan, hipStream_t s) {
  if (group == 128) launch<XT, 128>(p, plan, s);
  else if (group == 64) launch<XT, 64>(p, plan, s);
  else launch<XT, 32>(p, plan, s);
}

}  // namespace
}  // namespace ikl
