// The kernels of y = x W^T over 4-bit weights for one type of x: for few rows
// and for many. Compiled once for each type.
#pragma once

#include "int4_linear.h"

namespace ikl {
namespace {

// What the scales of W carry beside their values, 8-bit rows' in the few rows'
// kernel at the end.
template <typename XT, bool LESS, bool Z>
constexpr float scale_carries() {
  if constexpr (__is_same(XT, i8_tag)) return S_CARRIES<Z>;
  else return 1.f / (LESS ? LESS_HELD<XT> : codes_as<XT>::HELD);
}

// --------------------------------------------------------------- few rows
constexpr int ROW_WAVES = 8;

// What a wave loads of one step, all of it on its way at once.
template <typename XT, int G, int MT, int NT>
struct RowsStep {
  static constexpr bool I8 = __is_same(XT, i8_tag);
  static constexpr int GPS = 128 / G;
  static constexpr int XP = I8 ? 2 : 4;  // 16-byte pieces of a row
  v4u32 w[NT], x[MT][XP];
  f32x4_t sc[NT][GPS];
  uint32_t z[NT][GPS];  // 16-bit rows: of the lane's four columns, a byte each; 8-bit rows: of its row of W
  float sx[MT][I8 ? GPS : 1];
};

// A workgroup owns NT tiles of 16 columns and MT tiles of 16 rows; its waves
// split the contraction in steps of 128 and meet in LDS. Bound: the read of W
// once, and below some 8 MB of it the latency of that read: DEPTH steps are on
// their way in registers. 1 x 2048 to 2 x 5632 with SiLU * up 5.5 us, 32 x 4096
// to 14336 of 8-bit rows 11.7 (2.7 TB/s).
//
// 16-bit rows: z X of a group comes from a matrix product with a row operand
// of ones, which lands in the same lanes as P; the matrix cores have the time.
template <typename XT, int G, int MT, int NT, int DEPTH, bool Z>
__global__ __launch_bounds__(64 * ROW_WAVES) void int4_rows_kernel(const Int4Params p) {
  using Step = RowsStep<XT, G, MT, NT>;
  constexpr bool I8 = Step::I8;
  constexpr int GPS = Step::GPS, DPG = 4 / GPS;  // groups a step, dwords a group
  __shared__ __attribute__((aligned(16))) float red[ROW_WAVES][NT * MT][64][4];
  const int tid = threadIdx.x, lane = tid & 63, hl = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const unsigned across = (unsigned)(p.tiles + NT - 1) / NT, down = blockIdx.x / across;
  const int tile0 = (int)(blockIdx.x - down * across) * NT;
  const int64_t row0 = (int64_t)down * (16 * MT);
  const char *xrow[MT];
  const float *xs[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {  // rows past the last read it again and are not stored
    int64_t r = row0 + 16 * m + hl;
    r = r < p.rows ? r : p.rows - 1;
    xrow[m] = p.x + r * p.x_st;
    xs[m] = p.xs + (I8 ? r * p.groups : 0);
  }
  int64_t tile[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) tile[n] = tile0 + n < p.tiles ? tile0 + n : p.tiles - 1;
  f32x4_t acc[NT][MT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[n][m] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  auto load = [&](int s, Step &t) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      t.w[n] = load16v_global(p.codes + (tile[n] * p.steps + s) * 1024 + (uint32_t)(16 * lane));
#pragma unroll
      for (int g = 0; g < GPS; ++g) {
        const int64_t at = (tile[n] * p.steps * GPS + s * GPS + g) * 16;
        t.sc[n][g] = *reinterpret_cast<const f32x4_t *>(p.scales + at + (uint32_t)(4 * q));
        if constexpr (Z) {
          if constexpr (I8) t.z[n][g] = p.zeros[at + (uint32_t)hl];
          else t.z[n][g] = *reinterpret_cast<const uint32_t *>(p.zeros + at + (uint32_t)(4 * q));
        }
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int g = 0; g < GPS; ++g) {
        // past the contraction: the row's start, for groups that are skipped
        const int step = s * GPS + g < p.groups ? s : 0, u = s * GPS + g < p.groups ? g : 0;
        if constexpr (!I8) {
#pragma unroll
          for (int i = 0; i < DPG; ++i)
            t.x[m][g * DPG + i] = load16v_global(xrow[m] + 2 * ((int64_t)step * 128 + dword_k<G>(u * DPG + i, q)));
        } else if constexpr (G >= 64) {
#pragma unroll
          for (int i = 0; i < DPG / 2; ++i)
            t.x[m][g * DPG / 2 + i] = load16v_global(xrow[m] + (int64_t)step * 128 + dword_k<G>(u * DPG + 2 * i, q));
        } else {
          const u32x2_t h = *reinterpret_cast<const u32x2_t *>(xrow[m] + (int64_t)step * 128 + dword_k<G>(u, q));
          t.x[m][g / 2][2 * (g & 1)] = h[0];
          t.x[m][g / 2][2 * (g & 1) + 1] = h[1];
        }
        if constexpr (I8) t.sx[m][g] = xs[m][step * GPS + u];
      }
    }
  };
  auto compute = [&](int s, const Step &t) {
#pragma unroll
    for (int g = 0; g < GPS; ++g) {
      if (GPS > 1 && s * GPS + g >= p.groups) continue;  // the contraction ends inside the step
      if constexpr (!I8) {
        const v4u32 ones = {codes_as<XT>::ONES, codes_as<XT>::ONES, codes_as<XT>::ONES, codes_as<XT>::ONES};
        f32x4_t X[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          X[m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < DPG; ++i) X[m] = mfma_ops<XT>::mma_k32(ones, t.x[m][g * DPG + i], X[m]);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          v4u32 a[DPG];
#pragma unroll
          for (int i = 0; i < DPG; ++i) a[i] = unpack16<XT>(t.w[n][g * DPG + i]);
          const f32x4_t sc = t.sc[n][g] * scale_carries<XT, false, Z>();
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            f32x4_t P = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < DPG; ++i) P = mfma_ops<XT>::mma_k32(a[i], t.x[m][g * DPG + i], P);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float z = Z ? (float)((t.z[n][g] >> (8 * i)) & 0xffu) : 8.f;
              acc[n][m][i] = fmaf(sc[i], fmaf(-z, X[m][i], P[i]), acc[n][m][i]);
            }
          }
        }
      } else {
        f32x2_t sx[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) sx[m] = row_scale(t.sx[m][g]);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          u32x2_t a[DPG];
#pragma unroll
          for (int i = 0; i < DPG; ++i)
            a[i] = Z ? unpack8(t.w[n][g * DPG + i], t.z[n][g] * 0x01010101u) : unpack8_sixteenfold(t.w[n][g * DPG + i]);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            i32x4_t P = {MAGIC, MAGIC, MAGIC, MAGIC};
            if constexpr (G >= 64) {
#pragma unroll
              for (int i = 0; i < DPG / 2; ++i)
                P = __builtin_amdgcn_mfma_i32_16x16x64_i8(
                    i32x4_t{(int)a[2 * i][0], (int)a[2 * i][1], (int)a[2 * i + 1][0], (int)a[2 * i + 1][1]},
                    __builtin_bit_cast(i32x4_t, t.x[m][g * DPG / 2 + i]), P, 0, 0, 0);
            } else {
              const v4u32 x = t.x[m][g / 2];
              P = __builtin_amdgcn_mfma_i32_16x16x32_i8(
                  __builtin_bit_cast(long, a[0]), __builtin_bit_cast(long, u32x2_t{x[2 * (g & 1)], x[2 * (g & 1) + 1]}), P, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
              acc[n][m][i] = fmaf(t.sc[n][g][i], fmaf(__int_as_float(P[i]), sx[m][0], sx[m][1]), acc[n][m][i]);
          }
        }
      }
    }
  };

  Step steps[DEPTH];
#pragma unroll
  for (int j = 0; j < DEPTH; ++j) {
    const int s = wave + ROW_WAVES * j;
    if (s < p.steps) load(s, steps[j]);
  }
  for (int base = wave; base < p.steps; base += ROW_WAVES * DEPTH) {
#pragma unroll
    for (int j = 0; j < DEPTH; ++j) {
      const int s = base + ROW_WAVES * j, next = s + ROW_WAVES * DEPTH;
      if (s < p.steps) compute(s, steps[j]);
      if (next < p.steps) load(next, steps[j]);
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m)
      *reinterpret_cast<f32x4_t *>(red[wave][n * MT + m][lane]) = I8 ? acc[n][m] * scale_carries<XT, false, Z>() : acc[n][m];
  __syncthreads();
  // lane l of an accumulator: columns 4 (l / 16) + i, row l % 16
  const int per = p.gated ? 2 : 1;
  for (int u = tid; u < NT * MT * 64 / per; u += 64 * ROW_WAVES) {
    // four threads of a row side by side, tile by tile
    const int c = u % (4 * NT / per), r = u / (4 * NT / per), n = c / 4 * per, m = r / 16, l = 16 * (c & 3) + r % 16;
    f32x4_t v[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      v[k] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      if (k >= per) continue;
#pragma unroll
      for (int h = 0; h < ROW_WAVES; ++h) v[k] += *reinterpret_cast<const f32x4_t *>(red[h][(n + k) * MT + m][l]);
    }
    const int64_t row = row0 + r;
    if (row >= p.rows || tile0 + n >= p.tiles) continue;
    const int col = tile_col(p, tile0 + n, c & 3);
    if (col < p.outs) finish<XT>(p, row, col, p.gated ? gate_up(v[0], v[1]) : v[0]);
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
// 16-bit rows: codes less their zero points, exact, by way of fp32, or (up to
// 64 rows a workgroup, where that costs more than it saves) the codes and X as
// in the few rows' kernel.
//
// Bound: the issue of vector instructions (a matrix instruction takes a slot
// too): of a wave's step of 128 8-bit rows by 64 columns 256 multiply-adds of
// the scales and 64 matrix instructions are 320 of 429 slots. 8192 x 4096 to
// 14336: 8-bit rows 567-608 us (1.6-1.7 POP/s; a library's int8 product 2.0 at
// 8192^3), bf16 rows 930 us (1.03 PFLOP/s; 10 registers spill, with zero points 15).
constexpr int VMCNT_0 = 0x0f70;  // s_waitcnt of vmcnt alone: its bits are 0-3 and 14-15
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

template <typename XT, int G, int MT, int WT, int NST, bool Z>
__global__ __launch_bounds__(256, WT > 2 ? 2 : 3) void int4_tiles_kernel(const Int4Params p, const int split) {
  constexpr bool I8 = __is_same(XT, i8_tag);
  constexpr int GPS = 128 / G, DPG = 4 / GPS;
  constexpr int BM = 16 * MT;
  constexpr int RB = I8 ? 128 : 256, RC = RB / 16;  // bytes and 16-byte chunks of a row's step
  constexpr int LOADS = BM * RC / 256;
  static_assert(LOADS >= 1, "every wave loads");
  // what s carries beside the column's scale
  constexpr bool LESS = !I8 && MT > 4;  // codes less their zero points
  constexpr float SCALE = scale_carries<XT, LESS, Z>();
  // At most 80 KB, for two workgroups on a CU: the rows' steps (at the end each
  // wave's accumulators of a row tile), a of the rows and less MAGIC times it
  // (groups of 32: a alone), the columns' scales and zero points, the codes.
  constexpr int TAIL = 4 * 16 * 16 * WT * 4;
  using scale_t = typename pick<(G >= 64), f32x2_t, float>::type;
  __shared__ __attribute__((aligned(16))) char mem[NST * BM * RB > TAIL ? NST * BM * RB : TAIL];
  __shared__ __attribute__((aligned(16))) scale_t xsc[2][I8 ? BM * GPS : 4];
  __shared__ __attribute__((aligned(16))) float wsc[2][4][GPS][16 * WT];
  __shared__ __attribute__((aligned(4))) uint8_t wz[2][Z ? 4 * GPS * 16 * WT : 1];
  __shared__ __attribute__((aligned(16))) char codes[NST][I8 ? 4 * WT * 1024 : 16];
  const int tid = threadIdx.x, lane = tid & 63, hl = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const unsigned across = (unsigned)(p.tiles + 4 * WT - 1) / (4 * WT), down = blockIdx.x / across;
  const int tile0 = ((int)(blockIdx.x - down * across) * 4 + wave) * WT;
  const int64_t row0 = (int64_t)down * BM;
  const int chunks = p.groups * (G * (I8 ? 1 : 2) / 16);  // of a row
  const int s0 = split > 1 ? (int)((int64_t)blockIdx.y * p.steps / split) : 0;
  const int s1 = split > 1 ? (int)((int64_t)(blockIdx.y + 1) * p.steps / split) : p.steps;

  // This thread's chunk of its first row; its others are 256 / RC rows apart.
  // Rows past the last: the last again.
  const int r0 = tid / RC, chunk = (tid % RC) ^ (r0 & 7);
  const int left = (int)(p.rows - 1 - row0 < BM ? p.rows - 1 - row0 : BM);  // rows behind the block's first
  const char *const xblock = p.x + row0 * p.x_st;
  // rows less than 16 MB apart (8-bit ones are): a block's offsets have 31 bits
  const bool near = I8 || (uint64_t)p.x_st < 1u << 24;
  auto rows_to_lds = [&](int s, int b) {
    // past the contraction: the row's last chunk, for groups that are skipped
    int over = 0;
    if (GPS > 1 && (s + 1) * RC > chunks) {
      over = s * RC + chunk - (chunks - 1);
      over = 16 * (over > 0 ? over : 0);
    }
    const char *from = xblock + (int64_t)s * RB;
    // The rows' offsets are computed anew each step: kept, they take registers
    // that the accumulators need.
    int r = r0;
    asm volatile("" : "+v"(r));
    auto load = [&](int u, const char *at) {
      __builtin_amdgcn_global_load_lds((global_ptr)at, (lds_ptr)(mem + b * (BM * RB) + 4096 * u + 1024 * wave), 16, 0, 0);
    };
    if (near) {
#pragma unroll
      for (int u = 0; u < LOADS; ++u) {
        const int row = r + u * (256 / RC) < left ? r + u * (256 / RC) : left;
        load(u, from + (uint32_t)(__umul24((uint32_t)row, (uint32_t)p.x_st) + 16u * chunk - over));
      }
    } else {
#pragma unroll
      for (int u = 0; u < LOADS; ++u) {
        const int row = r + u * (256 / RC) < left ? r + u * (256 / RC) : left;
        load(u, from + ((int64_t)row * p.x_st + (16 * chunk - over)));
      }
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
        const f32x2_t a = row_scale(held_x[g]);  // by every thread of the row, the same
        if constexpr (G >= 64) xsc[b][g * BM + tid % BM] = a;
        else xsc[b][g * BM + tid % BM] = a[0];
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
  // A step's rows and codes are NST - 1 steps on their way, its scales one. The
  // scales' loads of a step are issued before the rows' of a later one, and
  // loads return in order: who has the first waits for no more.
  constexpr int FLIGHT = LOADS + (I8 ? WT : 0);  // a step's loads to LDS
  auto ahead = [&](int s, int b) {
    rows_to_lds(s, b);
    if constexpr (I8) codes_ahead(s, b);
  };
#pragma unroll
  for (int j = 0; j < NST - 1; ++j) ahead(s0 + j < s1 ? s0 + j : s1 - 1, j);
  if constexpr (!I8) codes_ahead(s0, 0);
  fetch(s0);
  put(0);
  // A barrier waits for LDS, not for loads that write it: their waits are here.
  __builtin_amdgcn_s_waitcnt(VMCNT_0);
  __syncthreads();
  int b = 0;  // s's buffer of rows and codes
  for (int s = s0; s < s1; ++s) {
    const int sb = (s - s0) & 1, last = b == 0 ? NST - 1 : b - 1;
    const int next = s + 1 < s1 ? s + 1 : s;
    // past the last step: the last again, so that every step asks for as much
    const int later = s + NST - 1 < s1 ? s + NST - 1 : s1 - 1;
    fetch(next);
    asm volatile("" ::: "memory");
    // buffer `last` was last read before the barrier that ended step s - 1
    if (I8) ahead(later, last);
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
        if constexpr (Z && (I8 || LESS)) {  // of this lane's row of W
          z = wz[sb][(wave * GPS + g) * 16 * WT + 16 * n + hl];
          z = I8 ? z * 0x01010101u : __float_as_uint((float)z * LESS_HELD<XT>);
        }
#pragma unroll
        for (int i = 0; i < DPG; ++i) {
          const uint32_t d = w[n][g * DPG + i];
          if constexpr (I8) {
            const u32x2_t v = Z ? unpack8(d, z) : unpack8_sixteenfold(d);
            a[n][i / 2][2 * (i & 1)] = v[0];
            a[n][i / 2][2 * (i & 1) + 1] = v[1];
          } else {
            a[n][i] = LESS ? unpack16_less<XT>(d, Z ? __uint_as_float(z) : 8.f * LESS_HELD<XT>) : unpack16<XT>(d);
          }
        }
      }
      if (!I8 && g == GPS - 1) {  // (a step that ends early is the last)
        codes_ahead(next, 0);
        asm volatile("" ::: "memory");
        ahead(later, last);
      }
      f32x4_t sc[WT];
#pragma unroll
      for (int n = 0; n < WT; ++n) sc[n] = *reinterpret_cast<const f32x4_t *>(&wsc[sb][wave][g][16 * n + 4 * q]);
      float zc[WT][4];  // zero points of the lane's columns
      if constexpr (!I8 && !LESS) {
#pragma unroll
        for (int n = 0; n < WT; ++n) {
          uint32_t z4 = 0;
          if constexpr (Z) z4 = *reinterpret_cast<const uint32_t *>(&wz[sb][(wave * GPS + g) * 16 * WT + 16 * n + 4 * q]);
#pragma unroll
          for (int i = 0; i < 4; ++i) zc[n][i] = Z ? (float)((z4 >> (8 * i)) & 0xffu) : 8.f;
        }
      }
      const char *xrow = mem + b * (BM * RB) + hl * RB;
      if constexpr (!I8) {
        // The next tile's rows are read ahead where the registers hold them.
        constexpr bool AHEAD = MT <= 4;
        v4u32 ahead[DPG];
        auto read = [&](int m) {
#pragma unroll
          for (int i = 0; i < DPG; ++i)
            ahead[i] = *reinterpret_cast<const v4u32 *>(xrow + 16 * m * RB + 16 * ((dword_k<G>(g * DPG + i, q) / 8) ^ (hl & 7)));
        };
        if (AHEAD) read(0);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          if (!AHEAD) read(m);
          v4u32 xv[DPG];
#pragma unroll
          for (int i = 0; i < DPG; ++i) xv[i] = ahead[i];
          if (AHEAD && m + 1 < MT) read(m + 1);
          f32x4_t X = {0.f, 0.f, 0.f, 0.f};
          if constexpr (!LESS) {
            const v4u32 ones = {codes_as<XT>::ONES, codes_as<XT>::ONES, codes_as<XT>::ONES, codes_as<XT>::ONES};
#pragma unroll
            for (int i = 0; i < DPG; ++i) X = mfma_ops<XT>::mma_k32(ones, xv[i], X);
          }
#pragma unroll
          for (int n = 0; n < WT; ++n) {
            f32x4_t P = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < DPG; ++i) P = mfma_ops<XT>::mma_k32(a[n][i], xv[i], P);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if constexpr (!LESS) P[i] = fmaf(-zc[n][i], X[i], P[i]);
              acc[n][m][i] = fmaf(sc[n][i], P[i], acc[n][m][i]);
            }
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
          sx[m % 3] = with_offset(xsc[sb][g * BM + 16 * m + hl]);
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
    put(sb ^ 1);
    // step s + 1's rows and codes are there when no more is on its way than
    // what was asked for after them
    constexpr int LATER = (NST - 2) * FLIGHT;
    __builtin_amdgcn_s_waitcnt(VMCNT_0 | (LATER & 15) | (LATER >> 4) << 14);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    b = b + 1 == NST ? 0 : b + 1;
  }
  if constexpr (NST > 2) {  // the last step's loads write where the tail does
    __builtin_amdgcn_s_waitcnt(VMCNT_0);
    __syncthreads();
  }
  // Through LDS, so that a row's columns leave side by side
  float *mine = reinterpret_cast<float *>(mem) + wave * 16 * 16 * WT;
  constexpr int CHUNKS = 4 * WT;  // of four columns, exchanged by row as the rows' are
  const int tiles = p.tiles - tile0;  // that this wave has
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int n = 0; n < WT; ++n)
      *reinterpret_cast<f32x4_t *>(mine + hl * 16 * WT + 4 * ((4 * n + q) ^ (hl % CHUNKS))) = acc[n][m];
    wave_lds_sync();
    const bool paired = p.gated && !p.part;
    const int units = paired ? WT / 2 : WT, shift = (WT == 4 ? 4 : 3) - paired;  // results of 16 columns; 4 units = 1 << shift
#pragma unroll
    for (int k = 0; k < WT; ++k) {  // 64 lanes: 4 WT / 4 of the tile's quads of columns
      if (k >= units) break;
      const int i = lane + 64 * k, r = i >> shift, c = i & ((1 << shift) - 1), n = (c >> 2) * (WT / units);
      const int64_t row = row0 + 16 * m + r;
      if (row >= p.rows || n >= tiles) continue;
      const float *at = mine + r * 16 * WT;
      const f32x4_t v = *reinterpret_cast<const f32x4_t *>(at + 4 * ((4 * n + (c & 3)) ^ (r % CHUNKS)));
      if (p.part) {
        float *to = p.part + ((int64_t)blockIdx.y * p.rows + row) * 16 * p.tiles + 16 * (tile0 + n) + 4 * (c & 3);
        *reinterpret_cast<f32x4_t *>(to) = v;
        continue;
      }
      const int col = tile_col(p, tile0 + n, c & 3);
      if (col < p.outs)
        finish<XT>(p, row, col, p.gated ? gate_up(v, *reinterpret_cast<const f32x4_t *>(at + 4 * ((4 * n + 4 + (c & 3)) ^ (r % CHUNKS)))) : v);
    }
    wave_lds_sync();
  }
}

template <typename XT, int G, bool Z>
void launch_tiles(const Int4Params &p, const Int4Plan &plan, dim3 grid, hipStream_t s) {
  constexpr int STAGES = __is_same(XT, i8_tag) && G == 32 ? 2 : 3;
  if (plan.mt == 2 && plan.nt == 8) int4_tiles_kernel<XT, G, 2, 2, 3, Z><<<grid, 256, 0, s>>>(p, plan.split);
  else if (plan.mt == 4 && plan.nt == 8) int4_tiles_kernel<XT, G, 4, 2, 3, Z><<<grid, 256, 0, s>>>(p, plan.split);
  else if (plan.mt == 4) int4_tiles_kernel<XT, G, 4, 4, STAGES, Z><<<grid, 256, 0, s>>>(p, plan.split);
  else int4_tiles_kernel<XT, G, 8, 4, 2, Z><<<grid, 256, 0, s>>>(p, plan.split);
}

template <typename XT, int G, bool Z>
void launch_rows(const Int4Params &p, const Int4Plan &plan, dim3 grid, hipStream_t s) {
  constexpr int WIDE = G == 32 ? 1 : 2;  // groups of 32: their scales take the registers
  const dim3 wg(64 * ROW_WAVES);
  if (plan.mt == 1 && plan.nt == 1) int4_rows_kernel<XT, G, 1, 1, 4, Z><<<grid, wg, 0, s>>>(p);
  else if (plan.mt == 1 && plan.nt == 2) int4_rows_kernel<XT, G, 1, 2, 3, Z><<<grid, wg, 0, s>>>(p);
  else if (plan.mt == 1) int4_rows_kernel<XT, G, 1, 4, WIDE, Z><<<grid, wg, 0, s>>>(p);
  else int4_rows_kernel<XT, G, 2, 4, __is_same(XT, i8_tag) ? WIDE : 1, Z><<<grid, wg, 0, s>>>(p);
}

template <typename XT, int G, bool Z>
void launch(const Int4Params &p, const Int4Plan &plan, hipStream_t s) {
  const dim3 grid((unsigned)(plan.blocks), (unsigned)plan.split);
  if (plan.few) launch_rows<XT, G, Z>(p, plan, grid, s);
  else launch_tiles<XT, G, Z>(p, plan, grid, s);
}

template <typename XT, int G>
void launch(const Int4Params &p, const Int4Plan &plan, hipStream_t s) {
  p.zeros ? launch<XT, G, true>(p, plan, s) : launch<XT, G, false>(p, plan, s);
}

template <typename XT>
void launch_group(const Int4Params &p, int group, const Int4Plan &plan, hipStream_t s) {
  if (group == 128) launch<XT, 128>(p, plan, s);
  else if (group == 64) launch<XT, 64>(p, plan, s);
  else launch<XT, 32>(p, plan, s);
}

}  // namespace
}  // namespace ikl
