// y = x W^T over 4-bit weights with a scale (and a zero point) for each output
// column and group of the contraction, for rows in 16 or in 8 bits: arguments,
// how a launch is cut, and the join of a split contraction.
#include "int4_linear.h"

namespace ikl {
namespace {

// Sums of a split contraction's parts, in their order, and the epilogue: a
// thread four columns of a row, of any type.
__global__ __launch_bounds__(256) void int4_join_kernel(const Int4Params p, const int split, const int quads) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / quads;
  if (row >= p.rows) return;
  const int c = (int)(i - row * quads), per = p.gated ? 2 : 1, tile = c / 4 * per, q = c & 3;
  const float *part = p.part + row * 16 * p.tiles + 16 * tile + 4 * q;
  const int64_t step = p.rows * 16 * p.tiles;
  f32x4_t v = {0.f, 0.f, 0.f, 0.f}, u = v;
  for (int z = 0; z < split; ++z, part += step) {
    v += *reinterpret_cast<const f32x4_t *>(part);
    if (p.gated) u += *reinterpret_cast<const f32x4_t *>(part + 16);
  }
  const int col = tile_col(p, tile, q);
  if (col < p.outs) finish<i8_tag>(p, row, col, p.gated ? gate_up(v, u) : v);
}

int64_t blocks_of(int64_t rows, int tiles, int mt, int nt) {
  return ((rows + 16 * mt - 1) / (16 * mt)) * ((tiles + nt - 1) / nt);
}

// Few rows or few columns: one workgroup a CU where that covers y, of one row
// tile and the fewest column tiles that do, else of two row tiles. us of bf16
// rows, weights from memory, by 1 / 2 / 4 column tiles: 16 x 4096 x 4096 7.0 /
// 7.5 / 9.1; 2048 columns from 5632 7.9 / 9.1 / 10.8; 14336 from 4096 21 / 13 /
// 9.9. Against the many rows' kernel: 64 x 4096 x 4096 9.9 and 13.4; 128 x 4096 x
// 4096 by two row tiles 15.1 and 16.6. A CU's eight waves alone keep up with a
// split contraction to 112 steps (64 x 14336 x 4096 23.7 and 25.9, 64 x 28672 x
// 4096 46 and 37), two row tiles of 16-bit rows to 56 (100 x 8192 x 4096 24.3 and
// 22.5; 8-bit ones 19.2 and 21.0, at 28672 55 and 46).
bool few_rows(int64_t rows, int tiles, int steps, bool gated, bool eight, Int4Plan &plan) {
  auto take = [&](int mt, int nt, int64_t most) {
    const int64_t blocks = blocks_of(rows, tiles, mt, nt);
    plan = {true, mt, nt, 1, blocks};
    return blocks <= most;
  };
  if (rows <= 16 || steps <= 112)
    for (int nt = gated ? 2 : 1; nt <= 4; nt *= 2)
      if (take(1, nt, 256)) return true;
  if (rows <= 16) return true;
  if (steps > (eight || rows <= 32 ? 112 : 56)) return false;
  return take(2, 4, rows <= 32 ? INT64_MAX : 256);
}

// Many rows: the cheapest by an estimate of what bounds a launch. A CU runs
// `slots` workgroups of a form at once (as most of its kernels are compiled; {2, 8}
// is 3 of 16-bit rows in groups of 128 with zero points, and {2, 8} and {4, 8} are 3
// and 2 of 8-bit rows in groups of 32): a round of them takes `start`, and for
// each step the longer of one workgroup's own time and of their tiles' work. A
// split contraction saves steps and pays for a second launch and for the parts'
// way through memory. Times in us, fitted to launches of 17 to 4096 rows by 512
// to 28672 and 1024 to 14336 (groups of 128, zero points), of which each form and
// split was measured: what is taken was 0.6 (16-bit rows) and 0.9 % (8-bit)
// slower than the fastest in the mean, 38 % at most (40 x 1024 x 9000).
// No blocks: no form's fit in a grid.
Int4Plan plan_of(int64_t rows, int tiles, int steps, bool gated, bool eight) {
  Int4Plan best{};
  if (few_rows(rows, tiles, steps, gated, eight, best)) return best;
  best = {};
  struct Form {
    int mt, nt, slots;
    double alone[2], tile[2];  // of a step: 16-bit rows, 8-bit rows
  };
  static const Form forms[] = {{2, 8, 4, {0.9, 0.79}, {0.0242, 0.0157}},
                               {4, 8, 3, {1.4, 0.88}, {0.019, 0.0123}},
                               {4, 16, 2, {1.6, 1.1}, {0.0186, 0.012}},
                               {8, 16, 2, {3.3, 1.7}, {0.0181, 0.0099}}};
  const double start = eight ? 4 : 3.1, join = eight ? 5.1 : 3.3, bytes_a_us = eight ? 15e6 : 8.8e6;
  double least = 1e30;
  for (const Form &f : forms) {
    const int64_t blocks = blocks_of(rows, tiles, f.mt, f.nt);
    if (blocks > max_grid(256)) continue;
    auto step = [&](int n) {
      const double work = n * f.mt * f.nt * f.tile[eight];
      return n == 0 ? 0. : work > f.alone[eight] ? work : f.alone[eight];
    };
    const int most = rows * tiles < 1 << 28 ? 16 : 1;  // the join's launch holds that many
    for (int split = 1; split <= most && (split == 1 || 2 * split <= steps); ++split) {
      const int64_t per_cu = (blocks * split + 255) / 256, full = per_cu / f.slots;
      const int rest = (int)(per_cu % f.slots);
      double us = (full * step(f.slots) + step(rest)) * ((steps + split - 1) / split) + (full + (rest > 0)) * start;
      if (split > 1) us += join + split * (double)rows * tiles * 16 * 8 / bytes_a_us;
      if (us < least) least = us, best = {false, f.mt, f.nt, split, blocks};
    }
  }
  return best;
}

int tiles_of(const ikl_int4_linear_args *a) { return (int)((a->out_cols + 15) / 16) * (a->gated ? 2 : 1); }
int steps_of(const ikl_int4_linear_args *a) { return (int)((a->cols + 127) / 128); }

// Bytes of the parts of a split contraction.
int64_t part_bytes(const ikl_int4_linear_args *a, const Int4Plan &plan) {
  return plan.split > 1 ? (int64_t)plan.split * a->rows * tiles_of(a) * 64 : 0;
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
  if (a->cols % a->group != 0 || a->cols >= (1 << 24) || a->out_cols >= (1 << 24))
    return fail(IKL_EUNSUPPORTED, "int4 linear: cols must be whole groups; cols and out_cols below 2^24");
  if (a->gated && a->residual) return fail(IKL_EUNSUPPORTED, "int4 linear: a gated weight takes no residual");
  return IKL_OK;
}

// check_args, then the plan of a launch that has rows.
int plan_args(const ikl_int4_linear_args *a, Int4Plan &plan) {
  if (const int bad = check_args(a)) return bad;
  if (a->rows < int64_t(1) << 40) plan = plan_of(a->rows, tiles_of(a), steps_of(a), a->gated != 0, a->x_scales != nullptr);
  return plan.blocks || !a->rows ? IKL_OK : fail(IKL_EINVAL, "int4 linear: too many rows for a launch");
}

}  // namespace
}  // namespace ikl

using namespace ikl;

extern "C" int64_t ikl_int4_linear_workspace_size(const ikl_int4_linear_args *a) {
  Int4Plan plan{};
  if (const int bad = plan_args(a, plan)) return bad;
  return part_bytes(a, plan);
}

extern "C" int32_t ikl_int4_linear_plan(const ikl_int4_linear_args *a) {
  Int4Plan plan{};
  if (const int bad = plan_args(a, plan)) return bad;
  return a->rows ? plan.split | plan.nt << 8 | plan.mt << 16 | plan.few << 24 : 0;
}

extern "C" int ikl_int4_linear(const ikl_int4_linear_args *a, void *stream) {
  Int4Plan plan{};
  if (const int bad = plan_args(a, plan)) return bad;
  if (a->rows == 0) return IKL_OK;
  const int64_t eb = a->dtype == IKL_F32 ? 4 : 2;
  if (!a->x || !a->codes || !a->scales || !a->y) return fail(IKL_EINVAL, "int4 linear: NULL tensor pointer");
  if (off16(a->x) || (!a->x_scales && a->rows > 1 && a->x_stride % 8 != 0) || ((uintptr_t)a->x_scales & 3u))
    return fail(IKL_EINVAL, "int4 linear: x rows must be 16-byte aligned");
  if (off16(a->codes) || off16(a->scales) || ((uintptr_t)a->zeros & 3u))
    return fail(IKL_EINVAL, "int4 linear: the weight must be 16-byte aligned");
  if (a->rows > 1 && a->y_stride < a->out_cols) return fail(IKL_EINVAL, "int4 linear: rows of y must not overlap");
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
  p.tiles = tiles_of(a);
  p.steps = steps_of(a);
  p.groups = (int32_t)(a->cols / a->group);
  p.gated = a->gated != 0;
  p.dtype = a->dtype;
  p.wide = (((uintptr_t)p.y | (uintptr_t)p.y_st | (uintptr_t)p.res | (p.res ? (uintptr_t)p.res_st : 0)) & (uintptr_t)(4 * eb - 1)) == 0;
  if (const int64_t need = part_bytes(a, plan)) {
    if (!a->workspace || off16(a->workspace) || a->workspace_bytes < need)
      return fail(IKL_EWORKSPACE, "int4 linear: the workspace is missing, too small or not 16-byte aligned");
    p.part = (float *)a->workspace;
  }
  hipStream_t s = (hipStream_t)stream;
  if (a->x_scales) launch_int4_i8(p, a->group, plan, s);
  else if (a->dtype == IKL_BF16) launch_int4_bf16(p, a->group, plan, s);
  else launch_int4_f16(p, a->group, plan, s);
  if (plan.split > 1) {
    const int quads = 4 * (p.gated ? p.tiles / 2 : p.tiles);
    int4_join_kernel<<<dim3((unsigned)((p.rows * quads + 255) / 256)), 256, 0, s>>>(p, plan.split, quads);
  }
  return check_launch("int4 linear");
}
