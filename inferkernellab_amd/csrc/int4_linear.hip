// y = x W^T over 4-bit weights with a scale (and a zero point) for each output
// column and group of the contraction, for rows in 16 or in 8 bits: arguments,
// how a launch is cut, and the join of a split contraction.
#include "int4_linear.h"

namespace ikl {
namespace {

// Sums of a split contraction's parts, in their order, and the epilogue: a
// thread four columns of a row.
__global__ __launch_bounds__(256) void int4_join_kernel(const Int4Params p, const int split, const int quads) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  const int64_t row = blockIdx.y;
  if (i >= quads) return;
  const int per = p.gated ? 2 : 1, tile = i / 4 * per, q = i & 3;
  const float *part = p.part + row * 16 * p.tiles + 16 * tile + 4 * q;
  const int64_t step = p.rows * 16 * p.tiles;
  f32x4_t v = {0.f, 0.f, 0.f, 0.f}, u = v;
  for (int z = 0; z < split; ++z, part += step) {
    v += *reinterpret_cast<const f32x4_t *>(part);
    if (p.gated) u += *reinterpret_cast<const f32x4_t *>(part + 16);
  }
  const int col = tile_col(p, tile, q);
  if (col < p.outs) finish(p, row, col, p.gated ? gate_up(v, u) : v);
}

Int4Plan plan_of(int64_t rows, int tiles, int steps) {
  if (rows <= 64) return {0, 0, 1};
  const int mt = rows <= 128 ? 4 : 8, wt = 4;
  const int64_t groups = ((rows + 16 * mt - 1) / (16 * mt)) * ((tiles + 4 * wt - 1) / (4 * wt));
  int split = 1;
  while (split < 16 && groups * split * 2 <= 512 && steps / (split * 2) >= 4) split *= 2;
  return {mt, wt, split};
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
  if (a->rows > 128LL * 65535) return fail(IKL_EINVAL, "int4 linear: too many rows for a launch");
  return IKL_OK;
}

}  // namespace
}  // namespace ikl

using namespace ikl;

extern "C" int64_t ikl_int4_linear_workspace_size(const ikl_int4_linear_args *a) {
  if (const int bad = check_args(a)) return bad;
  return part_bytes(a, plan_of(a->rows, tiles_of(a), steps_of(a)));
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
  p.tiles = tiles_of(a);
  p.steps = steps_of(a);
  p.groups = (int32_t)(a->cols / a->group);
  p.gated = a->gated != 0;
  p.dtype = a->dtype;
  p.wide = (((uintptr_t)p.y | (uintptr_t)p.y_st | (uintptr_t)p.res | (p.res ? (uintptr_t)p.res_st : 0)) & (uintptr_t)(4 * eb - 1)) == 0;
  const Int4Plan plan = plan_of(a->rows, p.tiles, p.steps);
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
    int4_join_kernel<<<dim3((unsigned)((quads + 255) / 256), (unsigned)p.rows), 256, 0, s>>>(p, plan.split, quads);
  }
  return check_launch("int4 linear");
}
