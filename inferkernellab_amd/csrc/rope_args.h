// What the kernels that rotate and append read: the parameters shared by the
// plain rotary append and the one with the heads' norms, and the checks of
// their arguments.
#pragma once

#include "ikl_common.h"

namespace ikl {

struct RopeParams {
  const char *q_in;
  char *q_out;
  int64_t qi_st, qi_sh, qo_st, qo_sh;  // bytes
  const char *key;
  const char *value;
  int64_t k_st, k_sh, v_st, v_sh;      // bytes
  const char *cos;
  const char *sin;
  int64_t cos_st, sin_st;              // bytes
  const void *slots;
  char *kc;
  char *vc;
  int64_t kc_sb, kc_st, kc_sh;         // bytes
  int64_t vc_sb, vc_st, vc_sh;         // bytes
  int64_t num_slots;
  int32_t block_size;
  int32_t num_heads;                   // 0 when q is not rotated
  int32_t num_kv_heads;
  int32_t half_chunks;                 // 16-byte chunks in half a row
};

inline bool al16(const void *ptr) { return ((uintptr_t)ptr & 15u) == 0; }

// Checks the arguments and fills *out; messages begin with `what`.
inline int rope_params(const ikl_rope_append_args *a, const char *what, RopeParams *out) {
  const std::string w(what);
  if (!a) return fail(IKL_EINVAL, w + ": null argument struct");
  if (a->num_tokens < 0) return fail(IKL_EINVAL, w + ": num_tokens must be non-negative");
  if (a->num_tokens == 0) return IKL_OK;  // *out is left as it is
  if (a->num_tokens > 0x7fffffffLL) return fail(IKL_EINVAL, w + ": too many tokens for one launch");
  if (a->block_size <= 0 || a->num_blocks <= 0 || a->num_kv_heads <= 0 || a->head_dim <= 0 || a->num_heads < 0)
    return fail(IKL_EINVAL, w + ": dimensions must be positive");
  if (!a->key || !a->value || !a->cos || !a->sin || !a->slots || !a->k_cache || !a->v_cache)
    return fail(IKL_EINVAL, w + ": null tensor pointer");
  if (a->num_heads > 0 && (!a->query || !a->query_out))
    return fail(IKL_EINVAL, w + ": query rotation needs query and query_out");
  if (a->slot_type != IKL_I32 && a->slot_type != IKL_I64)
    return fail(IKL_EINVAL, w + ": slots must use int32 or int64");
  int eb;
  switch (a->dtype) {
    case IKL_F16:
    case IKL_BF16: eb = 2; break;
    case IKL_F32: eb = 4; break;
    default: return fail(IKL_EINVAL, w + ": unsupported dtype");
  }
  const bool fp8 = a->cache_dtype == IKL_FP8_E4M3;
  if (a->cache_dtype != 0 && a->cache_dtype != a->dtype && !fp8)
    return fail(IKL_EINVAL, w + ": cache_dtype must be 0, the tensor dtype or IKL_FP8_E4M3");
  const int64_t row = (int64_t)a->head_dim * eb;
  if (row % 32 != 0)
    return fail(IKL_EUNSUPPORTED, w + ": head_dim * element size must be a multiple of 32 bytes");
  if (fp8 && (a->head_dim % 8 != 0 || a->head_dim > 512))
    return fail(IKL_EUNSUPPORTED, w + ": the FP8 cache needs head_dim a multiple of 8, at most 512");
  if (fp8 && (!a->k_scale || !a->v_scale)) return fail(IKL_EINVAL, w + ": the FP8 cache needs k_scale and v_scale");
  const int ceb = fp8 ? 1 : eb;  // cache bytes per element
  RopeParams &p = *out;
  p.q_in = (const char *)a->query;
  p.q_out = (char *)a->query_out;
  p.qi_st = a->q_stride_t * eb;
  p.qi_sh = a->q_stride_h * eb;
  p.qo_st = a->q_out_stride_t * eb;
  p.qo_sh = a->q_out_stride_h * eb;
  p.key = (const char *)a->key;
  p.value = (const char *)a->value;
  p.k_st = a->key_stride_t * eb;
  p.k_sh = a->key_stride_h * eb;
  p.v_st = a->value_stride_t * eb;
  p.v_sh = a->value_stride_h * eb;
  p.cos = (const char *)a->cos;
  p.sin = (const char *)a->sin;
  p.cos_st = a->cos_stride_t * eb;
  p.sin_st = a->sin_stride_t * eb;
  p.slots = a->slots;
  p.kc = (char *)a->k_cache;
  p.vc = (char *)a->v_cache;
  p.kc_sb = a->k_stride_block * ceb;
  p.kc_st = a->k_stride_token * ceb;
  p.kc_sh = a->k_stride_head * ceb;
  p.vc_sb = a->v_stride_block * ceb;
  p.vc_st = a->v_stride_token * ceb;
  p.vc_sh = a->v_stride_head * ceb;
  p.num_slots = a->num_blocks * (int64_t)a->block_size;
  p.block_size = a->block_size;
  p.num_heads = a->num_heads;
  p.num_kv_heads = a->num_kv_heads;
  p.half_chunks = (int32_t)(row / 32);
  const bool ok = al16(a->key) && al16(a->value) && al16(a->cos) && al16(a->sin) && al16(a->k_cache) &&
                  al16(a->v_cache) && (a->num_heads == 0 || (al16(a->query) && al16(a->query_out))) &&
                  p.qi_st % 16 == 0 && p.qi_sh % 16 == 0 && p.qo_st % 16 == 0 && p.qo_sh % 16 == 0 &&
                  p.k_st % 16 == 0 && p.k_sh % 16 == 0 && p.v_st % 16 == 0 && p.v_sh % 16 == 0 &&
                  p.cos_st % 16 == 0 && p.sin_st % 16 == 0 && p.kc_sb % 16 == 0 && p.kc_st % 16 == 0 &&
                  p.kc_sh % 16 == 0 && p.vc_sb % 16 == 0 && p.vc_st % 16 == 0 && p.vc_sh % 16 == 0;
  if (!ok) return fail(IKL_EINVAL, w + ": rows must be 16-byte aligned");
  if (fp8) {
    if (((uintptr_t)a->k_scale & 3u) || ((uintptr_t)a->v_scale & 3u))
      return fail(IKL_EINVAL, w + ": misaligned scale tensor");
    if ((int64_t)a->num_heads + 2 * (int64_t)a->num_kv_heads > 0x7fffffffLL)
      return fail(IKL_EINVAL, w + ": too many heads");
  }
  return IKL_OK;
}

}  // namespace ikl
