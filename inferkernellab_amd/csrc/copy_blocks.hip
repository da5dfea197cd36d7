// Pages of the cache copied to other pages over all layers: the copies of a
// forked request or of a compaction. A page is a dense run of bytes in every
// layout of the cache, so it is copied as such; K, V and an FP8 cache's scales
// go in one launch. Bound: memory. The stores are non-temporal: what is written
// is not read again soon, and kept out of the caches it leaves them to the reads
// (32 pages of 32 layers, 134 MB: 31.0 -> 24.4 us, 5.5 TB/s; 512 of 16 layers, 1.07
// GB: 224 -> 221 us, 4.9 TB/s, where a plain copy of 1 GiB runs at 5.2). 2 or 8
// pieces a thread and workgroups of 512 are within 3 % of these.
//
// A list of pairs that the host holds travels in the launch's arguments, PAIRS
// at a time: no upload, no wait, and a captured launch keeps its pairs.
#include <new>
#include <vector>

#include "ikl_common.h"

namespace ikl {
namespace {

constexpr int PAIRS = 384;  // 3 KB of the 4 KB of arguments
constexpr int FEW = 16;
constexpr int COPY_THREADS = 256;
constexpr int UNITS = 4;    // pieces a thread has in flight

struct CopyTensor {
  char *base;
  int64_t stride_layer, stride_block, units;  // units: pieces per page
};
struct CopyParams {
  CopyTensor tensor[IKL_COPY_MAX_TENSORS];
  int64_t first[IKL_COPY_MAX_TENSORS + 1];  // first workgroup of each tensor's share, of one pair and layer
  int64_t num_blocks;
  int64_t first_pair;  // of this launch
  int32_t num_layers;
  int32_t num_tensors;
};
template <int N>
struct HostPairs {
  int32_t src[N], dst[N];
  __device__ inline int64_t from(int64_t i) const { return src[i]; }
  __device__ inline int64_t to(int64_t i) const { return dst[i]; }
};
template <typename IdxT>
struct DevicePairs {
  const IdxT *src, *dst;
  __device__ inline int64_t from(int64_t i) const { return (int64_t)src[i]; }
  __device__ inline int64_t to(int64_t i) const { return (int64_t)dst[i]; }
};

template <typename Unit>
__device__ inline void store_out(Unit *p, const Unit &v) {
  *p = v;
}
__device__ inline void store_out(u32x4 *p, const u32x4 &v) {
  __builtin_nontemporal_store((v4u32){v.x, v.y, v.z, v.w}, reinterpret_cast<v4u32 *>(p));
}

template <typename Unit, typename Pairs>
__global__ __launch_bounds__(COPY_THREADS) void copy_blocks_kernel(const CopyParams p, const Pairs pairs) {
  // workgroup = (pair, layer, part of the page's tensors)
  const int64_t parts = p.first[p.num_tensors];
  const int64_t page = blockIdx.x / parts, part = blockIdx.x - page * parts;
  const int64_t in_launch = page / p.num_layers, layer = page - in_launch * p.num_layers;
  const int64_t pair = p.first_pair + in_launch;
  int n = 0;
  while (n + 1 < p.num_tensors && part >= p.first[n + 1]) ++n;
  const int64_t from = pairs.from(pair), to = pairs.to(pair);
  if (from < 0 || from >= p.num_blocks || to < 0 || to >= p.num_blocks) return;
  const CopyTensor &t = p.tensor[n];
  char *at = t.base + layer * t.stride_layer;
  const Unit *src = reinterpret_cast<const Unit *>(at + from * t.stride_block);
  Unit *dst = reinterpret_cast<Unit *>(at + to * t.stride_block);
  const int64_t first = (part - p.first[n]) * (COPY_THREADS * UNITS) + threadIdx.x;
  Unit u[UNITS];
#pragma unroll
  for (int i = 0; i < UNITS; ++i)
    if (first + i * COPY_THREADS < t.units) u[i] = src[first + i * COPY_THREADS];
#pragma unroll
  for (int i = 0; i < UNITS; ++i)
    if (first + i * COPY_THREADS < t.units) store_out(dst + first + i * COPY_THREADS, u[i]);
}

// In as few launches as hold the workgroups.
template <typename Unit, typename Pairs>
int launch(CopyParams p, const Pairs &pairs, int64_t count, hipStream_t s) {
  int64_t each, all;  // workgroups of a pair, of all pairs
  if (__builtin_mul_overflow((int64_t)p.num_layers, p.first[p.num_tensors], &each) || each > max_grid(COPY_THREADS) ||
      __builtin_mul_overflow(each, count, &all) || all > 0x7fffffffLL)
    return fail(IKL_EINVAL, "copy blocks: too many pages for one call");
  const int64_t most = max_grid(COPY_THREADS) / each;
  for (p.first_pair = 0; p.first_pair < count; p.first_pair += most) {
    const int64_t n = count - p.first_pair < most ? count - p.first_pair : most;
    copy_blocks_kernel<Unit, Pairs><<<dim3((unsigned)(n * each)), COPY_THREADS, 0, s>>>(p, pairs);
    if (const int bad = check_launch("copy blocks launch"); bad != IKL_OK) return bad;
  }
  return IKL_OK;
}

// Pieces of 16, 4 or 1 bytes: the largest that addresses, strides and sizes of
// every page are a multiple of.
template <typename Pairs>
int launch(CopyParams p, int unit, const Pairs &pairs, int64_t count, hipStream_t s) {
  for (int n = 0; n < p.num_tensors; ++n) {
    p.tensor[n].units /= unit;
    const int64_t per = COPY_THREADS * UNITS;
    p.first[n + 1] = p.first[n] + (p.tensor[n].units + per - 1) / per;
  }
  if (unit == 16) return launch<u32x4, Pairs>(p, pairs, count, s);
  if (unit == 4) return launch<uint32_t, Pairs>(p, pairs, count, s);
  return launch<uint8_t, Pairs>(p, pairs, count, s);
}

// What a list on the host may not hold.
template <typename IdxT>
int check_pairs(const IdxT *src, const IdxT *dst, int64_t count, int64_t blocks) {
  std::vector<uint8_t> use((size_t)blocks, 0);
  for (int64_t i = 0; i < count; ++i) {
    if (src[i] < 0 || src[i] >= blocks || dst[i] < 0 || dst[i] >= blocks)
      return fail(IKL_EINVAL, "copy blocks: invalid block id");
    if (use[(size_t)dst[i]] & 2) return fail(IKL_EINVAL, "copy blocks: a block is written twice");
    use[(size_t)dst[i]] |= 2;
    use[(size_t)src[i]] |= 1;
  }
  for (int64_t i = 0; i < count; ++i)
    if (use[(size_t)dst[i]] & 1) return fail(IKL_EINVAL, "copy blocks: a block is both read and written");
  return IKL_OK;
}

template <int N, typename IdxT>
int launch_host(const CopyParams &p, int unit, const IdxT *src, const IdxT *dst, int64_t count, hipStream_t s) {
  HostPairs<N> pairs;
  for (int64_t j = 0; j < N; ++j) {
    pairs.src[j] = j < count ? (int32_t)src[j] : -1;
    pairs.dst[j] = j < count ? (int32_t)dst[j] : -1;
  }
  return launch(p, unit, pairs, count, s);
}

template <typename IdxT>
int copy_host(const CopyParams &p, int unit, const void *src, const void *dst, int64_t count, hipStream_t s) {
  const IdxT *from = (const IdxT *)src, *to = (const IdxT *)dst;
  if (const int bad = check_pairs(from, to, count, p.num_blocks); bad != IKL_OK) return bad;
  if (count <= FEW) return launch_host<FEW>(p, unit, from, to, count, s);
  for (int64_t i = 0; i < count; i += PAIRS)
    if (const int bad = launch_host<PAIRS>(p, unit, from + i, to + i, count - i < PAIRS ? count - i : PAIRS, s); bad != IKL_OK)
      return bad;
  return IKL_OK;
}

}  // namespace
}  // namespace ikl

using namespace ikl;

extern "C" int ikl_copy_blocks(const ikl_copy_blocks_args *a, void *stream) {
  if (!a) return fail(IKL_EINVAL, "copy blocks: null argument struct");
  if (a->num_pairs < 0) return fail(IKL_EINVAL, "copy blocks: num_pairs must be non-negative");
  if (a->num_tensors < 1 || a->num_tensors > IKL_COPY_MAX_TENSORS)
    return fail(IKL_EINVAL, "copy blocks: num_tensors must be 1 .. IKL_COPY_MAX_TENSORS");
  if (a->num_layers <= 0 || a->num_layers > 0x7fffffffLL || a->num_blocks <= 0 || a->num_blocks > 0x7fffffffLL)
    return fail(IKL_EINVAL, "copy blocks: dimensions must be positive");
  if (a->index_type != IKL_I32 && a->index_type != IKL_I64)
    return fail(IKL_EINVAL, "copy blocks: block ids must use int32 or int64");
  CopyParams p = {};
  p.num_blocks = a->num_blocks;
  p.num_layers = (int32_t)a->num_layers;
  p.num_tensors = a->num_tensors;
  uintptr_t bits = 0;  // of all addresses, strides and sizes
  for (int n = 0; n < a->num_tensors; ++n) {
    if (!a->base[n]) return fail(IKL_EINVAL, "copy blocks: null tensor pointer");
    if (a->page_bytes[n] <= 0) return fail(IKL_EINVAL, "copy blocks: dimensions must be positive");
    p.tensor[n] = CopyTensor{(char *)a->base[n], a->stride_layer[n], a->stride_block[n], a->page_bytes[n]};
    bits |= (uintptr_t)a->base[n] | (uintptr_t)a->stride_layer[n] | (uintptr_t)a->stride_block[n] |
            (uintptr_t)a->page_bytes[n];
  }
  if (a->num_pairs == 0) return IKL_OK;
  if (!a->src || !a->dst) return fail(IKL_EINVAL, "copy blocks: null block ids");
  const int unit = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
  hipStream_t s = (hipStream_t)stream;
  const bool i64 = a->index_type == IKL_I64;
  if (a->pairs_on_host) {
    try {
      return i64 ? copy_host<int64_t>(p, unit, a->src, a->dst, a->num_pairs, s)
                 : copy_host<int32_t>(p, unit, a->src, a->dst, a->num_pairs, s);
    } catch (const std::bad_alloc &) {
      return fail(IKL_EINVAL, "copy blocks: out of host memory");
    }
  }
  if (i64) return launch(p, unit, DevicePairs<int64_t>{(const int64_t *)a->src, (const int64_t *)a->dst}, a->num_pairs, s);
  return launch(p, unit, DevicePairs<int32_t>{(const int32_t *)a->src, (const int32_t *)a->dst}, a->num_pairs, s);
}
