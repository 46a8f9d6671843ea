// kvcopy.cu -- copies of whole KV pages inside their pools: forking a sequence's partly filled
// page, packing the live pages of a pool.  The reference clones whole caches instead
// (crates/higgs-engine/src/prompt_cache.rs:186-224 stores a cloned AnyCache).
//
// page dst[i] := page src[i] for every pair i, layer and pool; no destination is a source or
// another pair's destination (the host checks), so the pairs commute and one launch needs no
// order among them.
//
// Bound: HBM, one read and one write of every page byte.  The page ids are host lists (the block
// pool is host memory), so they travel as kernel parameters: no copy to the device comes before
// the launch.  One warp moves one piece of a page, at most 4 KB: eight 16-byte loads per lane are
// in flight before the first store, and the division of the piece's index is paid once per 4 KB.
// B200: 500 pages of 36 layers (2.36 GB moved) 354 us = 6.67 TB/s; 77 pages of a 4-bit cache (94 MB)
// 16.9 us = 5.5 TB/s, start and drain included; four pages of 28 layers 3.8 us, of which most is the launch.
#include <algorithm>
#include <new>
#include <vector>

#include "common.cuh"

namespace higgs {
namespace {

constexpr int kCopyThreads = 256;
constexpr int kCopyVecs = 8;                          // 16-byte vectors per lane
constexpr int64_t kPieceBytes = 32 * 16 * kCopyVecs;  // 4 KB
constexpr int kMaxPools = 8;

struct CopyPool {
  char* base;
  int64_t layer_stride, page_stride, page_bytes;
  int pieces;         // of one page
  int64_t first, n;   // pieces of the launch before this pool's, pieces of this pool
};

template <int CAP>
struct CopyArgs {
  CopyPool pool[kMaxPools];
  int n_pools, n_pairs;
  int32_t src[CAP], dst[CAP];
};

template <int CAP>
__global__ void __launch_bounds__(kCopyThreads) kv_copy_pages_kernel(const __grid_constant__ CopyArgs<CAP> a) {
  pdl_wait();
  pdl_launch();
  const int64_t u = (int64_t)blockIdx.x * (kCopyThreads / 32) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  int p = 0;
  while (p < a.n_pools && u >= a.pool[p].first + a.pool[p].n) ++p;
  if (p == a.n_pools) return;
  const CopyPool& q = a.pool[p];
  // piece fastest, then the pair, then the layer: n_pairs * pieces fits 32 bits (checked)
  const int64_t v = u - q.first;
  const int per_layer = a.n_pairs * q.pieces;
  const int layer = (int)(v / per_layer), w = (int)(v % per_layer);
  const int pair = w / q.pieces, piece = w % q.pieces;
  const int64_t at = (int64_t)piece * kPieceBytes;
  const int vecs = (int)(min((int64_t)kPieceBytes, q.page_bytes - at) >> 4);
  char* const layer_base = q.base + layer * q.layer_stride + at;
  const uint4* src = reinterpret_cast<const uint4*>(layer_base + a.src[pair] * q.page_stride);
  uint4* dst = reinterpret_cast<uint4*>(layer_base + a.dst[pair] * q.page_stride);
  uint4 r[kCopyVecs];
#pragma unroll
  for (int i = 0; i < kCopyVecs; ++i)
    if (lane + 32 * i < vecs) r[i] = __ldcs(src + lane + 32 * i);
#pragma unroll
  for (int i = 0; i < kCopyVecs; ++i)
    if (lane + 32 * i < vecs) __stcs(dst + lane + 32 * i, r[i]);
}

template <int CAP>
int launch_copy(const higgs_kv_pool* pools, int n_pools, const int32_t* src, const int32_t* dst, int n,
                cudaStream_t st) {
  CopyArgs<CAP> a;
  a.n_pools = n_pools;
  a.n_pairs = n;
  int64_t total = 0;
  for (int i = 0; i < n_pools; ++i) {
    CopyPool& q = a.pool[i];
    q.base = (char*)pools[i].base;
    q.layer_stride = pools[i].layer_stride;
    q.page_stride = pools[i].page_stride;
    q.page_bytes = pools[i].page_bytes;
    q.pieces = (int)((q.page_bytes + kPieceBytes - 1) / kPieceBytes);
    q.first = total;
    q.n = (int64_t)pools[i].layers * n * q.pieces;
    total += q.n;
  }
  std::copy(src, src + n, a.src);
  std::copy(dst, dst + n, a.dst);
  const int64_t grid = (total + kCopyThreads / 32 - 1) / (kCopyThreads / 32);
  HG_CHECK_ARG(grid <= INT32_MAX, "higgs_kv_copy_pages: too many bytes for one call");
  HG_CUDA(launch_pdl(kv_copy_pages_kernel<CAP>, dim3((unsigned)grid), dim3(kCopyThreads), 0, st, a));
  return HIGGS_OK;
}

// No byte belongs to pages of two layers: a layer's pages before the next layer's, or the layers of a
// page before the next page.
bool layers_apart(const higgs_kv_pool& p) {
  if (p.layers == 1) return true;
  typedef __int128 wide;
  const wide pages = p.num_pages == 1 ? 0 : (wide)(p.num_pages - 1) * p.page_stride;
  return p.layer_stride >= p.page_bytes &&
         (p.layer_stride >= pages + p.page_bytes || p.page_stride >= (wide)(p.layers - 1) * p.layer_stride + p.page_bytes);
}

// The pairs fit the pools and commute: ids in range, no destination twice, none among the sources.
int check_pairs(const int32_t* src, const int32_t* dst, int n, int64_t pages) {
  for (int i = 0; i < n; ++i)
    HG_CHECK_ARG(src[i] >= 0 && src[i] < pages && dst[i] >= 0 && dst[i] < pages,
                 "higgs_kv_copy_pages: page id outside the pools");
  std::vector<int32_t> d(dst, dst + n), s(src, src + n);
  std::sort(d.begin(), d.end());
  std::sort(s.begin(), s.end());
  HG_CHECK_ARG(std::adjacent_find(d.begin(), d.end()) == d.end(),
               "higgs_kv_copy_pages: a page is the destination of two copies");
  for (size_t i = 0, j = 0; i < d.size() && j < s.size();) {
    HG_CHECK_ARG(d[i] != s[j], "higgs_kv_copy_pages: a destination is also a source");
    d[i] < s[j] ? ++i : ++j;
  }
  return HIGGS_OK;
}

}  // namespace
}  // namespace higgs

using namespace higgs;

extern "C" int higgs_kv_copy_pages(higgs_ctx* ctx, const higgs_kv_pool* pools, int n_pools, const int32_t* src,
                                   const int32_t* dst, int n, void* stream) try {
  HG_CHECK_ARG(ctx && pools, "higgs_kv_copy_pages: null argument");
  HG_CHECK_ARG(n >= 0 && (n == 0 || (src && dst)), "higgs_kv_copy_pages: bad page lists");
  HG_CHECK_ARG(n_pools > 0 && n_pools <= kMaxPools, "higgs_kv_copy_pages: 1 to 8 pools");
  int64_t pages = INT32_MAX;
  for (int i = 0; i < n_pools; ++i) {
    const higgs_kv_pool& p = pools[i];
    HG_CHECK_ARG(p.base && p.layers > 0 && p.num_pages > 0 && p.page_bytes > 0, "higgs_kv_copy_pages: empty pool");
    HG_CHECK_ARG((((uintptr_t)p.base | p.page_bytes | p.page_stride | p.layer_stride) & 15) == 0,
                 "higgs_kv_copy_pages: bases, strides and page sizes must be multiples of 16 bytes");
    HG_CHECK_ARG(p.num_pages == 1 || p.page_stride >= p.page_bytes,
                 "higgs_kv_copy_pages: pages overlap");
    HG_CHECK_ARG(layers_apart(p), "higgs_kv_copy_pages: layers overlap");
    HG_CHECK_ARG(p.page_bytes <= (int64_t)1 << 30, "higgs_kv_copy_pages: page larger than 1 GiB");
    pages = std::min(pages, p.num_pages);
  }
  if (n == 0) return HIGGS_OK;
  if (int rc = check_pairs(src, dst, n, pages)) return rc;
  HG_DEVICE(ctx);
  // parameters are copied at every launch, so short lists use a short argument block
  constexpr int kSmall = 16, kMiddle = 128, kLarge = 1024;
  for (int i = 0; i < n; i += kLarge) {
    const int m = std::min(kLarge, n - i);
    const auto launch = m <= kSmall ? launch_copy<kSmall> : m <= kMiddle ? launch_copy<kMiddle> : launch_copy<kLarge>;
    if (int rc = launch(pools, n_pools, src + i, dst + i, m, (cudaStream_t)stream)) return rc;
  }
  return HIGGS_OK;
} catch (const std::bad_alloc&) {
  return fail(HIGGS_ERR_STATE, "higgs_kv_copy_pages: out of host memory");
}
