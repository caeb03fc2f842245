// Copies of whole cache pages, the same pairs in every layer's pool: forking a
// row (its partial last page), copying a prefix, compacting a pool.
//
// pool_l[dst_i] = pool_l[src_i].  Nothing but bytes: a page is n_heads * 4 KiB,
// read once and written once.  No destination is another pair's source or
// destination (the host checks), so the copies may run in any order, all layers in one launch.
// The pairs and the pool addresses travel as kernel arguments: no upload, no
// device list to keep alive, and a captured launch holds its own copy.
//
// Bound by memory.  30 layers of 16 heads: 301 pages 217 us, 5.45 TB/s read and
// written (a copy of 1 GiB reaches 5.18); a prefix of 19 pages to seven rows
// 48.6 us; one page 2.8 us.  The stores are non-temporal, so they do not push
// out what is still to be read: with plain ones the prefix, whose reads the
// caches can serve six times of seven, takes 79.6 us and the 301 pages 225.9.
// One workgroup that reads a source's segment once and writes all its copies
// was slower (54.3 us), having fewer loads in flight.
#include <new>
#include <vector>

#include "attn_tile.h"
#include "common.h"
#include "kv_layout.h"

namespace yapd {
namespace {

constexpr int kLayers = 64;   // pools and ...
constexpr int kPairs = 384;   // ... pairs of one launch: kernel arguments hold 4 KiB
constexpr int kWords = 1024;  // 16-byte words a workgroup copies

struct CopyParams {
  uint16_t* pool[kLayers];
  int32_t src[kPairs], dst[kPairs];
  int words;  // 16-byte words of a page
};

// blockIdx = (segment of a page, pair, layer)
__global__ __launch_bounds__(256) void kv_copy_pages_kernel(const CopyParams P) {
  const int64_t page_elems = static_cast<int64_t>(P.words) * 8;
  uint16_t* pool = P.pool[blockIdx.z];
  const uint16_t* src = pool + P.src[blockIdx.y] * page_elems;
  uint16_t* dst = pool + P.dst[blockIdx.y] * page_elems;
  const int w0 = blockIdx.x * kWords + threadIdx.x;
  u32x4_t v[kWords / 256];
#pragma unroll
  for (int i = 0; i < kWords / 256; ++i)
    if (w0 + 256 * i < P.words) v[i] = load16(src + (w0 + 256 * i) * 8);
#pragma unroll
  for (int i = 0; i < kWords / 256; ++i)
    if (w0 + 256 * i < P.words)
      __builtin_nontemporal_store(v[i], reinterpret_cast<u32x4_t*>(dst + (w0 + 256 * i) * 8));
}

// Whether the pairs may be copied in any order: ids inside the pool, every
// destination once and no source among them.  YAPD_OK or YAPD_EINVAL.
int check_pairs(const int32_t* src, const int32_t* dst, int n_pairs, int64_t n_pages) {
  std::vector<bool> is_dst;
  try {
    is_dst.assign(static_cast<size_t>(n_pages), false);
  } catch (const std::bad_alloc&) {
    set_error("kv_copy_pages: out of host memory");
    return YAPD_EINVAL;
  }
  for (int i = 0; i < n_pairs; ++i) {
    YAPD_REQUIRE(src[i] >= 0 && src[i] < n_pages && dst[i] >= 0 && dst[i] < n_pages,
                 "kv_copy_pages: pair %d (%d -> %d) outside the pool's %lld pages", i, src[i], dst[i],
                 static_cast<long long>(n_pages));
    YAPD_REQUIRE(!is_dst[dst[i]], "kv_copy_pages: page %d is the destination of two pairs", dst[i]);
    is_dst[dst[i]] = true;
  }
  for (int i = 0; i < n_pairs; ++i)
    YAPD_REQUIRE(!is_dst[src[i]], "kv_copy_pages: page %d is a source and a destination", src[i]);
  return YAPD_OK;
}

}  // namespace
}  // namespace yapd

extern "C" int yapd_kv_copy_pages(void* const* kv_pools, int n_layers, int64_t n_pages, int n_heads, const int32_t* src,
                                  const int32_t* dst, int n_pairs, void* stream) {
  YAPD_REQUIRE(n_pairs >= 0 && n_layers >= 1 && n_heads >= 1 && n_heads <= 4096, "kv_copy_pages: empty shape");
  YAPD_REQUIRE(n_pages >= 1 && n_pages <= INT32_MAX, "kv_copy_pages: need 1 <= n_pages < 2^31");
  YAPD_REQUIRE(kv_pools && (n_pairs == 0 || (src && dst)), "kv_copy_pages: NULL pointer");
  for (int l = 0; l < n_layers; ++l)
    YAPD_REQUIRE(kv_pools[l] && (reinterpret_cast<uintptr_t>(kv_pools[l]) & 15u) == 0,
                 "kv_copy_pages: layer %d's pool must be non-NULL and 16-byte aligned", l);
  if (int rc = yapd::check_pairs(src, dst, n_pairs, n_pages)) return rc;
  yapd::CopyParams P;
  P.words = 2 * n_heads * yapd::kHeadTile / 8;
  const unsigned segs = (P.words + yapd::kWords - 1) / yapd::kWords;
  for (int l0 = 0; l0 < n_layers; l0 += yapd::kLayers) {
    const int nl = n_layers - l0 < yapd::kLayers ? n_layers - l0 : yapd::kLayers;
    for (int l = 0; l < nl; ++l) P.pool[l] = static_cast<uint16_t*>(kv_pools[l0 + l]);
    for (int p0 = 0; p0 < n_pairs; p0 += yapd::kPairs) {
      const int np = n_pairs - p0 < yapd::kPairs ? n_pairs - p0 : yapd::kPairs;
      for (int i = 0; i < np; ++i) {
        P.src[i] = src[p0 + i];
        P.dst[i] = dst[p0 + i];
      }
      hipLaunchKernelGGL(yapd::kv_copy_pages_kernel, dim3(segs, np, nl), dim3(256), 0, static_cast<hipStream_t>(stream),
                         P);
      YAPD_LAUNCH_CHECK("kv_copy_pages_kernel launch");
    }
  }
  return YAPD_OK;
}
