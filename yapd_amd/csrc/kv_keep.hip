// The accepted nodes of drafted trees moved to consecutive positions, in every layer's pool.
//
// For row r with base b: new[b + i] = old[b + kept_i], i < n_kept, K and V of every head and layer.  A wave holds all of a
// (row, head, layer)'s values, at most 64 tokens, before it writes the first, so any indices may be given: a
// position may be read after the call has given it another token.
//
// Bound by the lines that V's columns touch: a token is 128 consecutive bytes of K and two bytes in each of 64
// pieces of V, every line of a page's head.  130 rows that keep 5 of 64 nodes on average, 30 layers of 16 heads, 147 us: 360 MB
// read and 183 written for 85 each of tokens, 3.7 TB/s.  Destination pages of V read, merged and written whole, 16
// values in registers instead of 64, 151 us; 16 values with plain stores 156.
#include "attn_tile.h"
#include "common.h"
#include "kv_layout.h"

namespace yapd {
namespace {

constexpr int kLayers = 64;  // pools of one launch
constexpr int kMaxKept = 64;

struct KeepParams {
  void* pool[kLayers];
  int64_t n_pages;
  const int32_t* table;
  int table_stride, table_cols;
  const int32_t* base;
  const int32_t* kept;
  int kept_stride, max_kept;
  const int32_t* n_kept;
  int H;
};

// T: uint16_t (bf16) or uint8_t.  blockIdx = (four heads, row, layer), a wave a head, lane = head dim.
template <class T>
__global__ __launch_bounds__(256) void kv_keep_kernel(const KeepParams P) {
  constexpr bool k8 = sizeof(T) == 1;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int h = blockIdx.x * 4 + wave, row = blockIdx.y;
  const int n = min(P.n_kept[row], P.max_kept);
  if (n <= 0) return;
  T* pool = static_cast<T*>(P.pool[blockIdx.z]);
  constexpr int64_t tile = k8 ? kTile8 : kHeadTile;
  // lane i: where token i comes from and goes to, as (page, slot) in one number, -1: outside what the row maps
  const int64_t b = P.base[row];
  auto place = [&](int64_t pos) -> int64_t {
    if (pos < 0 || pos >= static_cast<int64_t>(P.table_cols) * kPageSize) return -1;
    const int64_t page = P.table[static_cast<int64_t>(row) * P.table_stride + pos / kPageSize];
    return page < 0 || page >= P.n_pages ? -1 : page * kPageSize + pos % kPageSize;
  };
  int64_t from = -1, to = -1;
  if (lane < n) {
    const int64_t node = P.kept[static_cast<int64_t>(row) * P.kept_stride + lane];
    from = node < 0 ? -1 : place(b + node);
    to = place(b + lane);
    if (to == from || from < 0) to = -1;
  }
  if (!__any(to >= 0)) return;
  const int64_t any = to >= 0 ? from : -1;
  auto lane64 = [](int64_t v, int i) {
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(v), i);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(static_cast<uint64_t>(v) >> 32), i);
    return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
  };
  uint32_t kv[kMaxKept];
#pragma unroll
  for (int c = 0; c < kMaxKept / 16; ++c) {
    if (16 * c >= n) break;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int64_t at = lane64(any, 16 * c + j);
      if (at < 0) continue;
      const int64_t page = at / kPageSize;
      const int slot = static_cast<int>(at % kPageSize);
      const T* k = pool + (page * 2 * P.H + h) * tile + slot * kHeadDim + lane;
      const T* v = pool + ((page * 2 + 1) * P.H + h) * tile + lane * kPageSize + slot;
      kv[16 * c + j] = static_cast<uint32_t>(*k) | static_cast<uint32_t>(*v) << 16;
    }
  }
  uint32_t scales = 0;
  if constexpr (k8) {
    if (to >= 0) {
      const uint8_t* s = pool + (from / kPageSize * 2 * P.H + h) * tile + kHeadTile + from % kPageSize;
      scales = static_cast<uint32_t>(s[0]) | static_cast<uint32_t>(s[P.H * tile]) << 8;
    }
  }
  // every value has arrived before the first is written
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
  for (int c = 0; c < kMaxKept / 16; ++c) {
    if (16 * c >= n) break;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const int64_t at = lane64(to, 16 * c + j);
      if (at < 0) continue;
      const int64_t page = at / kPageSize;
      const int slot = static_cast<int>(at % kPageSize);
      pool[(page * 2 * P.H + h) * tile + slot * kHeadDim + lane] = static_cast<T>(kv[16 * c + j]);
      pool[((page * 2 + 1) * P.H + h) * tile + lane * kPageSize + slot] = static_cast<T>(kv[16 * c + j] >> 16);
    }
  }
  if constexpr (k8) {
    if (to >= 0) {
      uint8_t* s = pool + (to / kPageSize * 2 * P.H + h) * tile + kHeadTile + to % kPageSize;
      s[0] = static_cast<uint8_t>(scales);
      s[P.H * tile] = static_cast<uint8_t>(scales >> 8);
    }
  }
}

}  // namespace
}  // namespace yapd

extern "C" int yapd_kv_keep(void* const* kv_pools, int n_layers, int bits, int64_t n_pages, int n_heads,
                            const int32_t* page_table, int table_stride, int table_cols, const int32_t* base,
                            const int32_t* kept, int kept_stride, int max_kept, const int32_t* n_kept, int rows,
                            void* stream) {
  YAPD_REQUIRE(kv_pools && page_table && base && kept && n_kept, "kv_keep: NULL pointer");
  YAPD_REQUIRE(bits == 8 || bits == 16, "kv_keep: bits must be 8 or 16 (got %d)", bits);
  YAPD_REQUIRE(n_layers >= 1 && rows >= 1 && rows <= 65535 && n_pages >= 1,
               "kv_keep: need layers, pages and 1 <= rows <= 65535");
  YAPD_REQUIRE(n_heads >= 4 && n_heads % 4 == 0 && n_heads <= 1024,
               "kv_keep: n_heads must be a multiple of 4, at most 1024 (got %d)", n_heads);
  YAPD_REQUIRE(max_kept >= 1 && max_kept <= yapd::kMaxKept && (rows == 1 || kept_stride >= max_kept),
               "kv_keep: need 1 <= max_kept <= 64 entries a row");
  YAPD_REQUIRE(table_cols >= 1 && (rows == 1 || table_stride >= table_cols), "kv_keep: bad table shape");
  for (int l = 0; l < n_layers; ++l)
    YAPD_REQUIRE(kv_pools[l] && (reinterpret_cast<uintptr_t>(kv_pools[l]) & 15u) == 0,
                 "kv_keep: layer %d's pool must be non-NULL and 16-byte aligned", l);
  // a pool given twice would be moved twice, in no order
  const uintptr_t bytes = static_cast<uintptr_t>(n_pages) * 2 * n_heads * (bits == 8 ? yapd::kTile8 : yapd::kHeadTile * 2);
  for (int l = 1; l < n_layers; ++l)
    for (int m = 0; m < l; ++m) {
      const uintptr_t x = reinterpret_cast<uintptr_t>(kv_pools[l]), y = reinterpret_cast<uintptr_t>(kv_pools[m]);
      YAPD_REQUIRE((x > y ? x - y : y - x) >= bytes, "kv_keep: the pools of layers %d and %d overlap", m, l);
    }
  yapd::KeepParams P;
  P.n_pages = n_pages;
  P.table = page_table;
  P.table_stride = table_stride;
  P.table_cols = table_cols;
  P.base = base;
  P.kept = kept;
  P.kept_stride = kept_stride;
  P.max_kept = max_kept;
  P.n_kept = n_kept;
  P.H = n_heads;
  for (int l0 = 0; l0 < n_layers; l0 += yapd::kLayers) {
    const int nl = n_layers - l0 < yapd::kLayers ? n_layers - l0 : yapd::kLayers;
    for (int l = 0; l < nl; ++l) P.pool[l] = kv_pools[l0 + l];
    const dim3 grid(n_heads / 4, rows, nl);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (bits == 8)
      hipLaunchKernelGGL((yapd::kv_keep_kernel<uint8_t>), grid, dim3(256), 0, st, P);
    else
      hipLaunchKernelGGL((yapd::kv_keep_kernel<uint16_t>), grid, dim3(256), 0, st, P);
    YAPD_LAUNCH_CHECK("kv_keep_kernel launch");
  }
  return YAPD_OK;
}
