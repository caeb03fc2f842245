// The 8-bit KV cache: fresh keys and values quantised as they are written into its pages, and pages
// read back as bf16.
//
// One scale a (token, head, plane), a power of two.  For the 64 values x of a token's head:
//   e = max(floor(log2 max|x|) - 6, -126),  c = clamp(round to even(x 2^-e), -127, 127),  value = c 2^e.
// |x - value| <= 2^(e-1), for max|x| >= 2^-120 (where e is not held to -126 and the largest code is at least 64) at most
// max|x| / 128; smaller vectors are off by up to 2^-127 whatever their size.  x 2^-e is exact, so a code is
// the same whoever computes it, and c 2^e is a bf16 value (7 bits), so reading back rounds nothing: attention
// over the codes and over the pages read back see the same keys.  (A scale of max|x| / 127 would halve the
// step for vectors just above a power of two, at the price of codes that depend on a division's rounding.)
// NaN is written as 0, an infinity as the largest finite bf16.
//
// Both are bound by memory.  37 chunks of 100 to 1500 tokens x 16 heads: written 35.5 us, 5.2 TB/s; with 0 to 2500
// earlier tokens read back 89.5 us, 5.2 TB/s.  Eight rows of one token: 4.1 us to write, 3.7 to read back up to 300.
#include "attn_tile.h"
#include "common.h"
#include "kv_layout.h"

namespace yapd {
namespace {

struct Write8Params {
  const uint16_t* x[2];  // k, v
  int64_t tok_stride[2];
  uint8_t* pool;
  int64_t n_pages;
  const int32_t* table;
  int table_stride, table_cols;
  const int32_t* pos0;
  const int32_t* q_start;  // [rows + 1], or NULL: row r's tokens are r * bl ..
  int rows, n_tokens, bl, H;
};

__device__ __forceinline__ int first_token(const Write8Params& P, int r) { return min(max(P.q_start[r], 0), P.n_tokens); }

// The 16 bf16 values of two 16-byte words as fp32: NaN as 0, infinities as the largest finite value.
__device__ __forceinline__ void finite16(u32x4_t a, u32x4_t b, float (&f)[16]) {
  const float top = __uint_as_float(0x7f7f0000u);
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    const uint32_t two = w < 4 ? a[w & 3] : b[w & 3];
    f[2 * w] = bf16lo(two);
    f[2 * w + 1] = bf16hi(two);
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) f[i] = f[i] == f[i] ? fminf(fmaxf(f[i], -top), top) : 0.f;
}

// Codes and scale bytes are stored apart, so a slot that two rows write may end with one's codes and the other's scale: the
// caller gives every position to one row.
// A wave: the tokens of one row on one page, one head.  Lane (t = lane % 16, g = lane / 16) has values 16g .. 16g + 15 of
// the page's token t.  Row r's pages are the slots from f(r) on, f(r) = q_start[r] / 16 + 2 r: n tokens touch at
// most n / 16 + 2 pages, which end at or before f(r + 1).
__global__ __launch_bounds__(256) void kv8_write_kernel(const Write8Params P) {
  __shared__ __attribute__((aligned(16))) uint8_t turn[4][kHeadTile];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int groups = P.H / 4;
  const int slot = static_cast<int>(blockIdx.x) / groups;
  const int h = (static_cast<int>(blockIdx.x) - slot * groups) * 4 + wave;
  int row, first, n, at;  // the row's tokens first .. first + n - 1, the slot's page of the row
  if (P.q_start == nullptr) {
    const int per = P.bl / kPageSize + 2;
    row = slot / per;
    first = row * P.bl;
    n = P.bl;
    at = slot - row * per;
  } else {
    int base = 0, left = P.rows;  // 64-way search for the last row with f(row) <= slot
    while (left > 1) {
      const int step = (left + 63) / 64;
      const int i = lane * step;
      const bool le = i < left && first_token(P, base + min(i, left - 1)) / kPageSize + 2 * (base + i) <= slot;
      const int to = (max(__popcll(__ballot(le)), 1) - 1) * step;
      base += to;
      left = min(step, left - to);
    }
    row = base;
    first = first_token(P, row);
    n = first_token(P, row + 1) - first;
    at = slot - first / kPageSize - 2 * row;
  }
  if (at < 0 || n <= 0) return;
  const int64_t p0 = P.pos0[row], p_end = p0 + n;
  const int64_t col = (p0 >= 0 ? p0 / kPageSize : -((kPageSize - 1 - p0) / kPageSize)) + at;
  if (col < 0 || col >= P.table_cols || col * kPageSize >= p_end) return;  // nothing there, or behind what the row maps
  const int64_t page = P.table[static_cast<int64_t>(row) * P.table_stride + col];
  if (page < 0 || page >= P.n_pages) return;
  const int t0 = static_cast<int>(max(p0 - col * kPageSize, int64_t{0}));
  const int t1 = static_cast<int>(min(p_end - col * kPageSize, int64_t{kPageSize}));  // the page's tokens [t0, t1)
  const int t = lane & 15, g = lane >> 4;
  const bool mine = t >= t0 && t < t1;
  const int64_t token = first + (col * kPageSize + min(max(t, t0), t1 - 1) - p0);  // others repeat one that is there
  u32x4_t raw[2][2];
#pragma unroll
  for (int pl = 0; pl < 2; ++pl) {
    const uint16_t* x = P.x[pl] + token * P.tok_stride[pl] + h * kHeadDim + 16 * g;
    raw[pl][0] = load16(x);
    raw[pl][1] = load16(x + 8);
  }
#pragma unroll
  for (int pl = 0; pl < 2; ++pl) {
    float f[16];
    finite16(raw[pl][0], raw[pl][1], f);
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(f[i]));
    top = max_xor16_32(top);
    const uint32_t e = static_cast<uint32_t>(max(static_cast<int>(__float_as_uint(top) >> 23) - 6, 1));
    const float inv = __uint_as_float((254u - e) << 23);  // 2^(127 - e), e in [1, 248]
    u32x4_t codes;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint32_t four = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = static_cast<int>(fminf(fmaxf(__builtin_rintf(f[4 * w + i] * inv), -127.f), 127.f));
        four |= (static_cast<uint32_t>(c) & 0xffu) << (8 * i);
      }
      codes[w] = four;
    }
    uint8_t* tile = P.pool + kv8_plane_offset(page, pl, h, P.H);
    if (mine && g == 0) tile[kHeadTile + t] = static_cast<uint8_t>(e);
    if (pl == 0) {
      if (mine) *reinterpret_cast<u32x4_t*>(tile + t * kHeadDim + 16 * g) = codes;
    } else {  // transposed in LDS: lane = head dim
      uint8_t* s = turn[wave];
#pragma unroll
      for (int i = 0; i < 16; ++i) s[(16 * g + i) * kPageSize + t] = static_cast<uint8_t>(codes[i >> 2] >> (8 * (i & 3)));
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      if (t1 - t0 == kPageSize) {
        *reinterpret_cast<u32x4_t*>(tile + lane * kPageSize) = *reinterpret_cast<const u32x4_t*>(s + lane * kPageSize);
      } else {  // the page's other tokens stay as they are
        for (int u = t0; u < t1; ++u) tile[lane * kPageSize + u] = s[lane * kPageSize + u];
      }
    }
  }
}

struct Unpack8Params {
  const uint8_t* pool8;
  int64_t n_pages8;
  const int32_t* table8;
  int stride8, cols8;
  const int32_t* kv_len;
  uint16_t* pool;
  int64_t n_pages;
  const int32_t* table;
  int stride, cols;
  int H;
};

constexpr int kTiles = 8;  // head planes of a workgroup, two at a time

// blockIdx = (eight head planes of a page, page of the row, row): half a workgroup to a plane, eight codes a thread.
__global__ __launch_bounds__(256) void kv8_unpack_kernel(const Unpack8Params P) {
  const int col = blockIdx.y, row = blockIdx.z;
  const int64_t kvl = min(int64_t{P.kv_len[row]}, static_cast<int64_t>(min(P.cols8, P.cols)) * kPageSize);
  if (static_cast<int64_t>(col) * kPageSize >= kvl) return;
  const int64_t from = P.table8[static_cast<int64_t>(row) * P.stride8 + col];
  const int64_t to = P.table[static_cast<int64_t>(row) * P.stride + col];
  if (from < 0 || from >= P.n_pages8 || to < 0 || to >= P.n_pages) return;
  const int i = threadIdx.x & 127;
  u32x2_t codes[kTiles / 2], sc[kTiles / 2];
#pragma unroll
  for (int j = 0; j < kTiles / 2; ++j) {
    const int pt = blockIdx.x * kTiles + 2 * j + (threadIdx.x >> 7);  // plane * H + head, below 2 H: H is a multiple of 4
    const uint8_t* tile = P.pool8 + (from * 2 * P.H + pt) * kTile8;
    codes[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x2_t*>(tile + 8 * i));
    // V: the codes are eight tokens of one head dim; K: eight head dims of token i / 8
    sc[j] = *reinterpret_cast<const u32x2_t*>(tile + kHeadTile + (pt >= P.H ? 8 * (i & 1) : (i >> 3 & 8)));
  }
#pragma unroll
  for (int j = 0; j < kTiles / 2; ++j) {
    const int pt = blockIdx.x * kTiles + 2 * j + (threadIdx.x >> 7);
    const bool is_v = pt >= P.H;
    const int u = i >> 3 & 7;
    const float one = kv8_scale((sc[j][u >> 2] >> (8 * (u & 3))) & 0xffu);
    u32x4_t out;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      float f[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int at = 2 * w + b;
        const float scale = is_v ? kv8_scale((sc[j][at >> 2] >> (8 * (at & 3))) & 0xffu) : one;
        f[b] = static_cast<float>(static_cast<int8_t>(codes[j][at >> 2] >> (8 * (at & 3)))) * scale;
      }
      out[w] = pack_bf16x2(f[0], f[1]);  // exact
    }
    __builtin_nontemporal_store(out, reinterpret_cast<u32x4_t*>(P.pool + (to * 2 * P.H + pt) * kHeadTile + 8 * i));
  }
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace yapd

extern "C" int yapd_kv8_write(const void* k, const void* v, int64_t k_tok_stride, int64_t v_tok_stride, void* kv_pool8,
                              int64_t n_pages, const int32_t* page_table, int table_stride, int table_cols,
                              const int32_t* pos0, const int32_t* q_start, int rows, int n_tokens, int n_heads,
                              void* stream) {
  YAPD_REQUIRE(k && v && kv_pool8 && page_table && pos0, "kv8_write: NULL pointer");
  YAPD_REQUIRE(yapd::al16(k) && yapd::al16(v) && yapd::al16(kv_pool8),
               "kv8_write: k, v and kv_pool8 must be 16-byte aligned");
  YAPD_REQUIRE(rows >= 1 && n_tokens >= 1 && n_pages >= 1, "kv8_write: empty shape");
  YAPD_REQUIRE(n_heads >= 4 && n_heads % 4 == 0 && n_heads <= 1024,
               "kv8_write: n_heads must be a multiple of 4, at most 1024 (got %d)", n_heads);
  YAPD_REQUIRE(k_tok_stride % 8 == 0 && v_tok_stride % 8 == 0 && k_tok_stride >= n_heads * yapd::kHeadDim &&
                   v_tok_stride >= n_heads * yapd::kHeadDim,
               "kv8_write: token strides must be multiples of 8, at least n_heads * 64");
  YAPD_REQUIRE(table_cols >= 1 && table_stride >= table_cols, "kv8_write: bad table shape");
  YAPD_REQUIRE(q_start != nullptr || n_tokens % rows == 0, "kv8_write: without q_start n_tokens must be a multiple of rows");
  const int bl = q_start ? 0 : n_tokens / rows;
  const int64_t slots = q_start ? n_tokens / yapd::kPageSize + 2 * static_cast<int64_t>(rows)
                                : static_cast<int64_t>(rows) * (bl / yapd::kPageSize + 2);
  YAPD_REQUIRE(slots * (n_heads / 4) < (int64_t{1} << 24), "kv8_write: too many tokens for one launch");
  yapd::Write8Params P{{static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v)},
                       {k_tok_stride, v_tok_stride},
                       static_cast<uint8_t*>(kv_pool8), n_pages, page_table, table_stride, table_cols, pos0, q_start,
                       rows, n_tokens, bl, n_heads};
  hipLaunchKernelGGL(yapd::kv8_write_kernel, dim3(static_cast<unsigned>(slots * (n_heads / 4))), dim3(256), 0,
                     static_cast<hipStream_t>(stream), P);
  YAPD_LAUNCH_CHECK("kv8_write_kernel launch");
  return YAPD_OK;
}

extern "C" int yapd_kv8_unpack(const void* kv_pool8, int64_t n_pages8, const int32_t* page_table8, int table8_stride,
                               int table8_cols, const int32_t* kv_len, int rows, int max_kv, int n_heads, void* kv_pool,
                               int64_t n_pages, const int32_t* page_table, int table_stride, int table_cols,
                               void* stream) {
  YAPD_REQUIRE(kv_pool8 && page_table8 && kv_len && kv_pool && page_table, "kv8_unpack: NULL pointer");
  YAPD_REQUIRE(yapd::al16(kv_pool8) && yapd::al16(kv_pool), "kv8_unpack: the pools must be 16-byte aligned");
  YAPD_REQUIRE(rows >= 1 && rows <= 65535 && max_kv >= 1 && n_pages8 >= 1 && n_pages >= 1,
               "kv8_unpack: need 1 <= rows <= 65535, max_kv >= 1 and pages");
  YAPD_REQUIRE(n_heads >= 4 && n_heads % 4 == 0 && n_heads <= 1024,
               "kv8_unpack: n_heads must be a multiple of 4, at most 1024 (got %d)", n_heads);
  YAPD_REQUIRE(table8_cols >= 1 && table8_stride >= table8_cols && table_cols >= 1 && table_stride >= table_cols,
               "kv8_unpack: bad table shape");
  int64_t cols = (static_cast<int64_t>(max_kv) + yapd::kPageSize - 1) / yapd::kPageSize;
  cols = cols < table8_cols ? cols : table8_cols;
  cols = cols < table_cols ? cols : table_cols;
  YAPD_REQUIRE(cols <= 65535 && rows * cols * (n_heads / 4) < (int64_t{1} << 24),
               "kv8_unpack: too many pages for one launch");
  const uintptr_t a = reinterpret_cast<uintptr_t>(kv_pool8), b = reinterpret_cast<uintptr_t>(kv_pool);
  YAPD_REQUIRE(a + static_cast<uintptr_t>(n_pages8) * 2 * n_heads * yapd::kTile8 <= b ||
                   b + static_cast<uintptr_t>(n_pages) * 2 * n_heads * yapd::kHeadTile * 2 <= a,
               "kv8_unpack: the pools overlap");
  yapd::Unpack8Params P{static_cast<const uint8_t*>(kv_pool8), n_pages8, page_table8, table8_stride, table8_cols, kv_len,
                        static_cast<uint16_t*>(kv_pool), n_pages, page_table, table_stride, table_cols, n_heads};
  hipLaunchKernelGGL(yapd::kv8_unpack_kernel, dim3(2 * n_heads / yapd::kTiles, static_cast<unsigned>(cols), rows),
                     dim3(256), 0, static_cast<hipStream_t>(stream), P);
  YAPD_LAUNCH_CHECK("kv8_unpack_kernel launch");
  return YAPD_OK;
}
