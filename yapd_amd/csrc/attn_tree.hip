// Attention for trees of drafted tokens over the paged KV cache, bf16 or 8-bit.
//
// Row r has n <= 64 nodes in the cache's slots ctx .. ctx + n - 1, ctx = kv_len[r] - n.  Node i sees
//   node j       iff bit j of mask_i is set (its ancestors, and itself),
//   key j < ctx  iff j < sinks or j > ctx + depth_i - window, depth_i = the other bits set in mask_i,
//   out = sum_j softmax_j(scale q . k_j) v_j over the keys seen.
// n = 1 is the next token of an ordinary decode.
//
// A wave takes up to 16 NQT nodes of a row, so a key is read once for most trees.  The keys seen
// are a list of chunks (the sinks', then those from the window's begin on), cut into `parts` (workgroups) and each
// part into W runs (waves); runs join in LDS, parts through a workspace and a second launch.  S^T = K Q^T and
// O^T += V^T P^T on v_mfma_f32_16x16x32_bf16, every lane owning one query and kKeys consecutive keys of a chunk:
//   bf16: chunks of 32 keys (two pages), 8 keys a lane;
//   8 bits: chunks of 64 keys (four pages), lane group g owning page g: 16 bytes are 16 head dims of a key, 16
//     tokens of a head dim or 16 tokens' scales, so every load is 16 bytes.  Which head dims a step of the product
//     with K takes is free as long as Q's fragments take the same.  Codes become bf16 (exact); K's scales
//     multiply the scores, V's the weights before they are rounded to bf16.
//
// Single tokens and long rows are bound by memory: 256 ragged rows of 60 to 4000 keys x 16 heads at 8 bits 202 us, 5.4
// TB/s (half of the vector unit's cycles are free; in bf16 the same takes 331); three rows of 13 nodes on 20000 to 30000 keys
// in bf16 57 us, 5.4 TB/s, 5 of it the join.  Trees at 8 bits are not: 130 rows of 1 to 64 nodes on up to 2033 keys
// 127 us, 3.2 TB/s.  A chunk costs a wave 230 vector instructions and a tile of 16 queries 110 more with 16 exponentials, at
// two waves a SIMD (223 registers) their chains are not hidden behind each other.  Measured and left out there (against
// 138): K's product on v_mfma_i32_16x16x64_i8 with Q in two bytes (no conversion of K; 184 registers) 145 us with one set
// of loads and 133 with two, but Q would be rounded; three waves a SIMD 208 (spills); 512 threads a head 179.
#include <algorithm>
#include <type_traits>

#include "attn_tile.h"
#include "common.h"
#include "kv_layout.h"

namespace yapd {
namespace {

constexpr int kCap = 1 << 30;  // window and sinks are held to this: positions minus window stay inside int32
constexpr int kMaxNodes = 64;  // bits of a mask

struct TreeParams {
  const uint16_t* q;  // token t, head h at t * q_stride + h * 64
  int64_t q_stride;
  const void* pool;
  int64_t n_pages;
  const int32_t* table;
  int table_stride, table_cols;
  const int32_t* kv_len;
  const int32_t* q_start;  // [rows + 1], or NULL: row r's nodes are r * max_q ..
  const int64_t* mask;     // [n_q]
  int rows, max_q, n_q, H;
  int window, sinks;
  int parts;
  float class_scale;  // of a row's cost (row_by_cost); 0: rows are taken as they come
  float* part_o;   // [parts, n_q, H, 64]
  float* part_ml;  // [parts, n_q, H, 2]
  float scale_log2;
  uint16_t* out;  // [n_q, H, 64]
};

// The nodes of a row that are computed: rows qs .. qs + qc - 1 of q and out.  false: it has none.
struct Tree {
  int qs, qc, n, kvl, ctx;
};
__device__ __forceinline__ bool find_tree(const TreeParams& P, int row, Tree& t) {
  t.qs = row * P.max_q;
  t.n = P.max_q;
  if (P.q_start != nullptr) {
    t.qs = min(max(P.q_start[row], 0), P.n_q);
    t.n = min(max(P.q_start[row + 1], 0), P.n_q) - t.qs;
  }
  t.qc = min(t.n, P.max_q);
  t.kvl = min(max(P.kv_len[row], 0), P.table_cols * kPageSize);
  t.ctx = t.kvl - t.n;
  return t.qc > 0;
}

constexpr int kSorted = 256;  // rows that are ordered by cost, four a lane; more of them were not measured
constexpr int kClasses = 64;

// Row `slot` by cost, the costliest first: the keys that it sees times what a chunk of them costs it.  A launch of more
// workgroups than the chip holds ends when the last one started does, and that one should be small.  Rows of one of 64
// classes stay as they come.  Every wave finds its row by itself, by halving the classes.
// us as they come, and so: 16 heads, 256 single tokens on 60 to 4000 keys at 8 bits 213, 202, bf16 352, 331; 130 trees of 1 to 64
// nodes 136, 127; 64 of 64 nodes on 200 to 1500 keys 66, 55, bf16 89, 78; 128 of them 116, 108, bf16 163, 146; equal rows lose
// up to 0.5.
template <int NQT>
__device__ __forceinline__ int row_by_cost(const TreeParams& P, int slot, int lane) {
  int cls[kSorted / 64];
#pragma unroll
  for (int j = 0; j < kSorted / 64; ++j) {
    const int r = lane + 64 * j;
    cls[j] = -1;
    if (r >= P.rows) continue;
    int n = P.max_q;
    if (P.q_start != nullptr) n = min(max(P.q_start[r + 1], 0), P.n_q) - min(max(P.q_start[r], 0), P.n_q);
    const int kvl = min(max(P.kv_len[r], 0), P.table_cols * kPageSize);
    // of two query tiles a chunk takes 230 instructions and 110 a tile; of more than 32 nodes half the waves go over it
    // (at 8 bits; a bf16 chunk converts nothing and takes fewer, and is ordered by the same numbers)
    const float each = NQT == 1 ? 1.f : n > 32 ? 900.f : n > 16 ? 450.f : 340.f;
    const float keys = fminf(static_cast<float>(kvl), static_cast<float>(P.window) + static_cast<float>(P.sinks) + n);
    cls[j] = n > 0 ? static_cast<int>(fminf(keys * each * P.class_scale, kClasses - 1.f)) : 0;
  }
  int lo = 0, hi = kClasses, above = 0;  // more than `slot` rows are in classes from lo on, `above` of them from hi on
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    int c = 0;
#pragma unroll
    for (int j = 0; j < kSorted / 64; ++j) c += static_cast<int>(__popcll(__ballot(cls[j] >= mid)));
    if (c > slot) {
      lo = mid;
    } else {
      hi = mid;
      above = c;
    }
  }
  int k = slot - above, row = 0;  // the k-th row of class lo
#pragma unroll
  for (int j = 0; j < kSorted / 64; ++j) {
    const uint64_t in = __ballot(cls[j] == lo);
    const int c = static_cast<int>(__popcll(in));
    const int before = __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(in >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(in), 0));
    const uint64_t at = __ballot(cls[j] == lo && before == k);
    if (k >= 0 && k < c) row = 64 * j + __ffsll(static_cast<unsigned long long>(at)) - 1;
    k -= c;
  }
  return __builtin_amdgcn_readfirstlane(row);
}

// Bits of the keys from `shift` positions behind the tree's first node on (before it where negative: the
// context's bits are set, down to 31 positions).
__device__ __forceinline__ uint32_t bits_from(uint64_t mask, int shift) {
  if (shift >= 0) return shift < 64 ? static_cast<uint32_t>(mask >> shift) : 0u;
  if (shift <= -32) return 0xffffffffu;
  return static_cast<uint32_t>(mask << -shift) | ((1u << -shift) - 1u);
}

// The row's page ids, 64 at a time: lane i holds the page of table column base + i (clamped).
struct TreePages {
  const int32_t* tab;
  int last_page, max_page, lane, base, v;
  __device__ __forceinline__ TreePages(const TreeParams& P, const Tree& t, int row, int first, int lane_)
      : tab(P.table + static_cast<int64_t>(row) * P.table_stride),
        last_page(max((t.kvl + kPageSize - 1) / kPageSize - 1, 0)),
        max_page(static_cast<int>(min(P.n_pages - 1, int64_t{0x7fffffff}))), lane(lane_) {
    load(first);
  }
  __device__ __forceinline__ void load(int b) {
    base = b;
    v = min(max(tab[min(base + lane, last_page)], 0), max_page);  // a bad table entry cannot fault
    asm volatile("" : "+v"(v));  // complete here: later uses wait on no load
  }
  // pages [pi, pi + n) are held, pi never falling and a multiple of n
  __device__ __forceinline__ void hold(int pi, int n) {
    if (pi + n - base > 64) load(pi);  // uniform
  }
  __device__ __forceinline__ int uniform(int pi) const { return __builtin_amdgcn_readlane(v, pi - base); }
  __device__ __forceinline__ int each(int pi) const { return __builtin_amdgcn_ds_bpermute((pi - base) << 2, v); }
};

// Four signed bytes as bf16.
__device__ __forceinline__ u32x2_t bytes_to_bf16(uint32_t four) {
  const float a = static_cast<float>(static_cast<int8_t>(four)), b = static_cast<float>(static_cast<int8_t>(four >> 8));
  const float c = static_cast<float>(static_cast<int8_t>(four >> 16)), d = static_cast<float>(static_cast<int8_t>(four >> 24));
  // the upper halves hold every bit of an integer of 8 bits
  return u32x2_t{__builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u),
                 __builtin_amdgcn_perm(__float_as_uint(d), __float_as_uint(c), 0x07060302u)};
}

// The exponent that scale byte i of the four in a word stands for.
__device__ __forceinline__ int exponent_of(uint32_t word, int i) { return static_cast<int>(word >> (8 * i) & 0xffu) - 127; }

// A product that is rounded wherever it is used: never fused into a sum.
__device__ __forceinline__ float rounded_product(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

// A chunk's loads, as they come.
template <bool k8>
struct Chunk;

template <>
struct Chunk<false> {
  static constexpr int kKeys = 8, kSize = 32;
  u32x4_t kf[2][2], vf[4];
  __device__ __forceinline__ void load(const TreeParams& P, TreePages& pages, int k0, int h, int g, int n) {
    const int pi = k0 / kPageSize;
    pages.hold(pi, 2);
    const int64_t pg0 = pages.uniform(pi), pg1 = pages.uniform(pi + 1);
    const uint16_t* pool = static_cast<const uint16_t*>(P.pool);
    // Row n of S^T tile i is key 8 (n / 4) + 4 i + n % 4, so that lane group g ends up with keys 8g .. 8g + 7.
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int key = 8 * (n >> 2) + 4 * i + (n & 3);
      const uint16_t* kp = pool + k_offset(key < kPageSize ? pg0 : pg1, h, P.H, key & (kPageSize - 1), 8 * g);
      kf[i][0] = load16_stream(kp);
      kf[i][1] = load16_stream(kp + 32);
    }
    const uint16_t* vp = pool + v_offset(g < 2 ? pg0 : pg1, h, P.H, 8 * (g & 1), n);
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) vf[mt] = load16_stream(vp + 16 * mt * kPageSize);
  }
  // seen: bit i set where some node sees this lane's key i; V of the others is cleared, so 0 * V is never NaN
  __device__ __forceinline__ void clear(uint32_t seen) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t keep = (seen >> (2 * w) & 1u ? 0x0000ffffu : 0u) | (seen >> (2 * w + 1) & 1u ? 0xffff0000u : 0u);
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) vf[mt][w] &= keep;
    }
  }
  static __device__ __forceinline__ int q_dim(int s, int g) { return 32 * s + 8 * g; }
};

template <>
struct Chunk<true> {
  static constexpr int kKeys = 16, kSize = 64;
  u32x4_t kf[4], vf[4], ks, vs;
  const uint8_t *kp, *tile;
  static __device__ __forceinline__ u32x4_t load16b(const uint8_t* p) {
    return *reinterpret_cast<const u32x4_t*>(p);  // cached: planes of 1040 bytes share lines with the next head's
  }
  __device__ __forceinline__ void load_k(const TreeParams& P, TreePages& pages, int k0, int h, int g, int n) {
    const int pi = k0 / kPageSize;
    pages.hold(pi, 4);
    const uint8_t* pool = static_cast<const uint8_t*>(P.pool);
    // Row n of S^T tile i is token 4 i + n % 4 of page n / 4, so that lane group g ends up with page g's tokens.
    kp = pool + kv8_plane_offset(pages.each(pi + (n >> 2)), 0, h, P.H) + (n & 3) * kHeadDim + 16 * g;
    tile = pool + kv8_plane_offset(pages.each(pi + g), 0, h, P.H);
    ks = load16b(tile + kHeadTile);
#pragma unroll
    for (int i = 0; i < 4; ++i) kf[i] = load16b(kp + 4 * i * kHeadDim);
  }
  __device__ __forceinline__ void load_v(const TreeParams& P, int n) {
    const uint8_t* vp = tile + static_cast<int64_t>(P.H) * kTile8;
    vs = load16b(vp + kHeadTile);
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) vf[mt] = load16b(vp + (16 * mt + n) * kPageSize);
  }
  static __device__ __forceinline__ int q_dim(int s, int g) { return 16 * g + 8 * s; }
};

// 16 codes as the operands of two products.
__device__ __forceinline__ void codes_to_bf16(const u32x4_t& c, bf16x8_t (&out)[2]) {
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const u32x2_t a = bytes_to_bf16(c[2 * s]), b = bytes_to_bf16(c[2 * s + 1]);
    out[s] = as_bf16x8(u32x4_t{a[0], a[1], b[0], b[1]});
  }
}

constexpr int kWaveFloats = 4 * 64 * 4;  // a wave's O^T tile in LDS: fragment mt of lane l at (mt * 64 + l) * 4

// W waves a head.  They take the chunks in runs; of rows with more than 16 NQT nodes every other one takes the
// nodes from 16 NQT on (the host gives those two waves at least), and two waves have each run.
template <bool k8, int NQT, int W>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(NQT > 1 ? 2 : k8 ? 4 : 3))) void attn_tree_kernel(const TreeParams P) {
  using C = Chunk<k8>;
  constexpr int HPW = 4 / W;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int w = wave % W, hsub = wave / W;
  const int groups = P.H / HPW;
  const int item = static_cast<int>(blockIdx.x) / groups;
  const int h = (static_cast<int>(blockIdx.x) - item * groups) * HPW + hsub;
  int row = item / P.parts;
  const int part = item - row * P.parts;
  if (P.class_scale > 0.f) row = row_by_cost<NQT>(P, row, lane);
  Tree t;
  if (!find_tree(P, row, t)) return;  // the whole workgroup
  const int g = lane >> 4, n = lane & 15;
  const int H = P.H;
  const bool halves = W > 1 && t.qc > 16 * NQT;
  const int half = halves ? w & 1 : 0, runs = halves ? W / 2 : W, run_w = halves ? w >> 1 : w;
  const int q0 = half * 16 * NQT;  // this wave's first node

  // Q^T fragments (B operand) and the masks of this lane's queries q0 + qt * 16 + n
  u32x4_t qraw[NQT][2];
  uint64_t mask[NQT];
#pragma unroll
  for (int qt = 0; qt < NQT; ++qt) {
    const int q = min(q0 + qt * 16 + n, t.qc - 1);
#pragma unroll
    for (int s = 0; s < 2; ++s)
      qraw[qt][s] = load16(P.q + (t.qs + q) * P.q_stride + h * kHeadDim + C::q_dim(s, g));
    mask[qt] = static_cast<uint64_t>(P.mask[t.qs + q]);
  }
  const uint64_t nodes = t.n >= 64 ? ~uint64_t{0} : (uint64_t{1} << t.n) - 1;
  int q_lo[NQT];  // context keys from here on are in the node's window
  int lo = 0, all_lo = -kCap;  // the first and the last window's begin
#pragma unroll
  for (int qt = 0; qt < NQT; ++qt) q_lo[qt] = -kCap;
  if (P.window < kCap) {
    lo = 0x7fffffff;
#pragma unroll
    for (int qt = 0; qt < NQT; ++qt) {
      const int q = min(q0 + qt * 16 + n, t.qc - 1);  // lanes without a node repeat the last
      // at most ctx: the window bounds the context, and a row's first nodes may be deeper than it
      const int depth = static_cast<int>(__popcll(mask[qt] & nodes & ~(uint64_t{1} << q)));
      q_lo[qt] = t.ctx + min(depth - P.window + 1, 0);
      lo = min(lo, q_lo[qt]);
      all_lo = max(all_lo, q_lo[qt]);
    }
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
      lo = min(lo, __shfl_xor(lo, d));
      all_lo = max(all_lo, __shfl_xor(all_lo, d));
    }
    lo = max(__builtin_amdgcn_readfirstlane(lo), 0);
    all_lo = __builtin_amdgcn_readfirstlane(all_lo);
  }

  // the list of chunks: entry c is chunk c below n_sink, chunk skip + c from there on; keys seen are below hi
  const int hi = t.kvl;
  const int cb = min(lo, hi) / C::kSize, ce = (hi + C::kSize - 1) / C::kSize;
  const int n_sink = min((min(P.sinks, hi) + C::kSize - 1) / C::kSize, cb);
  const int skip = cb - n_sink, n_chunks = n_sink + ce - cb;
  const auto chunk = [&](int c) { return c < n_sink ? c : c + skip; };

  f32x4_t o[NQT][4];
  float m[NQT], mref[NQT], l[NQT];
#pragma unroll
  for (int qt = 0; qt < NQT; ++qt) {
    m[qt] = -INFINITY;
    mref[qt] = l[qt] = 0.f;
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) o[qt][mt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  // this wave's run of the list
  const int all_runs = P.parts * runs, run = part * runs + run_w;
  const int each_run = n_chunks / all_runs, more_runs = n_chunks - each_run * all_runs;  // the first ones have one more
  const int c0 = each_run * run + min(run, more_runs), c1 = c0 + each_run + (run < more_runs ? 1 : 0);
  bf16x8_t qf[NQT][2];
  const auto take_queries = [&] {
#pragma unroll
    for (int qt = 0; qt < NQT; ++qt) {
      const bool live = q0 + qt * 16 + n < t.qc;
#pragma unroll
      for (int s = 0; s < 2; ++s) qf[qt][s] = as_bf16x8(live ? qraw[qt][s] : u32x4_t{0u, 0u, 0u, 0u});
      mask[qt] = live ? mask[qt] & nodes : 0;
    }
  };
  if (c0 < c1) {
    TreePages pages(P, t, row, chunk(c0) * (C::kSize / kPageSize), lane);
    const auto is_edge = [&](int k0) { return k0 + C::kSize > t.ctx || (k0 < all_lo && k0 + C::kSize > P.sinks); };
    // The scores of tile qt become weights, against the maximum as it is now.  Exponents are taken as s scale - mref, mref
    // the maximum times scale, rounded once and the same wherever it is used; the old sums are rescaled only where some
    // query's maximum has moved, by the factor between its references (exactly 1 for the others).
    const auto weights = [&](int qt, int key0, bool edge, float (&sv)[C::kKeys]) {
      if (edge) {
        const uint32_t bits = bits_from(mask[qt], key0 - t.ctx);
#pragma unroll
        for (int i = 0; i < C::kKeys; ++i)
          sv[i] = (bits >> i & 1u) && (key0 + i >= q_lo[qt] || key0 + i < P.sinks) ? sv[i] : -INFINITY;
      }
      float cm = sv[0];
#pragma unroll
      for (int i = 1; i < C::kKeys; ++i) cm = fmaxf(cm, sv[i]);
      cm = max_xor16_32(cm);
      if (__any(cm > m[qt])) {
        m[qt] = fmaxf(m[qt], cm);
        // no key seen yet: exponents against 0 give weights of 0 instead of NaN
        const float to = m[qt] == -INFINITY ? 0.f : rounded_product(m[qt], P.scale_log2);
        const float alpha = __builtin_amdgcn_exp2f(fminf(mref[qt] - to, 0.f));  // a first maximum's is of sums that are 0
        mref[qt] = to;
        l[qt] *= alpha;
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) o[qt][mt] *= alpha;
      }
      float ps = 0.f;
#pragma unroll
      for (int i = 0; i < C::kKeys; ++i) {
        sv[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[i], P.scale_log2, -mref[qt]));
        ps += sv[i];
      }
      l[qt] += ps;
    };
    if constexpr (k8) {
      C x;
      x.load_k(P, pages, chunk(c0) * C::kSize, h, g, n);
      x.load_v(P, n);
      take_queries();
      // A chunk's codes are operands before its products begin, so the registers they came in take the next chunk's.
      auto step = [&](int c, auto more) {
        const int k0 = chunk(c) * C::kSize, key0 = k0 + C::kKeys * g;
        const bool edge = is_edge(k0);  // uniform
        bf16x8_t kb[4][2], vb[4][2];
        const u32x4_t ks = x.ks, vs = x.vs;
#pragma unroll
        for (int i = 0; i < 4; ++i) codes_to_bf16(x.kf[i], kb[i]);
        u32x4_t pw[NQT][2];
#pragma unroll
        for (int qt = 0; qt < NQT; ++qt) {
          if (qt > 0 && q0 + qt * 16 >= t.qc) break;  // uniform
          float sv[16];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            f32x4_t s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kb[i][0], qf[qt][0], f32x4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kb[i][1], qf[qt][1], s, 0, 0, 0);
            // s[j] = q n . codes of key key0 + 4 i + j
#pragma unroll
            for (int j = 0; j < 4; ++j) sv[4 * i + j] = __builtin_ldexpf(s[j], exponent_of(ks[i], j));
          }
          weights(qt, key0, edge, sv);
          // The weights times V's scales in bf16, the operand type of the product with V: each is off by at most 2^-8 of
          // itself.  A key that a query does not see has a weight of 0 there whatever its scale byte is.
#pragma unroll
          for (int i = 0; i < 8; ++i)
            pw[qt][i >> 2][i & 3] = pack_bf16x2(__builtin_ldexpf(sv[2 * i], exponent_of(vs[i >> 1], 2 * i & 3)),
                                                __builtin_ldexpf(sv[2 * i + 1], exponent_of(vs[i >> 1], (2 * i + 1) & 3)));
        }
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) codes_to_bf16(x.vf[mt], vb[mt]);
        if constexpr (more.value) {
          x.load_k(P, pages, chunk(c + 1) * C::kSize, h, g, n);
          x.load_v(P, n);
        }
#pragma unroll
        for (int qt = 0; qt < NQT; ++qt) {
          if (qt > 0 && q0 + qt * 16 >= t.qc) break;
#pragma unroll
          for (int mt = 0; mt < 4; ++mt)
#pragma unroll
            for (int st = 0; st < 2; ++st)
              o[qt][mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vb[mt][st], as_bf16x8(pw[qt][st]), o[qt][mt], 0, 0, 0);
        }
      };
      int c = c0;
      for (; c + 1 < c1; ++c) step(c, std::true_type{});
      step(c, std::false_type{});
    } else {
      C a, b;
      a.load(P, pages, chunk(c0) * C::kSize, h, g, n);
      take_queries();
      uint32_t any_lo = 0, any_hi = 0;  // nodes that some node of the wave sees
#pragma unroll
      for (int qt = 0; qt < NQT; ++qt) {
        any_lo |= static_cast<uint32_t>(mask[qt]);
        any_hi |= static_cast<uint32_t>(mask[qt] >> 32);
      }
#pragma unroll
      for (int d = 1; d < 16; d <<= 1) {
        any_lo |= __shfl_xor(any_lo, d);
        any_hi |= __shfl_xor(any_hi, d);
      }
      const uint64_t any = static_cast<uint64_t>(any_hi) << 32 | any_lo;
      // bit i: some node of the wave sees this lane's key i of the chunk
      const auto seen_of = [&](int key0) {
        uint32_t seen = bits_from(any, key0 - t.ctx);
#pragma unroll
        for (int i = 0; i < C::kKeys; ++i)
          if (key0 + i < lo && key0 + i >= P.sinks) seen &= ~(1u << i);
        return seen;
      };
      auto step = [&](int c, C& x) {
        const int k0 = chunk(c) * C::kSize, key0 = k0 + C::kKeys * g;
        const bool edge = is_edge(k0);  // uniform
        if (edge) x.clear(seen_of(key0));
#pragma unroll
        for (int qt = 0; qt < NQT; ++qt) {
          if (qt > 0 && q0 + qt * 16 >= t.qc) break;  // uniform
          float sv[8];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            f32x4_t s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(x.kf[i][0]), qf[qt][0],
                                                                f32x4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(x.kf[i][1]), qf[qt][1], s, 0, 0, 0);
#pragma unroll
            for (int j = 0; j < 4; ++j) sv[4 * i + j] = s[j];
          }
          weights(qt, key0, edge, sv);
          // P in bf16, the operand type of the product with V: each weight is off by at most 2^-8 of itself
          u32x4_t pw;
#pragma unroll
          for (int i = 0; i < 4; ++i) pw[i] = pack_bf16x2(sv[2 * i], sv[2 * i + 1]);
#pragma unroll
          for (int mt = 0; mt < 4; ++mt)
            o[qt][mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(x.vf[mt]), as_bf16x8(pw), o[qt][mt], 0, 0, 0);
        }
      };
      // chunk c + 1 is on its way while chunk c is multiplied
      int c = c0;
      for (; c + 2 < c1; c += 2) {
        b.load(P, pages, chunk(c + 1) * C::kSize, h, g, n);
        step(c, a);
        a.load(P, pages, chunk(c + 2) * C::kSize, h, g, n);
        step(c + 1, b);
      }
      if (c + 1 < c1) {
        b.load(P, pages, chunk(c + 1) * C::kSize, h, g, n);
        step(c, a);
        step(c + 1, b);
      } else {
        step(c, a);
      }
    }
  }

  // o[qt][mt][j] = O^T[hd = 16mt + 4g + j][q = q0 + qt*16 + n].  With several runs: their
  // O^T, m and l go to LDS, and run r's wave joins the fragments mt = r, r + runs, ..
  __shared__ __attribute__((aligned(16))) float s_o[W > 1 ? 4 * kWaveFloats : 4];
  __shared__ float s_ml[W > 1 ? 4 * 32 : 2];
#pragma unroll
  for (int qt = 0; qt < NQT; ++qt) {
    if (qt > 0 && qt * 16 >= t.qc) break;  // uniform in the workgroup
    const int q = q0 + qt * 16 + n;
    const int64_t token = t.qs + q;
    float M = m[qt] == -INFINITY ? m[qt] : mref[qt], L = sum_xor16_32(l[qt]);
    auto finish = [&](int mt, f32x4_t acc) {
      if (q >= t.qc) return;
      const int64_t at = (token * H + h) * kHeadDim + 16 * mt + 4 * g;
      if (P.parts == 1) {
        // L = 0 only for a node that sees no key: zeros, not NaN
        const float inv = L == 0.f ? 0.f : 1.f / L;
        u32x2_t w2;
        w2[0] = pack_bf16x2(acc[0] * inv, acc[1] * inv);
        w2[1] = pack_bf16x2(acc[2] * inv, acc[3] * inv);
        *reinterpret_cast<u32x2_t*>(P.out + at) = w2;
      } else {
        *reinterpret_cast<f32x4_t*>(P.part_o + static_cast<int64_t>(part) * P.n_q * H * kHeadDim + at) = acc;
        if (mt == 0 && g == 0) {
          float* ml = P.part_ml + (static_cast<int64_t>(part) * P.n_q * H + token * H + h) * 2;
          ml[0] = M;
          ml[1] = L;
        }
      }
    };
    if constexpr (W == 1) {
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) finish(mt, o[qt][mt]);
    } else {
      if (qt > 0) __syncthreads();  // the previous tile has been read
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
        *reinterpret_cast<f32x4_t*>(s_o + wave * kWaveFloats + (mt * 64 + lane) * 4) = o[qt][mt];
      if (g == 0) {
        s_ml[wave * 32 + n] = M;
        s_ml[wave * 32 + 16 + n] = L;
      }
      __syncthreads();
      // the waves whose queries these are: hsub * W + half, every (halves ? 2 : 1)-th
      const int w0 = hsub * W + half, stride = halves ? 2 : 1;
      M = -INFINITY;
      for (int r = 0; r < runs; ++r) M = fmaxf(M, s_ml[(w0 + r * stride) * 32 + n]);
      const float mref = M == -INFINITY ? 0.f : M;
      float sc[W];
      L = 0.f;
#pragma unroll
      for (int r = 0; r < W; ++r) {
        if (r >= runs) break;
        const float* ml = s_ml + (w0 + r * stride) * 32 + n;
        sc[r] = __builtin_amdgcn_exp2f(ml[0] - mref);
        L += sc[r] * ml[16];
      }
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        if ((mt & (runs - 1)) != run_w) continue;  // runs is 1, 2 or 4
        f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int r = 0; r < W; ++r) {
          if (r >= runs) break;
          acc += sc[r] * *reinterpret_cast<const f32x4_t*>(s_o + (w0 + r * stride) * kWaveFloats + (mt * 64 + lane) * 4);
        }
        finish(mt, acc);
      }
    }
  }
}

// Joins the parts of every node: thread (node, head, 4 head-dim values).  Eight parts' values are requested
// before the first is used, so up to eight parts cost one memory latency: what bounds it.
__global__ __launch_bounds__(256) void attn_tree_join_kernel(const TreeParams P) {
  constexpr int kAtOnce = 8;
  const int lane = threadIdx.x & 63;
  // there are parts only where (node, head) pairs are few: they fit 32 bits
  const uint32_t pair = blockIdx.x * 16 + (threadIdx.x >> 4);
  const uint32_t row_q = pair / static_cast<uint32_t>(P.H);
  const int h = static_cast<int>(pair - row_q * P.H);
  const int r = static_cast<int>(row_q / P.max_q), i = static_cast<int>(row_q - static_cast<uint32_t>(r) * P.max_q);
  if (r >= P.rows) return;
  Tree t;
  if (!find_tree(P, r, t) || i >= t.qc) return;
  const int64_t step = static_cast<int64_t>(P.n_q) * P.H;
  const int64_t at = static_cast<int64_t>(t.qs + i) * P.H + h;
  float M = -INFINITY, L = 0.f;
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < P.parts; s0 += kAtOnce) {
    float2 ml[kAtOnce];
    f32x4_t po[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      const int64_t from = min(s0 + j, P.parts - 1) * step + at;
      ml[j] = *reinterpret_cast<const float2*>(P.part_ml + from * 2);
      po[j] = *reinterpret_cast<const f32x4_t*>(P.part_o + from * kHeadDim + (lane & 15) * 4);
    }
    float mn = M;
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) mn = fmaxf(mn, ml[j].x);  // the last part's again past the end
    const float mref = mn == -INFINITY ? 0.f : mn;
    const float alpha = __builtin_amdgcn_exp2f(M - mref);
    M = mn;
    L *= alpha;
    acc *= alpha;
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      if (s0 + j >= P.parts) break;
      const float w = __builtin_amdgcn_exp2f(ml[j].x - mref);
      L += w * ml[j].y;
      acc += w * po[j];
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  u32x2_t w2;
  w2[0] = pack_bf16x2(acc[0] * inv, acc[1] * inv);
  w2[1] = pack_bf16x2(acc[2] * inv, acc[3] * inv);
  *reinterpret_cast<u32x2_t*>(P.out + at * kHeadDim + (lane & 15) * 4) = w2;
}

// How a call is cut: nqt query tiles of 16 a wave, w waves a head, parts.
struct Cut {
  int nqt, w, parts;
};

// Waves to a head's chunks: four where each has something to do, because four waves on one row's keys end together and
// leave less of a tail than one wave on each of four rows.  us a call with 1, 2 and 4 waves a head, 16 heads:
//   one token, 8 bits: one row of 1500 keys 29.0, 17.2, 8.5 (cut into parts); 64 ragged rows of 60 to 2000 keys 51.0,
//   37.5, 36.7; 256 of them 136, 120, 114; 256 of 60 to 4000 266, 235, 217; but 256 rows of 350 keys 36.3, 38.0, 41.4, of 90
//   14.2, 16.3, 22.3, of 15 8.2, 12.2, 19.0.  24 nodes: 16 rows of 200 to 1500 44, 26.6, 17.0; 128 of them 70.6, 66.5, 68.3;
//   128 of 350 26.6, 32.3, 38.0.
// So six chunks a wave where the pairs fill the chip with one wave each, two where they do not.
// Parts: as many as bring the workgroups to 512 (to 256 where a wave has two query tiles and so fewer fit a CU), of at least
// four chunks.  One part and as cut here: one token on 1500 keys 13.4, 8.5; eight rows of 60 to 2000 16.9, 11.9;
// three rows of 13 nodes on 30000 keys 197, 59; four rows of 24 nodes on 1500 keys 15.3, 13.3.
constexpr int64_t kFull = 1024;  // (row, head) pairs that fill the chip with a wave each

Cut cut_of(int rows, int max_q, int n_heads, int window, int sinks, int max_kv, int bits) {
  Cut c;
  c.nqt = max_q <= 16 ? 1 : 2;
  const int64_t keys = std::min<int64_t>(max_kv, static_cast<int64_t>(window) + sinks + max_q);
  const int size = bits == 8 ? 64 : 32;
  const int64_t chunks = (keys + size - 1) / size;
  const int64_t pairs = static_cast<int64_t>(rows) * n_heads;
  const int64_t few = pairs >= kFull ? 6 : 2;  // chunks a wave
  c.w = chunks >= 4 * few ? 4 : chunks >= 2 * few ? 2 : 1;
  if (max_q > 32) c.w = std::max(c.w, 2);
  c.parts = 1;
  const int64_t wanted = c.nqt == 1 ? 512 : 256;
  if (c.w == 4) c.parts = static_cast<int>(std::max<int64_t>(1, std::min(wanted / pairs, chunks / 4)));
  return c;
}

template <bool k8, int NQT>
void launch_tiles(const TreeParams& P, const Cut& c, hipStream_t st) {
  const unsigned grid = static_cast<unsigned>(static_cast<int64_t>(P.rows) * P.parts * (P.H / (4 / c.w)));
  if (c.w == 4)
    hipLaunchKernelGGL((attn_tree_kernel<k8, NQT, 4>), dim3(grid), dim3(256), 0, st, P);
  else if (c.w == 2)
    hipLaunchKernelGGL((attn_tree_kernel<k8, NQT, 2>), dim3(grid), dim3(256), 0, st, P);
  else
    hipLaunchKernelGGL((attn_tree_kernel<k8, NQT, 1>), dim3(grid), dim3(256), 0, st, P);
}

template <bool k8>
void launch(const TreeParams& P, const Cut& c, hipStream_t st) {
  if (c.nqt == 1)
    launch_tiles<k8, 1>(P, c, st);
  else
    launch_tiles<k8, 2>(P, c, st);
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Whether any of n blocks of `bytes`, `pitch` >= bytes apart from a on, shares a byte with [b, b + b_bytes).
bool overlap(const void* a, int64_t n, int64_t pitch, int64_t bytes, const void* b, int64_t b_bytes) {
  const int64_t from = static_cast<int64_t>(reinterpret_cast<uintptr_t>(b)) - static_cast<int64_t>(reinterpret_cast<uintptr_t>(a));
  const int64_t first = from < bytes ? 0 : (from - bytes) / pitch + 1;  // the first block that ends behind b
  return first < n && first * pitch < from + b_bytes;
}

// packed: max_q is only a bound of the rows' nodes, which does not bound the window
int tree_checks(int rows, int max_q, int n_q, int packed, int n_heads, int window, int sinks, int max_kv, int bits) {
  YAPD_REQUIRE(bits == 8 || bits == 16, "attn_tree: bits must be 8 or 16 (got %d)", bits);
  YAPD_REQUIRE(rows >= 1 && max_q >= 1 && n_q >= 1, "attn_tree: need rows, max_q and n_q >= 1 (got %d, %d, %d)", rows,
               max_q, n_q);
  YAPD_REQUIRE(max_q <= kMaxNodes, "attn_tree: a tree has at most 64 nodes (got max_q = %d)", max_q);
  YAPD_REQUIRE(n_heads >= 4 && n_heads % 4 == 0 && n_heads <= 1024,
               "attn_tree: n_heads must be a multiple of 4, at most 1024 (got %d)", n_heads);
  YAPD_REQUIRE(window >= (packed ? 1 : max_q) && sinks >= 0, "attn_tree: need window >= %s and sinks >= 0 (got %d, %d)",
               packed ? "1" : "max_q", window, sinks);
  YAPD_REQUIRE(max_kv >= 1, "attn_tree: max_kv must be >= 1 (got %d)", max_kv);
  return YAPD_OK;
}

}  // namespace
}  // namespace yapd

extern "C" int64_t yapd_attn_tree_workspace(int rows, int max_q, int n_q, int n_heads, int window, int sinks, int max_kv,
                                            int bits) {
  if (yapd::tree_checks(rows, max_q, n_q, 0, n_heads, window, sinks, max_kv, bits) != YAPD_OK) return -1;
  const yapd::Cut c = yapd::cut_of(rows, max_q, n_heads, window, sinks, max_kv, bits);
  return c.parts == 1 ? 0 : static_cast<int64_t>(c.parts) * n_q * n_heads * (yapd::kHeadDim + 2);
}

extern "C" int yapd_attn_tree(const void* q, int64_t q_tok_stride, const void* kv_pool, int bits, int64_t n_pages,
                              const int32_t* page_table, int table_stride, int table_cols, const int32_t* kv_len,
                              const int32_t* q_start, const int64_t* mask, int rows, int max_q, int n_q, int n_heads,
                              int window, int sinks, int max_kv, float scale, float* workspace, int64_t workspace_floats,
                              void* out, void* stream) {
  YAPD_REQUIRE(q && kv_pool && page_table && kv_len && mask && out, "attn_tree: NULL pointer");
  if (int rc = yapd::tree_checks(rows, max_q, n_q, q_start != nullptr, n_heads, window, sinks, max_kv, bits)) return rc;
  YAPD_REQUIRE(yapd::al16(q) && yapd::al16(kv_pool) && yapd::al16(out),
               "attn_tree: q, kv_pool and out must be 16-byte aligned");
  YAPD_REQUIRE(q_tok_stride >= static_cast<int64_t>(n_heads) * yapd::kHeadDim && q_tok_stride % 8 == 0,
               "attn_tree: q_tok_stride must be a multiple of 8, at least n_heads * 64");
  YAPD_REQUIRE(n_pages >= 1 && table_cols >= 1 && table_stride >= table_cols, "attn_tree: empty pool or table");
  YAPD_REQUIRE(table_cols <= yapd::kCap / yapd::kPageSize, "attn_tree: table_cols must be at most 2^26");
  YAPD_REQUIRE(q_start != nullptr || n_q == static_cast<int64_t>(rows) * max_q,
               "attn_tree: without q_start n_q must be rows * max_q");
  YAPD_REQUIRE(scale >= 1e-30f && scale <= 1e30f, "attn_tree: scale must be in [1e-30, 1e30]");
  const yapd::Cut c = yapd::cut_of(rows, max_q, n_heads, window, sinks, max_kv, bits);
  YAPD_REQUIRE(static_cast<int64_t>(rows) * c.parts * n_heads < (int64_t{1} << 22), "attn_tree: too many rows for one launch");
  const int64_t tokens = static_cast<int64_t>(c.parts) * n_q * n_heads;
  YAPD_REQUIRE(c.parts == 1 || (workspace && yapd::al16(workspace) && workspace_floats >= tokens * (yapd::kHeadDim + 2)),
               "attn_tree: the workspace must be 16-byte aligned and hold %lld floats",
               static_cast<long long>(tokens * (yapd::kHeadDim + 2)));
  const int64_t out_bytes = static_cast<int64_t>(n_q) * n_heads * yapd::kHeadDim * 2;
  YAPD_REQUIRE(!yapd::overlap(q, n_q, q_tok_stride * 2, out_bytes / n_q, out, out_bytes), "attn_tree: out overlaps q");
  const int64_t pool_bytes = n_pages * 2 * n_heads * (bits == 8 ? yapd::kTile8 : yapd::kHeadTile * 2);
  YAPD_REQUIRE(!yapd::overlap(kv_pool, 1, pool_bytes, pool_bytes, out, out_bytes), "attn_tree: out overlaps the pool");
  yapd::TreeParams P;
  P.q = static_cast<const uint16_t*>(q);
  P.q_stride = q_tok_stride;
  P.pool = kv_pool;
  P.n_pages = n_pages;
  P.table = page_table;
  P.table_stride = table_stride;
  P.table_cols = table_cols;
  P.kv_len = kv_len;
  P.q_start = q_start;
  P.mask = mask;
  P.rows = rows;
  P.max_q = max_q;
  P.n_q = n_q;
  P.H = n_heads;
  P.window = std::min(window, yapd::kCap);
  P.sinks = std::min(sinks, yapd::kCap);
  P.parts = c.parts;
  // Workgroups that the chip does not hold at once: two a CU with two query tiles, else four.
  const int64_t groups = static_cast<int64_t>(rows) * n_heads * c.w / 4, held = c.nqt == 1 ? 1024 : 512;
  P.class_scale = 0.f;
  if (c.parts == 1 && rows > 1 && rows <= yapd::kSorted && groups > held) {
    const double most = std::min<double>(std::min<double>(max_kv, table_cols * 16.0),
                                         static_cast<double>(P.window) + P.sinks + max_q);
    P.class_scale = static_cast<float>(yapd::kClasses / (most * (c.nqt == 1 ? 1.0 : 900.0)));
  }
  P.part_o = workspace;
  P.part_ml = c.parts == 1 ? nullptr : workspace + tokens * yapd::kHeadDim;
  P.scale_log2 = scale * 1.4426950408889634f;
  P.out = static_cast<uint16_t*>(out);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (bits == 8)
    yapd::launch<true>(P, c, st);
  else
    yapd::launch<false>(P, c, st);
  YAPD_LAUNCH_CHECK("attn_tree_kernel launch");
  if (c.parts > 1) {
    const int64_t pairs = static_cast<int64_t>(rows) * max_q * n_heads;
    hipLaunchKernelGGL(yapd::attn_tree_join_kernel, dim3(static_cast<unsigned>((pairs + 15) / 16)), dim3(256), 0, st, P);
    YAPD_LAUNCH_CHECK("attn_tree_join_kernel launch");
  }
  return YAPD_OK;
}
