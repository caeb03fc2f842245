// Paged-KV attention with a sliding window and sink tokens.
//
// Query i of row r stands at position p = kv_len[r] - n(r) + i and sees key
// j iff  j < hi  and  (j < sinks  or  j > p - window),  hi = p + 1 (causal) or
// kv_len[r] (block: the later positions of its own block too):
//   out = sum_j softmax_j(scale q . k_j) v_j   over the visible j.
// What a step reads is bounded by window + sinks keys a row, so it needs no
// host plan: every workgroup derives its key range from the device lengths,
// and a captured launch follows them as they grow.
//
// A row's queries are cut into tiles of 16 NQT; a tile's visible keys are a
// list of 32-key chunks: the sinks' chunks, then those from the first query's
// window on.  The list is cut into `parts` (workgroups) and each part into KS
// runs (waves); runs join in LDS, parts through a workspace and a second
// launch.  Chunk arithmetic is that of the paged block attention: S^T = K Q^T
// and O^T += V^T P^T on v_mfma_f32_16x16x32_bf16, every lane owning one query.
//
// Short tiles are bound by memory: 256 ragged rows of one token on up to 1088 keys
// x 16 heads 169 us, 5.9 TB/s; three rows on 16384 keys 37.0 us, 5.5 TB/s; 130
// blocks of 32 on up to 565 keys 61 us, 4.8 TB/s.  One row on 1028 keys takes 8.2 us:
// length, page ids and keys are loads that wait for each other, and one CU fetches
// about 50 GB/s.
#include <algorithm>

#include "attn_tile.h"
#include "common.h"
#include "kv_layout.h"
#include "lds_dma.h"

namespace yapd {
namespace {

constexpr int kChunk = 32;        // keys per inner step (two pages)
constexpr int kCap = 1 << 30;     // window and sinks are held to this: p - window stays inside int32

struct WindowParams {
  const uint16_t* q;    // token t, head h at t * q_stride + h * 64
  int64_t q_stride;
  const uint16_t* pool;
  int64_t n_pages;
  const int32_t* table;
  int table_stride, table_cols;
  const int32_t* kv_len;
  const int32_t* q_start;  // [rows + 1], or NULL: row r's queries are r * max_q ..
  int rows, max_q, n_q, H;
  int window, sinks, causal;
  int parts;
  float* part_o;   // [parts, n_q, H, 64]
  float* part_ml;  // [parts, n_q, H, 2]
  float scale_log2;
  uint16_t* out;  // [n_q, H, 64]
};

// A tile of one row's queries: rows qs .. qs + qc - 1 of q / out at positions p0, p0 + 1, ...
struct Tile {
  int row, qs, qc, p0, kvl;
};

__device__ __forceinline__ int first_query(const WindowParams& P, int r) {
  return min(max(P.q_start[r], 0), P.n_q);
}

// Tile `slot` of the launch.  Uniform rows have ceil(max_q / TQ) slots each;
// of packed rows, row r's tiles start at slot f(r) = q_start[r] / TQ + r: its
// ceil(n / TQ) tiles end at or before f(r + 1), and f grows with r, so the row
// is found by a 64-way search.  false: the slot holds no query.
template <int TQ>
__device__ __forceinline__ bool find_tile(const WindowParams& P, int slot, int lane, Tile& t) {
  int first, n;  // n: the row's queries, also those past max_q, which have positions but no tile
  if (P.q_start == nullptr) {
    const int per = (P.max_q + TQ - 1) / TQ;
    t.row = slot / per;
    t.qs = t.row * P.max_q;
    n = P.max_q;
    first = (slot - t.row * per) * TQ;
  } else {
    int base = 0, left = P.rows;
    while (left > 1) {
      const int step = (left + 63) / 64;
      const int i = lane * step;
      const bool le = i < left && first_query(P, base + min(i, left - 1)) / TQ + base + i <= slot;
      const int at = (max(__popcll(__ballot(le)), 1) - 1) * step;
      base += at;
      left = min(step, left - at);
    }
    t.row = base;
    t.qs = first_query(P, base);
    n = max(first_query(P, base + 1) - t.qs, 0);
    first = (slot - t.qs / TQ - base) * TQ;
  }
  t.qc = min(n, P.max_q);
  if (first < 0 || first >= t.qc) return false;
  t.kvl = min(max(P.kv_len[t.row], 0), P.table_cols * kPageSize);
  t.p0 = t.kvl - n + first;
  t.qs += first;
  t.qc = min(TQ, t.qc - first);
  return true;
}

// The chunks (of C keys) that some query of a tile sees: list entry c is chunk
// c below n_sink, chunk skip + c from there on.
struct ChunkList {
  int lo, hi;  // keys seen: [0, sinks) and [lo, hi), both below hi
  int n_sink, skip, n;
  __device__ __forceinline__ ChunkList(const WindowParams& P, const Tile& t, int C) {
    const int last = t.p0 + t.qc - 1;
    lo = max(t.p0 - P.window + 1, 0);
    hi = max(P.causal ? min(t.kvl, last + 1) : t.kvl, 0);
    const int cb = min(lo, hi) / C, ce = (hi + C - 1) / C;
    n_sink = min((min(P.sinks, hi) + C - 1) / C, cb);
    skip = cb - n_sink;
    n = n_sink + ce - cb;
  }
  __device__ __forceinline__ int chunk(int c) const { return c < n_sink ? c : c + skip; }
};

// The row's page ids, 64 at a time: lane i holds the page of table column
// base + i (clamped), and a chunk picks its pages with readlane.
struct Pages {
  const int32_t* tab;
  int last_page, max_page, lane, base, v;
  __device__ __forceinline__ Pages(const WindowParams& P, const Tile& t, int first, int lane_)
      : tab(P.table + static_cast<int64_t>(t.row) * P.table_stride),
        last_page(max((t.kvl + kPageSize - 1) / kPageSize - 1, 0)),
        max_page(static_cast<int>(min(P.n_pages - 1, int64_t{0x7fffffff}))), lane(lane_) {
    load(min(first, last_page));
  }
  __device__ __forceinline__ void load(int b) {
    base = b;
    v = tab[min(base + lane, last_page)];
    asm volatile("" ::"v"(v));  // complete here: later uses wait on no load
  }
  __device__ __forceinline__ int operator()(int pi) {
    pi = min(pi, last_page);
    if (pi - base >= 64) load(pi);  // uniform: pi is the same for the wave, and never falls
    return min(max(__builtin_amdgcn_readlane(v, pi - base), 0), max_page);  // a bad table entry cannot fault
  }
};

constexpr int kWaveFloats = 4 * 64 * 4;  // a wave's O^T tile in LDS: fragment mt of lane l at (mt * 64 + l) * 4

// Chunk c + 1 is on its way while chunk c is multiplied.
template <int NQT, int KS, int HPW>
__global__ __launch_bounds__(64 * KS * HPW) __attribute__((amdgpu_waves_per_eu(NQT > 2 ? 2 : NQT == 2 ? 3 : 4))) void
attn_window_kernel(const WindowParams P) {
  constexpr int TQ = 16 * NQT;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int ks = wave % KS, hsub = wave / KS;
  const int groups = P.H / HPW;
  const int item = static_cast<int>(blockIdx.x) / groups;
  const int h = (static_cast<int>(blockIdx.x) - item * groups) * HPW + hsub;
  const int slot = item / P.parts, part = item - slot * P.parts;
  Tile t;
  if (!find_tile<TQ>(P, slot, lane, t)) return;  // the whole workgroup
  const int g = lane >> 4, n = lane & 15;
  const int H = P.H;
  const ChunkList cl(P, t, kChunk);

  // Q^T fragments (B operand): lane holds Q[q = qt*16 + n][hd = s*32 + 8g .. +7]
  bf16x8_t qf[NQT][2];
#pragma unroll
  for (int qt = 0; qt < NQT; ++qt) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      u32x4_t v = {0u, 0u, 0u, 0u};
      if (qt * 16 + n < t.qc) v = load16(P.q + (t.qs + qt * 16 + n) * P.q_stride + h * kHeadDim + s * 32 + 8 * g);
      qf[qt][s] = as_bf16x8(v);
    }
  }
  f32x4_t o[NQT][4];
  float m[NQT], l[NQT];
#pragma unroll
  for (int qt = 0; qt < NQT; ++qt) {
    m[qt] = -INFINITY;
    l[qt] = 0.f;
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) o[qt][mt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  // this wave's run of the list
  const int64_t runs = static_cast<int64_t>(P.parts) * KS, run = static_cast<int64_t>(part) * KS + ks;
  const int c0 = static_cast<int>(cl.n * run / runs), c1 = static_cast<int>(cl.n * (run + 1) / runs);
  if (c0 < c1) {
    Pages page_of(P, t, cl.chunk(c0) * (kChunk / kPageSize), lane);
    // Key served by row n of S^T tile i: 8*(n/4) + 4i + n%4, so that lane group g
    // ends up holding keys 8g .. 8g+7 of the chunk.
    const int key_t0 = 8 * (n >> 2) + (n & 3);
    auto load_chunk = [&](int k0, u32x4_t (&kf)[2][2], u32x4_t (&vf)[4]) {
      const int pi0 = k0 / kPageSize;
      const int64_t pg0 = page_of(pi0), pg1 = page_of(pi0 + 1);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int key = key_t0 + 4 * i;
        const int64_t pg = key < kPageSize ? pg0 : pg1;
        const uint16_t* kp = P.pool + k_offset(pg, h, H, key & (kPageSize - 1), 8 * g);
        kf[i][0] = load16_stream(kp);
        kf[i][1] = load16_stream(kp + 32);
      }
      const int64_t pg = g < 2 ? pg0 : pg1;
      const uint16_t* vp = P.pool + v_offset(pg, h, H, 8 * (g & 1), n);
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) vf[mt] = load16_stream(vp + 16 * mt * kPageSize);
    };
    const int last = t.p0 + t.qc - 1;
    const int all_lo = last - P.window + 1;                 // keys from here on are in every query's window
    const int all_hi = P.causal ? min(t.kvl, t.p0 + 1) : t.kvl;  // keys below are before every query's end

    u32x4_t ka[2][2], va[4], kn[2][2], vn[4];
    load_chunk(cl.chunk(c0) * kChunk, ka, va);
    auto step = [&](int c, u32x4_t (&kf)[2][2], u32x4_t (&vf)[4]) {
      const int k0 = cl.chunk(c) * kChunk;
      const bool mask = k0 + kChunk > all_hi || (k0 < all_lo && k0 + kChunk > P.sinks);
      if (mask) {
        // V of keys that no query of the tile sees (behind the window, past the
        // end, stale slots of the last page): cleared, so 0 * V is never NaN
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int key = k0 + 8 * g + 2 * w;
          const bool see0 = key < cl.hi && (key >= cl.lo || key < P.sinks);
          const bool see1 = key + 1 < cl.hi && (key + 1 >= cl.lo || key + 1 < P.sinks);
          const uint32_t keep = (see0 ? 0x0000ffffu : 0u) | (see1 ? 0xffff0000u : 0u);
#pragma unroll
          for (int mt = 0; mt < 4; ++mt) vf[mt][w] &= keep;
        }
      }
#pragma unroll
      for (int qt = 0; qt < NQT; ++qt) {
        f32x4_t s[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          s[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(kf[i][0]), qf[qt][0],
                                                         f32x4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
          s[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(kf[i][1]), qf[qt][1], s[i], 0, 0, 0);
        }
        // s[i][j] = S[q = n][key 8g + 4i + j]
        float sv[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) sv[i] = s[i >> 2][i & 3] * P.scale_log2;
        if (mask) {  // uniform
          const int p = t.p0 + qt * 16 + n;
          const int q_hi = P.causal ? min(t.kvl, p + 1) : t.kvl, q_lo = p - P.window + 1;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int key = k0 + 8 * g + i;
            sv[i] = key < q_hi && (key >= q_lo || key < P.sinks) ? sv[i] : -INFINITY;
          }
        }
        float cm = sv[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) cm = fmaxf(cm, sv[i]);
        cm = max_xor16_32(cm);
        const float mn = fmaxf(m[qt], cm);
        // no key seen yet: exponents against 0 give alpha = 0 and p = 0 instead of NaN
        const float mref = mn == -INFINITY ? 0.f : mn;
        const float alpha = __builtin_amdgcn_exp2f(m[qt] - mref);
        float p[8], ps = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          p[i] = __builtin_amdgcn_exp2f(sv[i] - mref);
          ps += p[i];
        }
        l[qt] = l[qt] * alpha + ps;
        m[qt] = mn;
        // P in bf16: the operand type of the product with V (a rounding of 2^-9 of each weight, averaged over keys)
        u32x4_t pw;
#pragma unroll
        for (int w = 0; w < 4; ++w) pw[w] = pack_bf16x2(p[2 * w], p[2 * w + 1]);
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
          o[qt][mt] *= alpha;
          o[qt][mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(vf[mt]), as_bf16x8(pw), o[qt][mt], 0, 0, 0);
        }
      }
    };
    // A load behind a branch of its own makes the wait before a chunk's use one for the next chunk's too, so the loop's
    // are unconditional and its end a copy of it: one row on 1028 keys 8.7 -> 8.1 us, 16 blocks of 32 14.2 -> 13.0.  For
    // three and four query tiles four copies of the step are too much code: 256 blocks of 64 176 -> 199.
    int c = c0;
    if constexpr (NQT <= 2) {
      for (; c + 2 < c1; c += 2) {
        load_chunk(cl.chunk(c + 1) * kChunk, kn, vn);
        step(c, ka, va);
        load_chunk(cl.chunk(c + 2) * kChunk, ka, va);
        step(c + 1, kn, vn);
      }
      if (c + 1 < c1) {
        load_chunk(cl.chunk(c + 1) * kChunk, kn, vn);
        step(c, ka, va);
        step(c + 1, kn, vn);
      } else {
        step(c, ka, va);
      }
    } else {
      for (; c < c1; c += 2) {
        if (c + 1 < c1) load_chunk(cl.chunk(c + 1) * kChunk, kn, vn);
        step(c, ka, va);
        if (c + 1 >= c1) break;
        if (c + 2 < c1) load_chunk(cl.chunk(c + 2) * kChunk, ka, va);
        step(c + 1, kn, vn);
      }
    }
  }

  // o[qt][mt][j] = O^T[hd = 16mt + 4g + j][q = qt*16 + n].  With KS runs: their
  // O^T, m and l go to LDS, and wave ks joins the fragments mt = ks, ks + KS, ..
  __shared__ __attribute__((aligned(16))) float s_o[KS > 1 ? HPW * KS * kWaveFloats : 4];
  __shared__ float s_ml[KS > 1 ? HPW * KS * 32 : 2];
#pragma unroll
  for (int qt = 0; qt < NQT; ++qt) {
    const int q = qt * 16 + n;
    const int64_t token = t.qs + q;
    float M = m[qt], L = sum_xor16_32(l[qt]);
    auto finish = [&](int mt, f32x4_t acc) {
      if (q >= t.qc) return;
      const int64_t at = (token * H + h) * kHeadDim + 16 * mt + 4 * g;
      if (P.parts == 1) {
        // L = 0 only for a query that sees no key (an empty row): zeros, not NaN
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
    if constexpr (KS == 1) {
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) finish(mt, o[qt][mt]);
    } else {
      float* so = s_o + hsub * KS * kWaveFloats;
      float* sml = s_ml + hsub * KS * 32;
      if (qt > 0) __syncthreads();  // the previous tile has been read
#pragma unroll
      for (int mt = 0; mt < 4; ++mt)
        *reinterpret_cast<f32x4_t*>(so + ks * kWaveFloats + (mt * 64 + lane) * 4) = o[qt][mt];
      if (g == 0) {
        sml[ks * 32 + n] = M;
        sml[ks * 32 + 16 + n] = L;
      }
      __syncthreads();
      M = -INFINITY;
#pragma unroll
      for (int w = 0; w < KS; ++w) M = fmaxf(M, sml[w * 32 + n]);
      const float mref = M == -INFINITY ? 0.f : M;
      float sc[KS];
      L = 0.f;
#pragma unroll
      for (int w = 0; w < KS; ++w) {
        sc[w] = __builtin_amdgcn_exp2f(sml[w * 32 + n] - mref);
        L += sc[w] * sml[w * 32 + 16 + n];
      }
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        if (mt % KS != ks) continue;
        f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < KS; ++w)
          acc += sc[w] * *reinterpret_cast<const f32x4_t*>(so + w * kWaveFloats + (mt * 64 + lane) * 4);
        finish(mt, acc);
      }
    }
  }
}

// Long runs of queries: a workgroup takes 128 queries of one head, 32 a wave,
// and brings 64-key chunks through a ring of two LDS stages, where the four
// waves share them, one barrier a chunk.  v_mfma_f32_32x32x16_bf16: S^T = K Q^T
// (M = keys, N = queries) leaves a lane one query and half of a tile's keys;
// K rows are permuted so that those are 8 consecutive keys per 16, the operand
// of O^T += V^T P^T, and 8 consecutive bf16 of a V^T row of a page.
//
// Bound by neither unit alone but by how little of the two overlaps: a wave's
// 32 x 64 scores are 123 vector instructions (64 of them the exponentials and
// their arguments) and 16 products, and within a wave the products with K, the
// softmax and the products with V follow each other; only waves that drift apart
// run one beside another.  8000 queries x 16 heads on a window of 2048: 92 us,
// 0.73 PF/s, at 1.9 GHz; without the products 61, without the exponentials 79; the
// vector unit issues in 44 % of the cycles, the matrix unit is busy in 28 %.  A
// third or fourth stage gains 2 to 4 % where workgroups are few and costs a
// workgroup of a CU where they are many (100 us); one workgroup a CU takes 1 us a
// chunk, its waves' chain of these steps.  From 65 queries on: 16 rows of 80 x 16
// heads 23.3 us, in tiles of 64 on single waves 38.9; 64 rows of 64 there 48.4, here 54.0.
//
// LDS: K rows of 128 bytes, 16-byte piece c of key j in slot c ^ (j / 2 & 7); V^T
// pages of 64 x 32 bytes, the halves swapped where hd & 8: the 16 lanes of a
// phase of a fragment read fill 16 distinct slots.
constexpr int kTileQ = 128, kTileChunk = 64, kStages = 2;
constexpr float kSlack = 8.f;
constexpr int kStage = 2 * kTileChunk * kHeadDim * 2;  // bytes

template <int CTRL>
__device__ __forceinline__ int dpp(int v) {
  return __builtin_amdgcn_mov_dpp(v, CTRL, 0xF, 0xF, true);  // no lane is out of range
}
// A wave's sum or maximum, uniform: quad permutes, half-row and row mirrors, then the four rows.
template <class Op>
__device__ __forceinline__ int wave_reduce(int v, Op op) {
  v = op(v, dpp<0xB1>(v));
  v = op(v, dpp<0x4E>(v));
  v = op(v, dpp<0x141>(v));
  v = op(v, dpp<0x140>(v));
  return op(op(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
            op(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}

// find_tile for packed rows that a wave holds one a lane: slot i is the i-th tile by weight, the heaviest first (the
// weight: keys before the tile, in tiles, up to the window).  All workgroups of a launch that fits the chip start at
// once, a CU has every 256th of them, and tiles of a row's begin weigh little: in the order of the rows some CUs have
// half as much again as the mean.  us by weight / in row order, 16 heads, prompts of 70 to 1500 tokens: 9 on a window
// of 512 27.2 / 33.0, of 4000 33.1 / 40.5; 20 (2300 workgroups) 51.0 / 55.4 and 58.4 / 68.1; but 40 (4600) 110.6 / 108.1,
// where the light tiles' start is no longer hidden behind heavy ones.
constexpr unsigned kWeighed = 2560;  // workgroups

__device__ __forceinline__ bool find_weighed_tile(const WindowParams& P, int slot, int lane, Tile& t) {
  const int r = min(lane, P.rows - 1);
  const int qs = first_query(P, r), qe = first_query(P, r + 1);
  const int len = min(max(P.kv_len[r], 0), P.table_cols * kPageSize);
  const int n = lane < P.rows ? max(qe - qs, 0) : 0;  // also those past max_q, which have positions but no tile
  const int n_tiled = min(n, P.max_q);
  const int tiles = (n_tiled + kTileQ - 1) / kTileQ, before = max(len - n, 0) / kTileQ;
  const auto add = [](int a, int b) { return a + b; };
  const auto larger = [](int a, int b) { return max(a, b); };
  const int top = wave_reduce(tiles > 0 ? min(tiles - 1 + before, (P.window + kTileQ - 1) / kTileQ) : 0, larger);
  const auto first_of = [&](int w) { return w > top ? tiles : min(max(w - before, 0), tiles); };  // tile of weight >= w
  if (slot >= wave_reduce(tiles, add)) return false;
  int lo = 0, hi = top + 1, above = 0;  // weights >= lo hold more than `slot` tiles, weights >= hi hold `above`, no more
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1, count = wave_reduce(tiles - first_of(mid), add);
    if (count > slot) {
      lo = mid;
    } else {
      hi = mid;
      above = count;
    }
  }
  const int k0 = first_of(lo), m = first_of(hi) - k0;  // this row's tiles of weight lo
  int sum = m;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int left = __shfl_up(sum, d);
    if (lane >= d) sum += left;
  }
  const int at = __ffsll(static_cast<unsigned long long>(__ballot(sum > slot - above))) - 1;
  const int first = __builtin_amdgcn_readlane(k0 + m - sum, at) + slot - above;
  t.row = at;
  t.kvl = __builtin_amdgcn_readlane(len, at);
  t.p0 = t.kvl - __builtin_amdgcn_readlane(n, at) + first * kTileQ;
  t.qs = __builtin_amdgcn_readlane(qs, at) + first * kTileQ;
  t.qc = min(kTileQ, __builtin_amdgcn_readlane(n_tiled, at) - first * kTileQ);
  return true;
}

// A product that is rounded wherever it is used: never fused into a sum.
__device__ __forceinline__ float rounded_product(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(4))) void attn_window_tile_kernel(const WindowParams P) {
  // dynamic: only the direct loads write it, which the compiler does not see as writes of a static array
  extern __shared__ __attribute__((aligned(16))) char ring[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int item = static_cast<int>(blockIdx.x) / P.H;
  const int h = static_cast<int>(blockIdx.x) - item * P.H;
  const int slot = item / P.parts, part = item - slot * P.parts;
  Tile t;
  if (P.q_start != nullptr && P.rows > 1 && P.rows <= 64 && gridDim.x <= kWeighed) {
    if (!find_weighed_tile(P, slot, lane, t)) return;  // the whole workgroup
  } else if (!find_tile<kTileQ>(P, slot, lane, t)) {
    return;
  }
  const int g = lane >> 5, n = lane & 31;
  const int H = P.H;
  const ChunkList cl(P, t, kTileChunk);
  const int c0 = static_cast<int>(static_cast<int64_t>(cl.n) * part / P.parts);
  const int c1 = static_cast<int>(static_cast<int64_t>(cl.n) * (part + 1) / P.parts);
  const int q = wave * 32 + n;  // this lane's query of the tile

  Pages page_of(P, t, cl.chunk(c0) * (kTileChunk / kPageSize), lane);
  // Wave w brings page w of a chunk: 2 KB of K and 2 KB of V^T, 1 KB an instruction.
  uint32_t k_ofs[2], v_ofs;
#pragma unroll
  for (int j = 0; j < 2; ++j) k_ofs[j] = (lane >> 3) * 128 + 16 * ((lane & 7) ^ ((4 * j + (lane >> 4)) & 7));
  v_ofs = (lane >> 1) * 32 + 16 * ((lane & 1) ^ (lane >> 4 & 1));
  const uint32_t k_plane = static_cast<uint32_t>(kv_plane_offset(0, 0, h, H) * 2);
  const uint32_t v_plane = static_cast<uint32_t>(kv_plane_offset(0, 1, h, H) * 2);
  auto issue = [&](int c, int st) {
    const int pi = cl.chunk(c) * (kTileChunk / kPageSize) + wave;
    const __amdgpu_buffer_rsrc_t rs = buffer_from(P.pool + kv_plane_offset(page_of(pi), 0, 0, H));
    char* to = ring + st * kStage + wave * 2048;
#pragma unroll
    for (int j = 0; j < 2; ++j) load_lds16(rs, k_ofs[j], k_plane + j * 1024, to + j * 1024);
#pragma unroll
    for (int j = 0; j < 2; ++j) load_lds16(rs, v_ofs, v_plane + j * 1024, to + kStage / 2 + j * 1024);
  };

  if (c0 < c1) issue(c0, 0);

  // Q^T fragments (B operand): lane holds Q[q][hd = 16s + 8g .. +7]
  bf16x8_t qf[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    u32x4_t v = {0u, 0u, 0u, 0u};
    if (q < t.qc) v = load16(P.q + (t.qs + q) * P.q_stride + h * kHeadDim + s * 16 + 8 * g);
    qf[s] = as_bf16x8(v);
  }
#pragma unroll
  for (int s = 0; s < 4; ++s) asm volatile("" ::"v"(qf[s]));  // complete before the loop, whose waits are its own

  f32x16_t o[2];
#pragma unroll
  for (int mt = 0; mt < 2; ++mt) o[mt] = f32x16_t{};
  float m = -INFINITY, mref = 0.f, l = 0.f;
  const float slack = kSlack / P.scale_log2;
  const bf16x2_t one2 = {static_cast<__bf16>(1.f), static_cast<__bf16>(1.f)};
  float inf = INFINITY;
  asm("" : "+s"(inf));  // opaque: the compiler turns v_med3 with a known +inf back into v_max
  // row n of an S^T tile: key 16 (n / 16) + 8 (n / 4 & 1) + 4 (n / 8 & 1) + n % 4 of its 32
  const int key_n = 16 * (n >> 4) + 8 * (n >> 2 & 1) + 4 * (n >> 3 & 1) + (n & 3);
  const int k_row = key_n * 128, k_sw = key_n >> 1 & 7;
  const int v_row = n * 32 + 16 * (g ^ (n >> 3 & 1));
  const int p = t.p0 + q;
  const int q_hi = P.causal ? min(t.kvl, p + 1) : t.kvl, q_lo = p - P.window + 1;
  // of this wave's queries: what all see, what any sees
  const int w_first = t.p0 + wave * 32, w_last = t.p0 + min(wave * 32 + 31, t.qc - 1);
  const bool w_any = wave * 32 < t.qc;
  const int all_hi = P.causal ? min(t.kvl, w_first + 1) : t.kvl, all_lo = w_last - P.window + 1;
  const int any_hi = P.causal ? min(t.kvl, w_last + 1) : t.kvl, any_lo = w_first - P.window + 1;
  // list entries whose keys are all seen by all of this wave's queries: nothing to skip, mask or clear
  const int clean_lo = max(cl.skip > 0 ? cl.n_sink : 0, (max(all_lo, 0) + kTileChunk - 1) / kTileChunk - cl.skip);
  const int clean_hi = w_any ? max(all_hi, 0) / kTileChunk - cl.skip : 0;

  f32x16_t s[2];
  u32x4_t vf[2][2];
  // O^T += V^T P^T and the sum of the weights, for the scores in s and the V^T fragments in vf
  auto add_chunk = [&](const char* vb) {
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {  // 16 keys: a page
      u32x4_t pw;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int e = 8 * (kk & 1) + 2 * w;
        const uint32_t two = pack_bf16x2(__builtin_amdgcn_exp2f(__builtin_fmaf(s[kk >> 1][e], P.scale_log2, -mref)),
                                         __builtin_amdgcn_exp2f(__builtin_fmaf(s[kk >> 1][e + 1], P.scale_log2, -mref)));
        pw[w] = two;

        // the sum of the weights as the product with V has them
        l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, two), one2, l, false);
      }
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        o[mt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(vf[kk & 1][mt]), as_bf16x8(pw), o[mt], 0, 0, 0);
        if (kk < 2) vf[kk & 1][mt] = *reinterpret_cast<const u32x4_t*>(vb + (kk + 2) * 2048 + mt * 1024 + v_row);
      }
    }
  };
  int st = 0;
  for (int c = c0;; ++c) {
    // The exponents are taken against m, which follows a query's maximum only when that
    // has left it by more than 2^kSlack.  The inner loop runs while none of the wave's has,
    // and keeps the accumulators in place (with the rescaling as a branch inside it, every
    // chunk paid 80 register copies).  It costs precision: against the maximum itself the
    // heaviest weight is 1, which bf16 holds, against one that lags it is rounded like the
    // others.  Relative error of 8000 queries on a window of 2048, spread 2: 2.18e-3, with no
    // slack 1.89e-3 in 102.4 us instead of 92.9 (the output's own rounding alone: 1.66e-3);
    // nine packed prompts 1.96e-3 and 1.82e-3, 27.8 and 28.6; 16 rows of 80 23.3 and 24.1.
    float mn = -INFINITY;
    char* vb = ring;
    bool moved = false;
    for (; c < c1; ++c) {
      const bool edge = c < clean_lo || c >= clean_hi;
      const int k0 = cl.chunk(c) * kTileChunk;
      char* const kb = ring + st * kStage;
      vb = kb + kStage / 2;
      // this wave's page of chunk c has landed
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (edge && (k0 + kTileChunk > cl.hi || (k0 < cl.lo && k0 + kTileChunk > P.sinks))) {
        // V of keys that no query of the tile sees is cleared, so 0 * V is never NaN: lane = head dim of the wave's page
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          u32x4_t* v = reinterpret_cast<u32x4_t*>(vb + wave * 2048 + lane * 32 + 16 * (half ^ (lane >> 3 & 1)));
          u32x4_t x = *v;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const int key = k0 + 16 * wave + 8 * half + 2 * w;
            const bool see0 = key < cl.hi && (key >= cl.lo || key < P.sinks);
            const bool see1 = key + 1 < cl.hi && (key + 1 >= cl.lo || key + 1 < P.sinks);
            x[w] &= (see0 ? 0x0000ffffu : 0u) | (see1 ? 0xffff0000u : 0u);
          }
          *v = x;
        }
      }
      // and everyone's, and every wave has read chunk c - 1: its stage takes chunk c + 1
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      st ^= 1;
      if (c + 1 < c1) issue(c + 1, st);
      if (edge && (!w_any || k0 >= any_hi || (k0 + kTileChunk <= any_lo && k0 >= P.sinks))) continue;  // no query of the wave sees it
      // all of a chunk's fragments are requested before the first is used
      u32x4_t kf[4][2];
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          kf[ks][i] = *reinterpret_cast<const u32x4_t*>(kb + i * 4096 + k_row + 16 * ((2 * ks + g) ^ k_sw));
      __builtin_amdgcn_sched_barrier(0);
      s[0] = f32x16_t{};
      s[1] = f32x16_t{};
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          s[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(kf[ks][i]), qf[ks], s[i], 0, 0, 0);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
          vf[kk][mt] = *reinterpret_cast<const u32x4_t*>(vb + kk * 2048 + mt * 1024 + v_row);
      __builtin_amdgcn_sched_barrier(0);
      // s[i][e] = S[q][key 32i + 16 (e / 8) + 8g + e % 8]
      if (edge) {  // uniform, as are the two below; element (i, e) of s is key kg + 32i + 16 (e / 8) + e % 8
        const int kg = k0 + 8 * g;
        if (k0 + kTileChunk > all_hi) {
          const int end = q_hi - kg;
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) s[i][e] = 32 * i + 16 * (e >> 3) + (e & 7) < end ? s[i][e] : -INFINITY;
        }
        if (k0 < all_lo && k0 + kTileChunk > P.sinks) {
          const int begin = q_lo - kg, sink_end = P.sinks - kg;
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int j = 32 * i + 16 * (e >> 3) + (e & 7);
              s[i][e] = j >= begin || j < sink_end ? s[i][e] : -INFINITY;
            }
        }
      }
      // v_med3 with +inf is a maximum that does not quiet its operands first, as v_max would have to
      float cm[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        cm[e] = fmaxf(__builtin_amdgcn_fmed3f(s[0][e], s[0][e + 8], inf), __builtin_amdgcn_fmed3f(s[1][e], s[1][e + 8], inf));
#pragma unroll
      for (int e = 1; e < 8; ++e) cm[0] = fmaxf(cm[0], cm[e]);
      const float2 both = swap32(cm[0]);
      mn = fmaxf(both.x, both.y);
      moved = __any(mn > m + slack);
      if (moved) break;
      __builtin_amdgcn_s_setprio(1);  // waves of a SIMD drift apart: one's products run beside another's exponentials
      add_chunk(vb);
      __builtin_amdgcn_s_setprio(0);
    }
    if (!moved) break;  // the last chunk is done
    // Of the wave's queries those move that have left their own maximum that far, so a query's sums depend on its own
    // scores alone.  The factor is taken between the references as the exponents had them: exactly 1 for a query that
    // stays, however often others move.  A first maximum's is of sums that are 0: held to 1, it cannot be infinite.
    const bool mine = mn > m + slack;
    const float to = mine ? rounded_product(mn, P.scale_log2) : mref;
    const float alpha = __builtin_amdgcn_exp2f(fminf(mref - to, 0.f));
    m = mine ? mn : m;
    mref = to;
    l *= alpha;
    o[0] *= alpha;
    o[1] *= alpha;
    add_chunk(vb);
  }
  const float2 lb = swap32(l);
  const float L = lb.x + lb.y;
  if (q >= t.qc) return;
  // o[mt][e] = O^T[hd = 32mt + 8 (e / 4) + 4g + e % 4][q]
  const int64_t token = t.qs + q, at = (token * H + h) * kHeadDim + 4 * g;
  if (P.parts == 1) {
    const float inv = L == 0.f ? 0.f : 1.f / L;  // no key seen: zeros, not NaN
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        u32x2_t w2;
        w2[0] = pack_bf16x2(o[mt][4 * b] * inv, o[mt][4 * b + 1] * inv);
        w2[1] = pack_bf16x2(o[mt][4 * b + 2] * inv, o[mt][4 * b + 3] * inv);
        *reinterpret_cast<u32x2_t*>(P.out + at + 32 * mt + 8 * b) = w2;
      }
    }
  } else {
    float* po = P.part_o + static_cast<int64_t>(part) * P.n_q * H * kHeadDim + at;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
      for (int b = 0; b < 4; ++b)
        *reinterpret_cast<f32x4_t*>(po + 32 * mt + 8 * b) =
            f32x4_t{o[mt][4 * b], o[mt][4 * b + 1], o[mt][4 * b + 2], o[mt][4 * b + 3]};
    }
    if (g == 0) {
      float* ml = P.part_ml + (static_cast<int64_t>(part) * P.n_q * H + token * H + h) * 2;
      ml[0] = m * P.scale_log2;  // as the other form has it
      ml[1] = L;
    }
  }
}

// Joins the parts of every query: thread (query, head, 4 head-dim values).  Eight parts' values are requested
// before the first is used, so up to eight parts cost one memory latency: what bounds it.
__global__ __launch_bounds__(256) void attn_window_join_kernel(const WindowParams P) {
  constexpr int kAtOnce = 8;
  const int lane = threadIdx.x & 63;
  // there are parts only where (query, head) pairs are few: they fit 32 bits
  const uint32_t pair = blockIdx.x * 16 + (threadIdx.x >> 4);
  const uint32_t row_q = pair / static_cast<uint32_t>(P.H);
  const int h = static_cast<int>(pair - row_q * P.H);
  const int r = static_cast<int>(row_q / P.max_q), i = static_cast<int>(row_q - static_cast<uint32_t>(r) * P.max_q);
  if (r >= P.rows) return;
  int qs = r * P.max_q, qc = P.max_q;
  if (P.q_start != nullptr) {
    qs = first_query(P, r);
    qc = min(max(first_query(P, r + 1) - qs, 0), P.max_q);
  }
  if (i >= qc) return;
  const int64_t step = static_cast<int64_t>(P.n_q) * P.H;
  const int64_t at = static_cast<int64_t>(qs + i) * P.H + h;
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

// How a call is cut: tq queries a tile (16, 32, 48, 64, or kTileQ: the tile
// kernel), ks waves to a part's chunks, parts.
struct Cut {
  int tq, ks, parts;
  int64_t slots;
};

// Waves to a head's chunks, by how many (tile, head) pairs there are; us a call with 1, 2 and 4 of them, 16 heads.
// One token, 804 of 1201 keys: one row 19.3, 11.7, 7.2; 32 rows (512 pairs) 30.5, 20.6, 20.3; 64 rows 37.0, 37.5, 38.0;
// 256 rows 139.5, 141.7, 144.1.  Blocks of 32: 32 rows 36.1, 22.8, 23.8; 64 rows 39.8, 41.5, 42.4; 128 rows 78.6, 83.0,
// 87.8, but 130 ragged rows of 100 to 2000 keys 65.7, 58.7, 60.3.  Blocks of 64: 64 rows 55.1, 48.7, 58.1.  One token
// on 61 keys, 300 rows: 16.5, 19.1, 22.1.
constexpr int64_t kFour = 512, kTwo = 2560;

// Parts: as many as bring the workgroups to `wanted`, of at least `least` chunks each.  us in one part and as cut here.
// Waves on short tiles, up to the number of CUs and 8 chunks; one token, 16 heads: 1400 keys 11.5, 8.4; 2000 keys 15.3,
// 8.9; 4000 keys 27.2, 11.3; 30000 keys 207, 27.6; four rows of 1400 keys 13.1, 9.8; eight of 4000 keys 35.0, 25.4.
// Below kCutChunks the second launch costs the host (2 us) more than it saves: 1028 keys 9.0, 8.2 in four parts; 804
// keys 7.6, 7.6.  The tile kernel, which gains until a CU holds three workgroups, and 16 chunks; 200 queries, 16 heads:
// 1400 keys 24, 17.9; 4200 keys 64, 21.3 (parts of 8 chunks 24.4); 1300 on 9300 keys 132, 76 (to two a CU 91).
constexpr int64_t kCutChunks = 40;

int parts_of(int64_t workgroups, int64_t wanted, int64_t chunks, int64_t least) {
  if (chunks < kCutChunks) return 1;
  return static_cast<int>(std::max<int64_t>(1, std::min(wanted / workgroups, chunks / least)));
}

Cut cut_of(int rows, int max_q, int n_q, bool packed, int n_heads, int window, int sinks, int max_kv) {
  Cut c;
  c.tq = max_q <= 64 ? (max_q + 15) / 16 * 16 : kTileQ;
  const int tq = c.tq;
  c.slots = packed ? n_q / tq + static_cast<int64_t>(rows) : static_cast<int64_t>(rows) * ((max_q + tq - 1) / tq);
  const int64_t tiles = std::min<int64_t>(c.slots, (n_q + tq - 1) / tq + rows);
  const int64_t keys = std::min<int64_t>(max_kv, static_cast<int64_t>(window) + sinks + tq);
  const int64_t chunks = (keys + kChunk - 1) / kChunk + 1;
  const int64_t pairs = tiles * n_heads;
  c.ks = tq == kTileQ ? 1 : pairs <= kFour && chunks >= 4 ? 4 : pairs <= kTwo && chunks >= 2 ? 2 : 1;
  c.parts = tq == kTileQ ? parts_of(pairs, 768, chunks, 16) : c.ks == 4 ? parts_of(pairs, 256, chunks, 8) : 1;
  return c;
}

template <int NQT>
void launch_tiles(const WindowParams& P, const Cut& c, hipStream_t st) {
  const int64_t items = c.slots * P.parts;
  if (c.ks == 4)
    hipLaunchKernelGGL((attn_window_kernel<NQT, 4, 1>), dim3(items * P.H), dim3(256), 0, st, P);
  else if (c.ks == 2)
    hipLaunchKernelGGL((attn_window_kernel<NQT, 2, 2>), dim3(items * (P.H / 2)), dim3(256), 0, st, P);
  else
    hipLaunchKernelGGL((attn_window_kernel<NQT, 1, 4>), dim3(items * (P.H / 4)), dim3(256), 0, st, P);
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Whether any of n blocks of `bytes`, `pitch` >= bytes apart from a on, shares a byte with [b, b + b_bytes).
bool overlap(const void* a, int64_t n, int64_t pitch, int64_t bytes, const void* b, int64_t b_bytes) {
  const int64_t from = static_cast<int64_t>(reinterpret_cast<uintptr_t>(b)) - static_cast<int64_t>(reinterpret_cast<uintptr_t>(a));
  const int64_t first = from < bytes ? 0 : (from - bytes) / pitch + 1;  // the first block that ends behind b
  return first < n && first * pitch < from + b_bytes;
}

int window_checks(int rows, int max_q, int n_q, int n_heads, int window, int sinks, int max_kv) {
  YAPD_REQUIRE(rows >= 1 && max_q >= 1 && n_q >= 1, "attn_window: need rows, max_q and n_q >= 1 (got %d, %d, %d)", rows,
               max_q, n_q);
  YAPD_REQUIRE(n_heads >= 4 && n_heads % 4 == 0 && n_heads <= 1024,
               "attn_window: n_heads must be a multiple of 4, at most 1024 (got %d)", n_heads);
  YAPD_REQUIRE(window >= 1 && sinks >= 0, "attn_window: need window >= 1 and sinks >= 0 (got %d, %d)", window, sinks);
  YAPD_REQUIRE(max_kv >= 1, "attn_window: max_kv must be >= 1 (got %d)", max_kv);
  return YAPD_OK;
}

}  // namespace
}  // namespace yapd

extern "C" int64_t yapd_attn_window_workspace(int rows, int max_q, int n_q, int packed, int n_heads, int window,
                                              int sinks, int max_kv) {
  if (yapd::window_checks(rows, max_q, n_q, n_heads, window, sinks, max_kv) != YAPD_OK) return -1;
  const yapd::Cut c = yapd::cut_of(rows, max_q, n_q, packed != 0, n_heads, window, sinks, max_kv);
  return c.parts == 1 ? 0 : static_cast<int64_t>(c.parts) * n_q * n_heads * (yapd::kHeadDim + 2);
}

extern "C" int yapd_attn_window(const void* q, int64_t q_tok_stride, const void* kv_pool, int64_t n_pages,
                                const int32_t* page_table, int table_stride, int table_cols, const int32_t* kv_len,
                                const int32_t* q_start, int rows, int max_q, int n_q, int n_heads, int window, int sinks,
                                int causal, int max_kv, float scale, float* workspace, int64_t workspace_floats,
                                void* out, void* stream) {
  YAPD_REQUIRE(q && kv_pool && page_table && kv_len && out, "attn_window: NULL pointer");
  if (int rc = yapd::window_checks(rows, max_q, n_q, n_heads, window, sinks, max_kv)) return rc;
  YAPD_REQUIRE(yapd::al16(q) && yapd::al16(kv_pool) && yapd::al16(out),
               "attn_window: q, kv_pool and out must be 16-byte aligned");
  YAPD_REQUIRE(q_tok_stride >= static_cast<int64_t>(n_heads) * yapd::kHeadDim && q_tok_stride % 8 == 0,
               "attn_window: q_tok_stride must be a multiple of 8, at least n_heads * 64");
  YAPD_REQUIRE(n_pages >= 1 && table_cols >= 1 && table_stride >= table_cols, "attn_window: empty pool or table");
  YAPD_REQUIRE(table_cols <= yapd::kCap / yapd::kPageSize, "attn_window: table_cols must be at most 2^26");
  YAPD_REQUIRE(q_start != nullptr || n_q == static_cast<int64_t>(rows) * max_q,
               "attn_window: without q_start n_q must be rows * max_q");
  // 8 / scale and scale * log2(e) * a score stay in range
  YAPD_REQUIRE(scale >= 1e-30f && scale <= 1e30f, "attn_window: scale must be in [1e-30, 1e30]");
  const yapd::Cut c = yapd::cut_of(rows, max_q, n_q, q_start != nullptr, n_heads, window, sinks, max_kv);
  YAPD_REQUIRE(c.slots * c.parts * n_heads < (int64_t{1} << 22), "attn_window: too many tiles for one launch");
  const int64_t tokens = static_cast<int64_t>(c.parts) * n_q * n_heads;
  YAPD_REQUIRE(c.parts == 1 || (workspace && yapd::al16(workspace) &&
                                workspace_floats >= tokens * (yapd::kHeadDim + 2)),
               "attn_window: the workspace must be 16-byte aligned and hold %lld floats",
               static_cast<long long>(tokens * (yapd::kHeadDim + 2)));
  const int64_t out_bytes = static_cast<int64_t>(n_q) * n_heads * yapd::kHeadDim * 2;
  YAPD_REQUIRE(!yapd::overlap(q, n_q, q_tok_stride * 2, out_bytes / n_q, out, out_bytes), "attn_window: out overlaps q");
  const int64_t pool_bytes = n_pages * 2 * n_heads * yapd::kHeadTile * 2;
  YAPD_REQUIRE(!yapd::overlap(kv_pool, 1, pool_bytes, pool_bytes, out, out_bytes), "attn_window: out overlaps the pool");
  yapd::WindowParams P;
  P.q = static_cast<const uint16_t*>(q);
  P.q_stride = q_tok_stride;
  P.pool = static_cast<const uint16_t*>(kv_pool);
  P.n_pages = n_pages;
  P.table = page_table;
  P.table_stride = table_stride;
  P.table_cols = table_cols;
  P.kv_len = kv_len;
  P.q_start = q_start;
  P.rows = rows;
  P.max_q = std::min(max_q, n_q);
  P.n_q = n_q;
  P.H = n_heads;
  P.window = std::min(window, yapd::kCap);
  P.sinks = std::min(sinks, yapd::kCap);
  P.causal = causal != 0;
  P.parts = c.parts;
  P.part_o = workspace;
  P.part_ml = c.parts == 1 ? nullptr : workspace + tokens * yapd::kHeadDim;
  P.scale_log2 = scale * 1.4426950408889634f;
  P.out = static_cast<uint16_t*>(out);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  switch (c.tq) {
    case 16: yapd::launch_tiles<1>(P, c, st); break;
    case 32: yapd::launch_tiles<2>(P, c, st); break;
    case 48: yapd::launch_tiles<3>(P, c, st); break;
    case 64: yapd::launch_tiles<4>(P, c, st); break;
    default:
      hipLaunchKernelGGL(yapd::attn_window_tile_kernel, dim3(static_cast<unsigned>(c.slots * P.parts * P.H)), dim3(256),
                         yapd::kStages * yapd::kStage, st, P);
  }
  YAPD_LAUNCH_CHECK("attn_window_kernel launch");
  if (c.parts > 1) {
    const int64_t pairs = static_cast<int64_t>(rows) * P.max_q * n_heads;
    hipLaunchKernelGGL(yapd::attn_window_join_kernel, dim3(static_cast<unsigned>((pairs + 15) / 16)), dim3(256), 0, st,
                       P);
    YAPD_LAUNCH_CHECK("attn_window_join_kernel launch");
  }
  return YAPD_OK;
}
