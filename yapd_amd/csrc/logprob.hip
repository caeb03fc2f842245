// Log probabilities of given tokens, with the entropy and the best alternatives.
//
// For a row x of V logits and its token t, with m = max x:
//   logZ = m + ln S,  S = sum e^(x - m)
//   logprob = x_t - logZ,  entropy = ln S - (sum (x - m) e^(x - m)) / S,
//   the k largest x (ties: the lowest index first) minus logZ.
// One pass over a row by one wave or eight: every lane keeps the running maximum and the two
// sums over its 16-byte granules, a tile of them in registers at a time, rescaled when
// the maximum grows; they are joined across lanes on DPP and across waves in LDS.
// What bounds many rows is HBM: 16384 rows of 8194 bf16 with four alternatives 53.5 us, 5.0 TB/s
// (one wave a row: with four, 71, bound by the instructions that every wave runs once);
// 900 of 100003 fp32 with twenty 73.6 us, 4.9 TB/s (65.3 without alternatives: what a row does once, and
// the second read).  64 rows of 8194 take 7.0 us: one wave's chain of load, sums, search
// for T, second read and ranks.
//
// The best k: with T the k-th largest lane maximum (found bit by bit with ballots; of
// several waves' rows a bound below it), at least k elements reach T, and few more.  They sit in
// the lanes whose maximum reaches T.  A row of one wave has them put their granules into LDS, tile
// by tile, where the wave looks at one lane's elements at a time.  A row of several waves
// keeps the maxima of (lane, three granules) pairs in LDS, and once T is known those that
// reach it are read again.  What reaches T goes to a list with its
// index, and each candidate counts the keys above its own: that is its rank.  Rows of many equal
// logits (a mask's -inf or lowest value among the best k) overflow the list;
// there one wave walks the row for what lies above T and the first k that equal it.
#include <cmath>

#include "attn_tile.h"
#include "common.h"

namespace yapd {
namespace {

constexpr int kMaxTop = 32;
constexpr int kList = 256;    // candidates of a row; (kMaxTop - 1) lanes' granules of 8 and one more fit
constexpr int kPairs = 256;   // (lane, granules) pairs of a wave that hold them
constexpr uint32_t kNone = 0x007fffffu;  // order_of(-inf)
constexpr float kLn2 = 0.6931471805599453f, kLog2e = 1.4426950408889634f;
constexpr float kGone = -200.f;  // 2^kGone is 0 in fp32: a bound for d where d 2^d is 0, also at d = -inf
constexpr float kHuge = 65536.f;

struct LogprobParams {
  const void* logits;
  int64_t seq_stride, pos_stride;  // elements
  uint32_t items, bl;
  int vocab, top_k;
  const int64_t* tokens;
  float* logprob;
  float* entropy;
  float* top_logprob;
  int64_t* top_token;
};

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xF, 0xF, true));  // no lane is out of range
}
// A wave's reduction on DPP: quad permutes, half-row and row mirrors, then the four rows.
template <class Op>
__device__ __forceinline__ float wave_reduce(float v, Op op) {
  v = op(v, dpp<0xB1>(v));
  v = op(v, dpp<0x4E>(v));
  v = op(v, dpp<0x141>(v));
  v = op(v, dpp<0x140>(v));
  const float2 a = swap16(v);
  const float2 b = swap32(op(a.x, a.y));
  return op(b.x, b.y);
}

// Floats as unsigned numbers in their order (-0 taken as +0); NaN is ordered as -inf.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x == x ? x + 0.f : -INFINITY);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}
// Larger value first, then lower index.
__device__ __forceinline__ uint64_t key_of(float x, int index) {
  return static_cast<uint64_t>(order_of(x)) << 32 | (0xffffffffu - static_cast<uint32_t>(index));
}

// Exponents are taken as 2^(x L - shift), L = log2(e), in one FMA.  The shift is m L
// rounded, the same number wherever it is used, and the result is corrected by
// what the rounding left out.  That is small while |m| is; beyond kHuge (far from
// any model's logits, but a mask may hold the type's lowest value) the exponent
// is (x - m) L.  0 where nothing is above -inf yet: sums of 0, not NaN.
// The shift is never fused into a sum (as __fmul_rn may be): the sums of an unchanged maximum
// would be scaled by what its rounding leaves out, tile by tile.
__device__ __forceinline__ float shift_of(float m) {
#pragma clang fp contract(off)
  return m == -INFINITY ? 0.f : m * kLog2e;
}
__device__ __forceinline__ float left_of(float m) {
  return fabsf(m) > kHuge ? 0.f : __builtin_fmaf(m, kLog2e, -shift_of(m));
}

// The sums s, t taken against the maximum m, against `to` >= m instead.
__device__ __forceinline__ void rescale(float& s, float& t, float m, float to) {
  if (m == -INFINITY) return;  // no value above -inf yet: 0, or NaN if there was one
  float down = shift_of(m) - shift_of(to);
  if (fabsf(m) > kHuge || fabsf(to) > kHuge) down = (m - to) * kLog2e - left_of(m) + left_of(to);
  const float a = __builtin_amdgcn_exp2f(down);
  t = (t + s * fmaxf(down, kGone)) * a;
  s *= a;
}

template <bool kWide>
__device__ __forceinline__ float element(const void* row, int64_t i) {
  if constexpr (kWide) return static_cast<const float*>(row)[i];
  return bf16_to_f32(static_cast<const uint16_t*>(row)[i]);
}

// The maximum of three without quieting its operands first (they come from memory, so the
// compiler would); a NaN operand is left out.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// Lanes below this one in a ballot.
__device__ __forceinline__ int below(uint64_t ballot) {
  return static_cast<int>(__builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(ballot >> 32),
                                                    __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(ballot), 0)));
}

// Orders the wave's LDS accesses: they run in order, and the compiler keeps them so.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// NW waves a row, ROWS rows a workgroup (each of one wave).  kWide: fp32 logits,
// 4 a granule, else bf16, 8 a granule.  RD granules of a lane are in registers at a time (a tile).
template <bool kWide, int NW, int ROWS, int RD>
__global__ __launch_bounds__(64 * NW * ROWS) void token_logprob_kernel(const LogprobParams P) {
  static_assert(NW == 1 || ROWS == 1, "rows of a workgroup do not wait for each other");
  constexpr int GE = kWide ? 4 : 8;  // elements of a granule
  constexpr int TH = 64 * NW;
  constexpr int LE = RD * GE;        // elements of a lane's tile
  constexpr int W = NW * ROWS;
  constexpr int SUB = NW == 1 ? RD : 3;  // granules of a lane to a maximum that is kept
  constexpr int kKept = 24;          // maxima of a lane in LDS; each is of as many SUB granules as it takes
  static_assert(RD % SUB == 0);
  constexpr int kBatch = 8;          // lanes of a wave that have their granules in LDS at a time
  __shared__ float s_stat[NW][3];
  __shared__ uint32_t s_bound[NW][2];
  __shared__ int s_count;
  __shared__ uint64_t s_list[ROWS][kList];
  // several waves a row: the maxima of (lane, SUB granules) pairs, their orders' upper halves, and those pairs that are
  // read again
  __shared__ uint16_t s_max[NW == 1 ? 1 : W][kKept][64];
  __shared__ uint16_t s_pair[NW == 1 ? 1 : W][kPairs];
  // one wave a row: the granules of lanes with candidates
  __shared__ u32x4_t s_gran[NW == 1 ? W : 1][kBatch][RD];
  const int wg_wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wave = wg_wave % NW;  // of the row
  const uint32_t item = blockIdx.x * ROWS + wg_wave / NW;
  if (item >= P.items) return;  // only where a row is one wave
  uint64_t* const list = s_list[wg_wave / NW];
  [[maybe_unused]] int* const count = &s_count;  // candidates of a row of several waves; past kList they are only counted
  if (NW > 1 && wave == 0 && lane == 0) *count = 0;
  const int V = P.vocab, k = P.top_k;
  const char* row = static_cast<const char*>(P.logits) +
                    (item / P.bl * P.seq_stride + item % P.bl * P.pos_stride) * (kWide ? 4 : 2);
  // granules are 16-byte aligned; the first and the last may reach over the row's
  // ends, by less than a granule, so never into a page that the row has no part of
  const int head = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15u) / (kWide ? 4 : 2));
  const char* base = row - head * (kWide ? 4 : 2);
  const int n_gran = static_cast<int>((static_cast<int64_t>(V) + head + GE - 1) / GE);
  const int64_t token = P.tokens[item];
  const float x_token = element<kWide>(row, min(max(token, int64_t{0}), int64_t{V - 1}));  // asked for before the row is

  float m = -INFINITY, s = 0.f, t = 0.f;  // of this lane: maximum, sum 2^d, sum d 2^d, d = (x - m) log2(e)
  uint32_t best_bound = kNone;            // order of T
  int n_list = 0;                         // candidates; past kList they are only counted
  int g0 = wave * 64;
  const int fold = (n_gran + SUB * TH * kKept - 1) / (SUB * TH * kKept);  // times SUB granules to a maximum in LDS
  int kept = 0, folds = 0;                                                // maxima there, and how often the last one was raised
  float folded = -INFINITY;
  // Order of the wave's n-th largest lane maximum (below kNone if it has fewer lanes).
  auto nth_maximum = [&](int n) {
    constexpr int kBits = kWide ? 32 : 16;  // of the order that a value of the type has
    const uint32_t mine = wave * 64 + lane < n_gran ? order_of(m) >> (32 - kBits) : 0;
    uint32_t o = 0;
#pragma unroll
    for (int b = kBits - 1; b >= 0; --b) {
      const uint32_t with = o | 1u << b;
      if (__popcll(__ballot(mine >= with)) >= n) o = with;
    }
    // exactly that value's order: the lower half of a bf16's is all ones where it is negative
    return kWide ? o : o << 16 | (o >> 15 ? 0u : 0xffffu);
  };
  auto append = [&](bool take, float x, int index) {
    const uint64_t taken = __ballot(take);
    if (taken == 0) return;
    int at = n_list;
    if constexpr (NW > 1) {
      if (lane == 0) at = atomicAdd(count, __popcll(taken));
      at = __builtin_amdgcn_readfirstlane(at);
    }
    const int to = at + below(taken);
    if (take && to < kList) list[to] = key_of(x, index);
    n_list += __popcll(taken);
  };
  while (g0 < n_gran) {
    const int rounds = min(RD, (n_gran - g0 + TH - 1) / TH);  // of this wave
    // Granule j of this lane's tile: g0 + lane + j * TH.  All are requested at once, without a branch (past the row's
    // end the last one again): the wave waits once.
    u32x4_t raw[RD];
    const char* const from = base + static_cast<int64_t>(g0) * 16;
#pragma unroll
    for (int j = 0; j < RD; ++j)
      raw[j] = *reinterpret_cast<const u32x4_t*>(from + static_cast<uint32_t>(min(lane + j * TH, n_gran - 1 - g0)) * 16u);
    auto value = [&](int j, int e) {
      if constexpr (kWide) return __uint_as_float(raw[j][e]);
      return (e & 1) ? bf16hi(raw[j][e >> 1]) : bf16lo(raw[j][e >> 1]);
    };
    // Elements before the row's start and behind its end become -inf: only the rounds
    // that hold the row's first granule or reach its last one have any.
#pragma unroll
    for (int j = 0; j < RD; ++j) {
      const int gj = g0 + j * TH;
      if (j < rounds && ((gj == 0 && head > 0) || n_gran - gj <= 64)) {
        const int i0 = (gj + lane) * GE - head;
#pragma unroll
        for (int e = 0; e < GE; ++e) {
          if (i0 + e >= 0 && i0 + e < V) continue;
          if constexpr (kWide)
            raw[j][e] = 0xff800000u;
          else
            raw[j][e >> 1] = (e & 1) ? (raw[j][e >> 1] & 0xffffu) | 0xff800000u : (raw[j][e >> 1] & 0xffff0000u) | 0xff80u;
        }
      }
    }
    float tm = -INFINITY;
#pragma unroll
    for (int j0 = 0; j0 < RD; j0 += SUB) {
      float sm = -INFINITY;
#pragma unroll
      for (int j = j0; j < j0 + SUB; ++j) {
        if (j < rounds) {
#pragma unroll
          for (int e = 0; e < GE; e += 2) sm = max3(sm, value(j, e), value(j, e + 1));
        }
      }
      tm = fmaxf(tm, sm);
      if (NW > 1 && k > 0 && j0 < rounds) {
        folded = fmaxf(folded, sm);
        s_max[wg_wave][kept][lane] = static_cast<uint16_t>(order_of(folded) >> 16);
        if (++folds == fold) {
          folded = -INFINITY;
          folds = 0;
          ++kept;
        }
      }
    }
    const float mn = fmaxf(m, tm);
    rescale(s, t, m, mn);
    m = mn;
    if (__builtin_expect(!__any(fabsf(m) > kHuge && m != -INFINITY), 1)) {
      const float c = shift_of(m);
#pragma unroll
      for (int j = 0; j < RD; ++j) {
        if (j < rounds) {
#pragma unroll
          for (int e = 0; e < GE; ++e) {
            const float d = __builtin_fmaf(value(j, e), kLog2e, -c);
            const float p = __builtin_amdgcn_exp2f(d);
            s += p;
            t = __builtin_fmaf(fmaxf(d, kGone), p, t);
          }
        }
      }
    } else {
      const float c = shift_of(m), far = fabsf(m) > kHuge && m != -INFINITY ? m : INFINITY;
#pragma unroll
      for (int j = 0; j < RD; ++j) {
        if (j < rounds) {
#pragma unroll 1
          for (int e = 0; e < GE; ++e) {
            const uint32_t w = raw[j][kWide ? e : e >> 1];
            const float x = kWide ? __uint_as_float(w) : (e & 1) ? bf16hi(w) : bf16lo(w);
            const float d = far != INFINITY ? (x - far) * kLog2e : __builtin_fmaf(x, kLog2e, -c);
            const float p = __builtin_amdgcn_exp2f(d);
            s += p;
            t = __builtin_fmaf(fmaxf(d, kGone), p, t);
          }
        }
      }
    }
    if constexpr (NW == 1) {
      if (k > 0) {
        best_bound = max(nth_maximum(k), kNone);
        const float limit = value_of(best_bound);
        uint64_t lanes = __ballot(tm >= limit && tm > -INFINITY);
        while (lanes != 0) {
          // the next kBatch candidate lanes put their granules into LDS
          const int slot = below(lanes);
          if ((lanes >> lane & 1) && slot < kBatch) {
#pragma unroll
            for (int j = 0; j < RD; ++j) s_gran[wg_wave][slot][j] = raw[j];
          }
          wave_fence();
#pragma unroll 1
          for (int b = 0; b < kBatch && lanes != 0; ++b) {
            const int from_lane = __ffsll(static_cast<unsigned long long>(lanes)) - 1;
            lanes &= lanes - 1;
#pragma unroll
            for (int e0 = 0; e0 < LE; e0 += 64) {  // element e of the lane's tile is e % GE of its granule e / GE
              const int e = e0 + lane, index = (g0 + from_lane + e / GE * TH) * GE + e % GE - head;
              float x = -INFINITY;
              if (e < LE) {
                if constexpr (kWide)
                  x = reinterpret_cast<const float*>(s_gran[wg_wave][b])[e];
                else
                  x = bf16_to_f32(reinterpret_cast<const uint16_t*>(s_gran[wg_wave][b])[e]);
              }
              append(x >= limit && x > -INFINITY && index >= 0 && index < V, x, index);
            }
          }
          wave_fence();
        }
      }
    }
    g0 += RD * TH;
  }
  // Reads the pairs that reach `limit` again and appends their elements that do.
  [[maybe_unused]] auto collect = [&](float limit) {
    int n_pair = 0;
    wave_fence();
    for (int i = 0; i < kept + (folds > 0); ++i) {
      const uint32_t o = s_max[wg_wave][i][lane];
      const bool take = o >= best_bound >> 16 && o > kNone >> 16;
      const uint64_t taken = __ballot(take);
      const int to = n_pair + below(taken);
      if (take && to < kPairs) s_pair[wg_wave][to] = static_cast<uint16_t>(i * 64 + lane);
      n_pair += __popcll(taken);
    }
    wave_fence();
    if (n_pair > kPairs) {  // as many equal ones at least: the list is given up
      if (lane == 0) atomicAdd(count, kList + 1);
      return;
    }
    const int per = SUB * GE * fold, n = n_pair * per;  // element f of the pairs: e = f % per of pair f / per
    constexpr int kAhead = 4;
    for (int f0 = 0; f0 < n; f0 += 64 * kAhead) {
      float x[kAhead];
      int index[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const int f = min(f0 + 64 * a + lane, n);
        const int pair = min(f, n - 1) / (fold == 1 ? SUB * GE : per), e = f - pair * per;
        const int id = s_pair[wg_wave][pair];
        const int granule = wave * 64 + (id & 63) + (id / 64 * fold * SUB + e / GE) * TH;
        index[a] = granule * GE + e % GE - head;
        x[a] = -INFINITY;
        if (f < n && index[a] >= 0 && index[a] < V) x[a] = element<kWide>(row, index[a]);
      }
#pragma unroll
      for (int a = 0; a < kAhead; ++a) append(x[a] >= limit && x[a] > -INFINITY, x[a], index[a]);
    }
  };

  // join: lanes, then waves
  auto larger = [](float a, float b) { return fmaxf(a, b); };
  auto plus = [](float a, float b) { return a + b; };
  const float wm = wave_reduce(m, larger);
  rescale(s, t, m, wm);
  s = wave_reduce(s, plus);
  t = wave_reduce(t, plus);
  float M = wm, S = s, T = t;
  if constexpr (NW > 1) {
    if (lane == 0) {
      s_stat[wave][0] = wm;
      s_stat[wave][1] = s;
      s_stat[wave][2] = t;
    }
    if (k > 0) {
      // Some wave has k lanes that reach its k-th largest maximum, and together they have k that reach the smallest
      // of their (k / NW)-th largest: both bound the row's k-th largest from below.
      const uint32_t kth = nth_maximum(k), part = nth_maximum((k + NW - 1) / NW);
      if (lane == 0) {
        s_bound[wave][0] = kth;
        s_bound[wave][1] = part;
      }
    }
    __syncthreads();
    if (k > 0) {
      uint32_t lowest = ~0u;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        best_bound = max(best_bound, s_bound[w][0]);
        lowest = min(lowest, s_bound[w][1]);
      }
      best_bound = __builtin_amdgcn_readfirstlane(max(best_bound, lowest));
      collect(value_of(best_bound));
      __syncthreads();
    }
    if (wave != 0) return;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, s_stat[w][0]);
    S = T = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      float ws = s_stat[w][1], wt = s_stat[w][2];
      rescale(ws, wt, s_stat[w][0], M);
      S += ws;
      T += wt;
    }
  }
  const float log2_s = __log2f(S);
  const float log_s = (log2_s - left_of(M)) * kLn2;
  if (lane == 0) {
    P.entropy[item] = (log2_s - T / S) * kLn2;
    P.logprob[item] = token < 0 ? 0.f : token >= V ? NAN : (x_token - M) - log_s;
  }
  if (k == 0) return;

  int n = NW == 1 ? n_list : __builtin_amdgcn_readfirstlane(*count);
  // a signalling NaN hides what a lane's maximum had seen before it: T still holds, the candidates may not
  if (S != S) n = kList + 1;
  if (n < k || n > kList) {
    // Fewer than k above -inf: the first ones at -inf (or NaN, which ranks there) follow.
    // Too many at or above the bound: those above it, and the first k that equal it.
    const bool rest = n < k;
    int n_equal = rest ? n : 0;
    if (!rest) n = 0;
    for (int i0 = 0; i0 < V && !(rest && n_equal >= k); i0 += 64) {
      const int i = i0 + lane;
      const float x = i < V ? element<kWide>(row, i) : 0.f;
      const uint32_t o = i < V ? order_of(x) : 0;
      const uint64_t equal = __ballot(o == best_bound);
      const bool take = (!rest && o > best_bound) || (o == best_bound && n_equal + below(equal) < k);
      const uint64_t taken = __ballot(take);
      const int to = n + below(taken);
      if (take && to < kList) list[to] = key_of(x, i);
      n += __popcll(taken);
      n_equal += __popcll(equal);
    }
    wave_fence();
  }
  float* top_logprob = P.top_logprob + static_cast<int64_t>(item) * k;
  int64_t* top_token = P.top_token + static_cast<int64_t>(item) * k;
  auto store = [&](int rank, uint64_t key) {
    const int index = static_cast<int>(0xffffffffu - static_cast<uint32_t>(key));
    top_logprob[rank] = (value_of(static_cast<uint32_t>(key >> 32)) - M) - log_s;  // a NaN's is -inf, but then log_s is NaN
    top_token[rank] = index;
  };
  if (n <= kList) {
    for (int i = lane; i < n; i += 64) {
      const uint64_t key = list[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += list[j] > key;
      if (rank < k) store(rank, key);
    }
    return;
  }
  // more than kList above the bound (the best ones packed into few lanes): k
  // passes, each for the largest key below the last one
  uint64_t last = ~0ull;
  for (int r = 0; r < k; ++r) {
    uint64_t best = 0;
    for (int i = lane; i < V; i += 64) {
      const uint64_t key = key_of(element<kWide>(row, i), i);
      if (key < last && key > best) best = key;
    }
    for (int d = 1; d < 64; d <<= 1) {
      const uint64_t o = __shfl_xor(best, d);
      best = o > best ? o : best;
    }
    last = best;
    if (lane == 0) store(r, best);
  }
}

template <bool kWide, int NW, int ROWS, int RD>
void launch(const LogprobParams& P, hipStream_t st) {
  hipLaunchKernelGGL((token_logprob_kernel<kWide, NW, ROWS, RD>), dim3((P.items + ROWS - 1) / ROWS), dim3(64 * NW * ROWS),
                     0, st, P);
}

// One wave a row where there are rows enough to fill the chip so (six a CU), or
// where a row is little work: what a wave does once (the search for T, the joins) is
// most of a short tile's work, and no workgroup waits.  Else eight waves a row.
// Tiles are as long as the row needs, up to 17 granules a lane (five waves a SIMD).
// us a call, one wave / eight, eight alternatives: 64 rows of 8194 bf16 10.2 / 7.0, 512 10.8 / 8.8, 1024 12.4 / 12.7,
// 2048 15.6 / 21.1, 16384 57 / 148; 1024 of 20000 22.0 / 18.5, 2048 25.8 / 30.8; 1024 of 16000 fp32 22.8 / 19.7, 4000
// 53.6 / 58.2; 512 of 300 4.6 / 6.3.  Rows of more than four such tiles keep eight waves at any number: 1024 of 60000
// 41.1 / 29.7, 3000 75.6 / 75.0.
// 17 granules are the speech vocabulary's row of 8194 bf16 (1025 granules, 16.02 a lane).  A row just longer takes a second
// tile of as many loads, most of them the last granule again: 2048 rows of 8704 15.6 us, of 8800 17.0, of 10000 18.4; 16384 rows
// 57.7, 63.1, 69.5, a step of 8 %.
// Between 512 and some thousand rows neither form fills the chip: at 2048 rows of 8194 (15.7 us; the bytes alone 6.5) one wave a
// row leaves a SIMD two waves, and what a row does once is exposed; two or four waves a row are not built there.
template <bool kWide>
void launch_rows(const LogprobParams& P, hipStream_t st) {
  const int64_t granules = (static_cast<int64_t>(P.vocab) + (kWide ? 3 : 7)) / (kWide ? 4 : 8) + 1;
  if (granules <= 3 * 64) {
    launch<kWide, 1, 4, 3>(P, st);
  } else if (P.items >= 1536 && granules <= 4 * 17 * 64) {
    if (granules <= 9 * 64)
      launch<kWide, 1, 4, 9>(P, st);
    else
      launch<kWide, 1, 4, 17>(P, st);
  } else if (granules <= 3 * 512) {
    launch<kWide, 8, 1, 3>(P, st);
  } else {
    launch<kWide, 8, 1, 9>(P, st);
  }
}

}  // namespace
}  // namespace yapd

extern "C" int yapd_token_logprobs(const void* logits, int wide, int64_t seq_stride, int64_t pos_stride, int rows, int bl,
                                   int vocab, const int64_t* tokens, int top_k, float* logprob, float* entropy,
                                   float* top_logprob, int64_t* top_token, void* stream) {
  YAPD_REQUIRE(rows >= 0 && bl >= 0, "token_logprobs: need rows and bl >= 0 (got %d, %d)", rows, bl);
  const int64_t items = static_cast<int64_t>(rows) * bl;
  YAPD_REQUIRE(items < (int64_t{1} << 22), "token_logprobs: rows * bl must be below 2^22");
  YAPD_REQUIRE(vocab >= 1 && vocab <= (1 << 30), "token_logprobs: need 1 <= vocab <= 2^30 (got %d)", vocab);
  YAPD_REQUIRE(top_k >= 0 && top_k <= yapd::kMaxTop && top_k <= vocab,
               "token_logprobs: top_k must be in [0, min(%d, vocab)] (got %d)", yapd::kMaxTop, top_k);
  if (items == 0) return YAPD_OK;
  YAPD_REQUIRE(logits && tokens && logprob && entropy && (top_k == 0 || (top_logprob && top_token)),
               "token_logprobs: NULL pointer");
  YAPD_REQUIRE((reinterpret_cast<uintptr_t>(logits) & (wide ? 3u : 1u)) == 0, "token_logprobs: misaligned logits");
  const yapd::LogprobParams P{logits, seq_stride, pos_stride, static_cast<uint32_t>(items), static_cast<uint32_t>(bl),
                              vocab, top_k, tokens, logprob, entropy, top_logprob, top_token};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (wide)
    yapd::launch_rows<true>(P, st);
  else
    yapd::launch_rows<false>(P, st);
  YAPD_LAUNCH_CHECK("token_logprob_kernel launch");
  return YAPD_OK;
}
