// Log probabilities of given tokens, with the entropy and the best alternatives.
//
// For a row x of V logits and its token t, with m = max x:
//   logZ = m + ln S,  S = sum e^(x - m)
//   logprob = x_t - logZ,  entropy = ln S - (sum (x - m) e^(x - m)) / S,
//   the k largest x (ties: the lowest index first) minus logZ.
// One workgroup a row, one pass over it: every lane keeps the running maximum
// and the two sums over its 16-byte granules, rescaled when the maximum grows;
// they are joined across lanes on DPP and across waves in LDS.  x - m is taken
// before its scaling to log2: rows at the type's largest or lowest value stay finite.
//
// The best k need no second pass: at least k elements reach the k-th largest
// of a wave's lane maxima (a binary search over ballots), so only elements at
// or above that are candidates -- a few more than k of them -- and go to a list in LDS
// with their index.  After the join only those that reach the largest of the
// waves' bounds are left, and each counts the keys above its own: that is its
// rank.  A row whose candidates do not fit (thousands of equal logits, such as
// a mask that leaves fewer than k tokens) takes k passes of a plain search.
#include <cmath>

#include "attn_tile.h"
#include "common.h"

namespace yapd {
namespace {

constexpr int kMaxTop = 32;
constexpr int kList = 1024;   // candidates of a row
constexpr int kFinal = 256;   // ... that reach the largest bound
constexpr float kLn2 = 0.6931471805599453f, kLog2e = 1.4426950408889634f;
constexpr float kGone = -150.f;  // e^kGone is 0 in fp32: a bound for d where d e^d is 0, also at d = -inf

struct LogprobParams {
  const void* logits;
  int64_t seq_stride, pos_stride;  // elements
  uint32_t bl;
  int vocab, top_k;
  const int64_t* tokens;
  float* logprob;
  float* entropy;
  float* top_logprob;
  int64_t* top_token;
};

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false));
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

// The sums s, t taken against the maximum m, against `to` >= m instead.
__device__ __forceinline__ void rescale(float& s, float& t, float m, float to) {
  if (m == -INFINITY) return;  // no value above -inf yet: 0, or NaN if there was one
  const float down = m - to, a = __builtin_amdgcn_exp2f(down * kLog2e);
  t = (t + s * fmaxf(down, kGone)) * a;
  s *= a;
}

template <bool kWide>
__device__ __forceinline__ float element(const void* row, int64_t i) {
  if constexpr (kWide) return static_cast<const float*>(row)[i];
  return bf16_to_f32(static_cast<const uint16_t*>(row)[i]);
}

// NW waves a row.  kWide: fp32 logits, 4 a granule, else bf16, 8 a granule.
// RD granules of a lane are in registers at a time (a tile).
template <bool kWide, int NW, int RD>
__global__ __launch_bounds__(64 * NW) void token_logprob_kernel(const LogprobParams P) {
  constexpr int GE = kWide ? 4 : 8;  // elements of a granule
  constexpr int TH = 64 * NW;
  __shared__ float s_stat[NW][3];
  __shared__ uint32_t s_bound[NW];
  __shared__ uint64_t s_list[kList];
  __shared__ uint64_t s_final[kFinal];
  __shared__ int s_count[2];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int64_t item = blockIdx.x;
  const int V = P.vocab, k = P.top_k;
  const char* row = static_cast<const char*>(P.logits) +
                    (blockIdx.x / P.bl * P.seq_stride + blockIdx.x % P.bl * P.pos_stride) * (kWide ? 4 : 2);
  // granules are 16-byte aligned; the first and the last may reach over the row's
  // ends, by less than a granule, so never into a page that the row has no part of
  const int head = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15u) / (kWide ? 4 : 2));
  const char* base = row - head * (kWide ? 4 : 2);
  const int n_gran = static_cast<int>((static_cast<int64_t>(V) + head + GE - 1) / GE);
  const int64_t token = P.tokens[item];
  if (threadIdx.x < 2) s_count[threadIdx.x] = 0;
  if (k > 0) __syncthreads();

  float m = -INFINITY, s = 0.f, t = 0.f;  // of this lane: maximum, sum e^d, sum d e^d, d = x - m
  uint32_t bound = 0;  // upper half of the order of the wave's k-th largest lane maximum so far
  for (int g0 = 0; g0 < n_gran; g0 += RD * TH) {
    const int gl = g0 + threadIdx.x;  // granule j of this lane: gl + j * TH
    const int rounds = min(RD, (n_gran - g0 - (wave << 6) + TH - 1) / TH);  // of this wave; <= 0: none
    if (rounds <= 0) break;
    u32x4_t raw[RD];
#pragma unroll
    for (int j = 0; j < RD; ++j) {
      const uint32_t none = kWide ? 0xff800000u : 0xff80ff80u;  // -inf
      raw[j] = u32x4_t{none, none, none, none};
      if (j < rounds && gl + j * TH < n_gran)
        raw[j] = *reinterpret_cast<const u32x4_t*>(base + static_cast<int64_t>(gl + j * TH) * 16);
    }
    auto value = [&](int j, int e) {
      if constexpr (kWide) return __uint_as_float(raw[j][e]);
      return (e & 1) ? bf16hi(raw[j][e >> 1]) : bf16lo(raw[j][e >> 1]);
    };
    // elements before the row's start and behind its end: -inf
#pragma unroll
    for (int j = 0; j < RD; ++j) {
      const int i0 = (gl + j * TH) * GE - head;
      if (j < rounds && __any(i0 < 0 || (i0 < V && i0 + GE > V))) {
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
    float gm[RD], mn = m;
#pragma unroll
    for (int j = 0; j < RD; ++j) {
      gm[j] = -INFINITY;
      if (j < rounds) {
#pragma unroll
        for (int e = 0; e < GE; ++e) gm[j] = fmaxf(gm[j], value(j, e));
        mn = fmaxf(mn, gm[j]);
      }
    }
    // nothing above -inf yet: exponents against 0 give sums of 0 instead of NaN
    const float c = mn == -INFINITY ? 0.f : mn;
    rescale(s, t, m, mn);
    m = mn;
#pragma unroll
    for (int j = 0; j < RD; ++j) {
      if (j < rounds) {
#pragma unroll
        for (int e = 0; e < GE; ++e) {
          const float d = value(j, e) - c;
          const float p = __builtin_amdgcn_exp2f(d * kLog2e);
          s += p;
          t = __builtin_fmaf(fmaxf(d, kGone), p, t);
        }
      }
    }
    if (k > 0) {
      const uint32_t mine = threadIdx.x < n_gran ? order_of(m) >> 16 : 0;
      bound = 0;
#pragma unroll
      for (int b = 15; b >= 0; --b) {
        const uint32_t c16 = bound | 1u << b;
        if (__popcll(__ballot(mine >= c16)) >= k) bound = c16;
      }
      const float limit = bound == 0 ? -INFINITY : value_of(bound << 16);
#pragma unroll
      for (int j = 0; j < RD; ++j) {
        if (j < rounds && __any(!(gm[j] < limit))) {
          const int i0 = (gl + j * TH) * GE - head;
#pragma unroll
          for (int e = 0; e < GE; ++e) {
            const float x = value(j, e);
            if (!(x < limit) && i0 + e >= 0 && i0 + e < V) {
              const int at = atomicAdd(&s_count[0], 1);
              if (at < kList) s_list[at] = key_of(x, i0 + e);
            }
          }
        }
      }
    }
  }

  // join: lanes, then waves
  auto larger = [](float a, float b) { return fmaxf(a, b); };
  auto plus = [](float a, float b) { return a + b; };
  const float wm = wave_reduce(m, larger);
  rescale(s, t, m, wm);
  s = wave_reduce(s, plus);
  t = wave_reduce(t, plus);
  if (lane == 0) {
    s_stat[wave][0] = wm;
    s_stat[wave][1] = s;
    s_stat[wave][2] = t;
    s_bound[wave] = bound;
  }
  __syncthreads();
  float M = -INFINITY;
  uint32_t top_bound = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    M = fmaxf(M, s_stat[w][0]);
    top_bound = max(top_bound, s_bound[w]);
  }
  float S = 0.f, T = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    float ws = s_stat[w][1], wt = s_stat[w][2];
    rescale(ws, wt, s_stat[w][0], M);
    S += ws;
    T += wt;
  }
  const float log_s = __log2f(S) * kLn2;
  if (threadIdx.x == 0) {
    P.entropy[item] = log_s - T / S;
    P.logprob[item] = token < 0 ? 0.f : token >= V ? NAN : (element<kWide>(row, token) - M) - log_s;
  }
  if (k == 0) return;

  float* top_logprob = P.top_logprob + item * k;
  int64_t* top_token = P.top_token + item * k;
  auto store = [&](int rank, uint64_t key) {
    const int index = static_cast<int>(0xffffffffu - static_cast<uint32_t>(key));
    top_logprob[rank] = (element<kWide>(row, index) - M) - log_s;
    top_token[rank] = index;
  };
  const int n_list = s_count[0];
  if (n_list <= kList) {
    for (int i = threadIdx.x; i < n_list; i += TH) {
      const uint64_t key = s_list[i];
      if (static_cast<uint32_t>(key >> 48) >= top_bound) {
        const int at = atomicAdd(&s_count[1], 1);
        if (at < kFinal) s_final[at] = key;
      }
    }
    __syncthreads();
    const int n = s_count[1];
    if (n <= kFinal) {
      for (int i = threadIdx.x; i < n; i += TH) {
        const uint64_t key = s_final[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += s_final[j] > key;
        if (rank < k) store(rank, key);
      }
      return;
    }
  }
  // k passes, each for the largest key below the last one
  uint64_t last = ~0ull;
  __syncthreads();
  for (int r = 0; r < k; ++r) {
    uint64_t best = 0;
    for (int i = threadIdx.x; i < V; i += TH) {
      const uint64_t key = key_of(element<kWide>(row, i), i);
      if (key < last && key > best) best = key;
    }
    for (int d = 1; d < 64; d <<= 1) {
      const uint64_t o = __shfl_xor(best, d);
      best = o > best ? o : best;
    }
    if (lane == 0) s_list[wave] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; ++w) best = s_list[w] > best ? s_list[w] : best;
    last = best;
    if (threadIdx.x == 0) store(r, best);
    __syncthreads();
  }
}

template <bool kWide, int NW, int RD>
void launch(const LogprobParams& P, int64_t items, hipStream_t st) {
  hipLaunchKernelGGL((token_logprob_kernel<kWide, NW, RD>), dim3(static_cast<unsigned>(items)), dim3(64 * NW), 0, st, P);
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
  yapd::LogprobParams P{logits, seq_stride, pos_stride, static_cast<uint32_t>(bl), vocab, top_k, tokens, logprob, entropy,
                          top_logprob, top_token};
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (wide)
    yapd::launch<true, 8, 9>(P, items, st);
  else
    yapd::launch<false, 4, 5>(P, items, st);
  YAPD_LAUNCH_CHECK("token_logprob_kernel launch");
  return YAPD_OK;
}
