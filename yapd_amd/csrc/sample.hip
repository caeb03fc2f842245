// Tokens drawn from logits with given random numbers: temperature, top-k, top-p and min-p.
//
// A row's tokens in order (larger logit first, of equal ones the lower index) have the weights
//   w_i = e^((x_i - max) / T);  W(n) = the sum of the first n.
// Each filter keeps a prefix of that order: top-k the first k; top-p the shortest whose weight is at least p W(k); min-p
// the tokens of w_i >= min_p.  So all three together keep the shortest, whose weight is the least, Z = min(W(k), W_p,
// W_m), and the token is the first whose inclusive sum exceeds u Z.  No token's membership is ever asked: three
// sums are looked for, in the same order.
//
// The row is not sorted, in either of two forms:
//   bf16 (sample_values): a bin a value.  Elements are counted, never weighed one by one; a value's weight is computed
//     once, in fp64, and is right to 4e-12 (an exponential to 2e-13, carried along 15 values by a ratio of that
//     precision).  Sums go by bins in a fixed order, so nothing depends on the order of atomics.
//   fp32, and bf16 rows outside sample_values' window: four bins a thread of equal width in x (in fp32, which keeps the
//     order).  The bins' prefix sums find the bin where a sum crosses a target, and that bin's elements, usually a few
//     dozen, go to a list where each adds up what precedes it.  A bin of more than kList elements (many equal or
//     nearly equal logits) is divided again, by the bits of (value, index), 10 to 12 a time.  Weights are fixed-point
//     numbers of 64 bits, rounded from exponentials right to 2e-13: their sums are exact, so they do not depend on the
//     order of LDS atomics either, and a border is off by V roundings of 2^-52 to 2^-39 besides.
//
// Measured, on the GPU alone.  One bf16 row of 8194: 10 us, a chain of some 15 steps between barriers, as long for
// any number of rows up to the CUs'.  4096 of them with all three filters, each row its own: 69 us, where the
// bytes take 13: four workgroups a CU, of whose time the vector unit's instructions are half and counting in LDS (two
// atomics a word) nearly as much, and each row's chain is hidden by three others only.  fp32, a row of 100003: 15 us for the
// largest, 50 with a temperature, 57 with top-p (three passes; instructions bound it: 67 an element before its weight was a
// polynomial within its bin, then 62 us).  300 such rows, 120 MB, 23 us as bytes: 110 us with a temperature, all filters with a
// small top-k 88 (300 rows on 256 CUs are two turns, and every pass fetches the rows again), settings of their own 103
// as the rows come and 75 the costliest first.
#include "attn_tile.h"
#include "common.h"

namespace yapd {
namespace {

constexpr int kList = 256;
constexpr double kLn2 = 0.69314718055994530942, kLog2e = 1.44269504088896340736;

struct SampleParams {
  const void* logits;
  int64_t seq_stride, pos_stride;  // elements
  uint32_t items, bl;
  int vocab;
  int shift;  // weights are multiples of 2^-shift
  const float* u;
  const float* temperature;  // [items], or NULL: the number beside it
  float temperature_all;
  const int32_t* top_k;
  int top_k_all;
  const float* top_p;
  float top_p_all;
  const float* min_p;
  float min_p_all;
  bool by_cost;  // rows are taken by cost (row_by_cost)
  int64_t* token;
  float* logprob;
};

// Floats as unsigned numbers in their order (-0 taken as +0).
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
// Larger value first, then lower index: descending numbers.
__device__ __forceinline__ uint64_t key_of(float x, int index) {
  return static_cast<uint64_t>(order_of(x)) << 32 | (0xffffffffu - static_cast<uint32_t>(index));
}

__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t o = static_cast<uint32_t>(key >> 32);
  return __uint_as_float(o ^ (o >> 31 ? 0x80000000u : 0xffffffffu));
}

// The largest and the least of three without quieting the operands first (they come from memory, so the compiler
// would); a NaN operand is left out.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float r;
  asm("v_min3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// 2^-t as a multiple of 2^-shift, for t >= 0: with r = t rounded, f = t - r, the Taylor polynomial of e^(-f ln 2)
// (|f ln 2| <= 0.347: off by 2e-13), rounded to an integer by adding 2^52.
__device__ __forceinline__ uint64_t weight_of(double t, int shift) {
  t = fmin(t, 100.0);  // 0 from 64 on
  const double r = __builtin_rint(t);
  const double a = (r - t) * kLn2;
  double p = 1.0 / 3628800;
  p = __builtin_fma(p, a, 1.0 / 362880);
  p = __builtin_fma(p, a, 1.0 / 40320);
  p = __builtin_fma(p, a, 1.0 / 5040);
  p = __builtin_fma(p, a, 1.0 / 720);
  p = __builtin_fma(p, a, 1.0 / 120);
  p = __builtin_fma(p, a, 1.0 / 24);
  p = __builtin_fma(p, a, 1.0 / 6);
  p = __builtin_fma(p, a, 0.5);
  p = __builtin_fma(p, a, 1.0);
  p = __builtin_fma(p, a, 1.0);
  const double v = __builtin_ldexp(p, shift - static_cast<int>(r)) + 0x1p52;
  return __builtin_bit_cast(uint64_t, v) - (uint64_t{0x433} << 52);
}

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int d) {
  const uint32_t lo = __shfl_up(static_cast<uint32_t>(v), d), hi = __shfl_up(static_cast<uint32_t>(v >> 32), d);
  return static_cast<uint64_t>(hi) << 32 | lo;
}
__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int d) {
  const uint32_t lo = __shfl_xor(static_cast<uint32_t>(v), d), hi = __shfl_xor(static_cast<uint32_t>(v >> 32), d);
  return static_cast<uint64_t>(hi) << 32 | lo;
}

enum Cross { kCount, kReach, kExceed };  // the first element whose inclusive count, or sum, is at least, or exceeds, a target

constexpr int kValues = 4096;             // bins of the bf16 form: one a value, 2047 on either side of the tiny ones
constexpr int kTiny = kValues / 2, kLow = kValues - 1;  // low ones are counted in kLow + lane: a mask's in one word would queue there
constexpr int kFloor = (127 - 10) * 128;  // |x| <= 2^-10 is tiny, 64 and above high: bits of the usual window's floor

template <int NT, bool kWide>
struct Shared {
  static constexpr int kBins = 4 * NT;
  union {
    struct {
      uint64_t mass[kBins], mass2[kBins];  // mass2 also holds keys, see `held`
      uint32_t count[kBins], count2[kBins];
    };
    uint32_t values[kValues + 63];
  };
  double power[kWide ? kBins : 1];  // the weight at a bin's begin, times 2^shift
  uint64_t key[kList], w[kList];
  uint64_t part[NT / 64], part2[NT / 64], z_min[NT / 64];
  double sum_a[NT / 64], sum_b[NT / 64];
  float fmx[NT / 64], fmn[NT / 64];
  uint32_t n, bad, n_held;
  // what a search found
  int bin;
  uint64_t base, sum;
  uint32_t base_count;
  uint64_t found;
  // the bf16 form's
  uint32_t first, bits, nth, ties, mixed;
  double z;
};

typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// 2^-t in 64 bits (0 from t = 1000 on), t >= 0: weight_of's polynomial.
__device__ __forceinline__ double exp2_neg(double t) {
  t = fmin(t, 1000.0);
  const double r = __builtin_rint(t), a = (r - t) * kLn2;
  double p = 1.0 / 3628800;
  p = __builtin_fma(p, a, 1.0 / 362880);
  p = __builtin_fma(p, a, 1.0 / 40320);
  p = __builtin_fma(p, a, 1.0 / 5040);
  p = __builtin_fma(p, a, 1.0 / 720);
  p = __builtin_fma(p, a, 1.0 / 120);
  p = __builtin_fma(p, a, 1.0 / 24);
  p = __builtin_fma(p, a, 1.0 / 6);
  p = __builtin_fma(p, a, 0.5);
  p = __builtin_fma(p, a, 1.0);
  p = __builtin_fma(p, a, 1.0);
  return t >= 1000.0 ? 0.0 : __builtin_ldexp(p, -static_cast<int>(r));
}

struct Settings {
  float T;
  int k;
  float top_p, min_p, u;
};

// Rows of bf16 logits, where a bin is one value: 16 octaves of positive and of negative values from a floor 2^f on, with
// a bin for what is smaller in magnitude (tiny; also high and low, beyond the window; a row whose largest logit is outside it
// moves the window there and counts again).  Elements are only counted; a bin's weight is its count times its
// value's, the values of 16 consecutive bins being an arithmetic progression (so their weights are a geometric one),
// and of equal logits the n-th is found by division.  Tiny values other than 0 go to a list as they are counted and are
// weighed one by one; low ones weigh less than 2^-60 together.  false, for the general form: low values that
// weigh more, more tiny ones than the list holds, or a token among several values of the tiny bin.
template <int NT, int RD>
__device__ __forceinline__ bool sample_values(const SampleParams& P, Shared<NT, false>& S, const u32x4_t* granules, int off,
                                              int n_gran, const Settings& s, uint32_t item) {
  constexpr int kPer = kValues / NT;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int V = P.vocab;
  // Granules that the row fills, in tiles of RD a thread, requested together (a row of one tile stays in registers), and
  // those it fills in part, one each of the first two threads, with -inf for what is beside the row.
  const int f0 = off > 0 ? 1 : 0, n_full = max((off + V) / 8 - f0, 0);
  const bool tail = (off + V) % 8 != 0 && (n_gran > 1 || off == 0);
  const bool has_edge = (tid == 0 && off > 0) || (tid == 1 && tail);
  const int edge_gi = tid == 0 ? 0 : n_gran - 1;
  u32x4_t held[RD], edge = {0, 0, 0, 0};
  auto load_tile = [&](int t0) {
#pragma unroll
    for (int j = 0; j < RD; ++j) held[j] = granules[min(f0 + t0 + tid + j * NT, n_gran - 1)];
  };
  load_tile(0);
  if (has_edge) {
    edge = granules[edge_gi];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = edge_gi * 8 + e - off;
      if (i < 0 || i >= V)
        edge[e >> 1] = (edge[e >> 1] & (e & 1 ? 0x0000ffffu : 0xffff0000u)) | (e & 1 ? 0xff800000u : 0x0000ff80u);
    }
  }
  auto each = [&](auto f) {
    if (has_edge) f(edge, edge_gi * 8 - off);
    for (int t0 = 0; t0 < n_full; t0 += NT * RD) {
      if (n_full > NT * RD) load_tile(t0);
#pragma unroll
      for (int j = 0; j < RD; ++j)
        if (t0 + tid + j * NT < n_full) f(held[j], (f0 + t0 + tid + j * NT) * 8 - off);
    }
  };
  int fl = kFloor;
  // a word's two magnitudes in values above the floor, 0 for tiny ones
  auto above_floor = [&](u16x2 m) {
    const u16x2 f = {static_cast<unsigned short>(fl), static_cast<unsigned short>(fl)};
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(m, f) - f);
  };
  // their bins: kTiny less that number, with the sign
  auto bins_of = [&](uint32_t word, uint32_t above) {
    const s16x2 sign = __builtin_bit_cast(s16x2, word) >> 15;
    const s16x2 y = (__builtin_bit_cast(s16x2, above) ^ sign) - sign;
    const short end = static_cast<short>(kLow + lane);
    const s16x2 mid = {kTiny, kTiny}, top = {end, end}, zero = {0, 0};
    return __builtin_elementwise_max(__builtin_elementwise_min(__builtin_elementwise_sub_sat(mid, y), top), zero);
  };
  auto value_of_bin = [&](int b) {
    const int y = kTiny - b;
    return __uint_as_float(static_cast<uint32_t>(fl + (y < 0 ? -y : y)) << 16 | (y < 0 ? 0x80000000u : 0u));
  };

  uint32_t c[kPer];  // elements of this thread's bins, tid * kPer and on
  float mx = 0.f;
  uint32_t tiny;
  for (int round = 0;; ++round) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) S.values[tid + j * NT] = 0;
    if (tid < 63) S.values[kValues + tid] = 0;
    if (tid == 0) {
      S.first = kValues;
      S.bad = S.n = 0;
    }
    __syncthreads();
    u16x2 most = {0, 0};  // magnitudes: above 0x7f80 a NaN's
    each([&](const u32x4_t& v, int) {
      u16x2 least = {0xffff, 0xffff};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const u16x2 m = __builtin_bit_cast(u16x2, v[w] & 0x7fff7fffu);
        most = __builtin_elementwise_max(most, m);
        least = __builtin_elementwise_min(least, m);
        const uint32_t at = __builtin_bit_cast(uint32_t, bins_of(v[w], above_floor(m)) << 2);  // bytes
        char* const to = reinterpret_cast<char*>(S.values);
        atomicAdd(reinterpret_cast<uint32_t*>(to + (at & 0xffffu)), 1u);
        atomicAdd(reinterpret_cast<uint32_t*>(to + (at >> 16)), 1u);
      }
      if (min(least[0], least[1]) <= fl) {  // a tiny value
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t bits = e & 1 ? v[e >> 1] >> 16 : v[e >> 1] & 0xffffu;
          if (static_cast<int>(bits & 0x7fffu) > fl || (bits & 0x7fffu) == 0) continue;
          const uint32_t to = atomicAdd(&S.n, 1u);
          if (to < kList) S.key[to] = bits;
        }
      }
    });
    if (__any(most[0] > 0x7f80 || most[1] > 0x7f80) && lane == 0) atomicOr(&S.bad, 1u);
    __syncthreads();
    if (S.bad) {
      if (tid == 0) {
        P.token[item] = -1;
        P.logprob[item] = __builtin_nanf("");
      }
      return true;
    }
    uint32_t first = kValues;
#pragma unroll
    for (int j = 0; j < kPer; j += 4) {
      const u32x4_t four = *reinterpret_cast<const u32x4_t*>(&S.values[tid * kPer + j]);
#pragma unroll
      for (int i = 0; i < 4; ++i) c[j + i] = four[i];
    }
    if (tid == NT - 1) c[kPer - 1] = 0;
#pragma unroll
    for (int j = kPer - 1; j >= 0; --j)
      if (c[j]) first = tid * kPer + j;
    for (int d = 1; d < 64; d <<= 1) first = min(first, __shfl_xor(first, d));
    if (lane == 0) atomicMin(&S.first, first);
    tiny = S.values[kTiny];
    const uint32_t high = S.values[0];
    __syncthreads();
    first = S.first;
    if (high == 0 && first < kLow && first != kTiny) {
      mx = value_of_bin(first);
      break;
    }
    if (round > 0) break;  // the largest is 0 and the first bin the tiny one
    // a window around the largest logit
    float m = -INFINITY;
    each([&](const u32x4_t& v, int) {
#pragma unroll
      for (int w = 0; w < 4; ++w) m = fmaxf(m, fmaxf(bf16lo(v[w]), bf16hi(v[w])));
    });
    for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
    if (lane == 0) S.fmx[wave] = m;
    __syncthreads();
    for (int w = 0; w < NT / 64; ++w) m = fmaxf(m, S.fmx[w]);
    if (fabsf(m) == INFINITY) {
      if (tid == 0) {
        P.token[item] = -1;
        P.logprob[item] = __builtin_nanf("");
      }
      return true;
    }
    mx = m + 0.f;
    const int mag = static_cast<int>(__float_as_uint(m) >> 16 & 0x7fffu);
    if (mx > 0.f)
      fl = max((mag - 2047 + 127) & ~127, 0);
    else if (mx < 0.f)
      fl = (mag - 1) & ~127;
    if (fl + 2047 > 0x7f80) return false;  // -inf would not be low
    __syncthreads();
  }

  const bool greedy = !(s.T > 0.f) || s.k == 1;
  const double scale = greedy ? 0.0 : kLog2e / static_cast<double>(s.T);
  auto t_of = [&](float x) { return (static_cast<double>(mx) - static_cast<double>(x)) * scale; };
  const bool by_min = s.min_p > 0.f;
  const double min_p = fminf(s.min_p, 1.f);

  // Tiny values other than 0 were listed; low ones weigh nothing next to the largest, or the row goes to the general form.
  double tiny_mass = 0.0, tiny_min = 0.0;
  const uint32_t listed = S.n;
  if (tiny && !greedy) {
    if (listed > kList) return false;
    const double zero = exp2_neg(t_of(0.f));
    tiny_mass = static_cast<double>(tiny - listed) * zero;
    tiny_min = zero >= min_p ? tiny_mass : 0.0;
    if (listed) {  // every thread adds them up in one order: by their bits (equal ones weigh the same)
      for (uint32_t i = tid; i < listed; i += NT) {
        const uint64_t mine = S.key[i];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < listed; ++j) rank += S.key[j] < mine || (S.key[j] == mine && j < i);
        S.w[rank] = __builtin_bit_cast(uint64_t, exp2_neg(t_of(__uint_as_float(static_cast<uint32_t>(mine) << 16))));
      }
      __syncthreads();
      for (uint32_t i = 0; i < listed; ++i) {
        const double w = __builtin_bit_cast(double, S.w[i]);
        tiny_mass += w;
        tiny_min += w >= min_p ? w : 0.0;
      }
    }
  }
  // From 84 octaves below the largest on, 2^24 of them weigh less than 2^-60: what top-k and top-p keep of those counts
  // for nothing.  Masked tokens are there, as -inf or as the type's lowest value.
  constexpr double kFar = 60.0 + 24.0;
  if (!greedy && t_of(-__uint_as_float(static_cast<uint32_t>(fl + 2047) << 16)) < kFar) {
    // what is beside the row was counted by the first two threads
    const uint32_t pads = static_cast<uint32_t>((f0 + (tail ? 1 : 0)) * 8 - (V - n_full * 8));
    const uint32_t pads_head = off > 0 ? (tail ? off : pads) : 0;
    if (__any(S.values[kLow + lane] > (lane == 0 ? pads_head : lane == 1 ? pads - pads_head : 0))) {
      // magnitudes up to here, rounded up, are nearer than that
      const float far = static_cast<float>(kFar / scale - static_cast<double>(mx));
      const uint32_t near = min((__float_as_uint(far) >> 16) + 1, 0x7f7fu);
      bool counts = false;
      each([&](const u32x4_t& v, int) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const s16x2 b = bins_of(v[w], above_floor(__builtin_bit_cast(u16x2, v[w] & 0x7fff7fffu)));
          counts |= (b[0] >= kLow && (v[w] & 0x7fffu) <= near) || (b[1] >= kLow && (v[w] >> 16 & 0x7fffu) <= near);
        }
      });
      if (__any(counts) && lane == 0) atomicOr(&S.bad, 1u);
      __syncthreads();
      if (S.bad) return false;
    }
  }
  if (tid == 0) S.mixed = listed != 0;

  double z = 1.0;
  if (greedy) {
    if (tid == 0) {
      S.bits = __float_as_uint(mx) >> 16;
      S.nth = 1;
      S.ties = S.values[S.first];
    }
    __syncthreads();
    if (mx == 0.f && S.mixed) return false;
  } else {
    const int b0 = tid * kPer;
    const double tiny_each = listed ? 0.5 : exp2_neg(fmax(t_of(0.f), 0.0));  // with others than 0 among them not used
    // The weights of this thread's values, from the first that occurs on: a progression of ratio r.  f(j, count, weight, mass).
    double w_first = 0.0, r = 0.0;
    int j_first = kPer;
#pragma unroll
    for (int j = kPer - 1; j >= 0; --j)
      if (c[j] && b0 + j != kTiny) j_first = j;
    if (j_first < kPer) {
      w_first = exp2_neg(t_of(value_of_bin(b0 + j_first)));
      r = exp2_neg((static_cast<double>(value_of_bin(b0 + 1)) - static_cast<double>(value_of_bin(b0 + 2))) * scale);
    }
    auto each_value = [&](auto f) {
      double w = w_first;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int b = b0 + j;
        const uint32_t n = c[j];
        if (j == 0 && b == kTiny) {
          f(b, n, tiny_each, tiny_mass);
        } else if (j >= j_first) {
          f(b, n, w, n * w);
          w *= r;
        }
      }
    };
    double mass = 0.0, min_mass = 0.0;
    uint32_t n = 0;
    each_value([&](int b, uint32_t count, double w, double m) {
      mass += m;
      n += count;
      if (by_min && b != kTiny && w >= min_p) min_mass += m;
    });
    // Sums are rounded, so they are added up in an order in which they never fall: the upper half of every 2d lanes adds
    // the lower half's sum to its own.  Rounding keeps order, so a lane's sum is at least the one before it, and the same
    // where the lane has no elements.  (Else a target between two roundings of one sum is met by a lane without any.)
    double mi = mass;
    uint32_t ni = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int from = (lane & -2 * d) + d - 1;  // the lower half's last
      const double ml = __shfl(mi, from);
      const uint32_t nl = __shfl(ni, from);
      if (lane & d) {
        mi += ml;
        ni += nl;
      }
    }
    if (by_min)
      for (int d = 1; d < 64; d <<= 1) min_mass += __shfl_xor(min_mass, d);
    if (lane == 63) {
      S.sum_b[wave] = mi;
      S.part[wave] = ni;
      S.sum_a[wave] = min_mass;
    }
    double me = __shfl_up(mi, 1);
    uint32_t ne = __shfl_up(ni, 1);
    if (lane == 0) me = ne = 0;
    __syncthreads();
    double before = 0.0, total = 0.0, z_min = tiny_min;
    uint32_t n_before = 0, n_total = 0;
    for (int w = 0; w < NT / 64; ++w) {
      if (w == wave) {
        before = total;
        n_before = n_total;
      }
      total += S.sum_b[w];
      z_min += S.sum_a[w];
      n_total += static_cast<uint32_t>(S.part[w]);
    }
    // The sums up to this thread's values; a thread's end is the next one's begin to the last bit, and the ends never
    // fall: exactly one thread meets a target, and it has elements.
    me += before;
    mi += before;
    ne += n_before;
    ni += n_before;

    z = total;
    const bool by_count = s.k > 0 && static_cast<uint32_t>(s.k) < n_total;
#pragma unroll 1
    for (int step = 0; step < 3; ++step) {
      Cross mode = kExceed;
      double target;
      if (step == 0) {
        if (!by_count) continue;
        mode = kCount;
        target = s.k;
      } else if (step == 1) {
        if (!(s.top_p < 1.f)) continue;
        mode = kReach;
        target = fmax(static_cast<double>(s.top_p) * z, 1e-30);
      } else {
        if (by_min) z = fmin(z, z_min);
        target = static_cast<double>(fminf(fmaxf(s.u, 0.f), 0x1.fffffep-1f)) * z;
      }
      const bool here = mode == kCount   ? ne < target && ni >= target
                        : mode == kReach ? me < target && mi >= target
                                         : me <= target && mi > target;
      if (here) {  // one thread: the value at which the target is met, else (by rounding) the last that occurs
        double run = me, base = me, w1 = 0.0;
        double count = ne, base_n = ne;
        int at = b0;
        uint32_t ties = 0;
        bool met = false;
        each_value([&](int b, uint32_t c, double w, double m) {
          if (met || c == 0 || (mode != kCount && w == 0.0)) return;
          at = b;
          ties = c;
          w1 = w;
          base = run;
          base_n = count;
          run += m;
          count += c;
          met = mode == kCount ? count >= target : mode == kReach ? run >= target : run > target;
        });
        double nth;
        if (mode == kCount) {
          nth = target - base_n;
        } else {
          nth = mode == kReach ? ceil((target - base) / w1) : floor((target - base) / w1) + 1.0;
          const double with = __builtin_fma(nth, w1, base), less = __builtin_fma(nth - 1.0, w1, base);
          if (mode == kReach ? less >= target : less > target)
            nth -= 1.0;
          else if (mode == kReach ? with < target : with <= target)
            nth += 1.0;
          nth = fmin(fmax(nth, 1.0), static_cast<double>(ties));
        }
        if (at == kTiny && S.mixed) S.mixed = 2;
        S.bits = at == kTiny ? 0u : __float_as_uint(value_of_bin(at)) >> 16;
        S.nth = static_cast<uint32_t>(nth);
        S.ties = ties;
        S.z = __builtin_fma(nth, w1, base);
      }
      __syncthreads();
      if (S.mixed == 2) return false;
      if (step < 2) {
        z = S.z;
        __syncthreads();
      }
    }
  }

  // the nth element of these bits (0: of either zero), in the order of the row
  const uint32_t bits = S.bits, nth = S.nth, ties = S.ties;
  const uint32_t both = bits << 16 | bits, care = bits ? 0xffffffffu : 0x7fff7fffu;
  auto store = [&](int64_t token) {
    P.token[item] = token;
    P.logprob[item] = greedy ? 0.f : static_cast<float>(-t_of(__uint_as_float(bits << 16)) * kLn2 - log(z));
  };
  if (ties <= kList) {
    if (tid == 0) S.n = 0;
    __syncthreads();
    each([&](const u32x4_t& v, int i0) {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t d = (v[w] ^ both) & care;
        if ((d & 0xffffu) == 0) S.key[atomicAdd(&S.n, 1u) % kList] = i0 + 2 * w;
        if ((d >> 16) == 0) S.key[atomicAdd(&S.n, 1u) % kList] = i0 + 2 * w + 1;
      }
    });
    __syncthreads();
    for (uint32_t i = tid; i < ties; i += NT) {
      const uint64_t mine = S.key[i];
      uint32_t rank = 0;
      for (uint32_t j = 0; j < ties; ++j) rank += S.key[j] < mine;
      if (rank == nth - 1) store(static_cast<int64_t>(mine));
    }
    return true;
  }
  uint32_t seen = 0;
  for (int g0 = 0; g0 < n_gran; g0 += NT) {
    const int gi = g0 + tid;
    uint32_t n = 0, match = 0;
    if (gi < n_gran) {
      const u32x4_t v = granules[gi];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int i = gi * 8 + e - off;
        const uint32_t d = (v[e >> 1] ^ both) & care;
        match |= (e & 1 ? d >> 16 : d & 0xffffu) == 0 && i >= 0 && i < V ? 1u << e : 0u;
      }
      n = __popc(match);
    }
    uint32_t ni = n;
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t l = __shfl_up(ni, d);
      if (lane >= d) ni += l;
    }
    __syncthreads();
    if (lane == 63) S.part[wave] = ni;
    __syncthreads();
    uint32_t before = seen, after = seen;
    for (int w = 0; w < NT / 64; ++w) {
      if (w == wave) before = after;
      after += static_cast<uint32_t>(S.part[w]);
    }
    const uint32_t left = nth - (before + ni - n);  // the wanted one's place among this thread's
    if (before + ni - n < nth && nth <= before + ni) {
      for (uint32_t i = 1; i < left; ++i) match &= match - 1;
      store(gi * 8 - off + __ffs(match) - 1);
    }
    seen = after;
    if (seen >= nth) break;
  }
  return true;
}

// Row `slot` by cost, the costliest first, where a CU holds one row, rows are more than CUs and settings differ: those
// with a temperature (three or four passes), then those of a small top-k, whose few elements are soon in a list, then those
// that want the largest logit alone.  What starts last should end soon.  A thread a row, at most NT of them.  Rows of
// bf16 or of fewer threads come as they are; ordering those was not measured.
template <int NT, bool kWide>
__device__ __forceinline__ uint32_t row_by_cost(const SampleParams& P, Shared<NT, kWide>& S, uint32_t slot) {
  const uint32_t i = threadIdx.x;
  const int lane = i & 63, wave = i >> 6;
  int cls = 3;  // no row
  if (i < P.items) {
    const float T = P.temperature ? P.temperature[i] : P.temperature_all;
    const int k = P.top_k ? P.top_k[i] : P.top_k_all;
    cls = !(T > 0.f) || k == 1 ? 2 : k > 0 && k <= kList ? 1 : 0;
  }
  uint64_t before = 0;  // of this wave's rows, those of its class that come before, and counts of the classes, 16 bits each
  uint64_t counts = 0;
#pragma unroll
  for (int c = 0; c < 3; ++c) {
    const uint64_t in = __ballot(cls == c);
    counts |= static_cast<uint64_t>(__popcll(in)) << (16 * c);
    if (cls == c) before = __popcll(in & ((uint64_t{1} << lane) - 1));
  }
  if (lane == 0) S.part[wave] = counts;
  __syncthreads();
  uint64_t all = 0, earlier = 0;
  for (int w = 0; w < NT / 64; ++w) {
    if (w == wave) earlier = all;
    all += S.part[w];
  }
  if (cls < 3) {
    uint32_t place = static_cast<uint32_t>(before + (earlier >> (16 * cls) & 0xffffu));
    for (int c = 0; c < cls; ++c) place += static_cast<uint32_t>(all >> (16 * c) & 0xffffu);
    if (place == slot) S.first = i;
  }
  __syncthreads();
  return S.first;
}

// One workgroup a row, which every pass reads again (from the caches: a speech vocabulary's row is 16 KB).
template <bool kWide, int NT>
__global__ __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(4))) void sample_kernel(const SampleParams P) {
  constexpr int G = kWide ? 4 : 8, kBytes = kWide ? 4 : 2, kBins = Shared<NT, kWide>::kBins;
  __shared__ Shared<NT, kWide> S;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint32_t item = blockIdx.x;
  if constexpr (kWide && NT == 1024) {
    if (P.by_cost) item = row_by_cost<NT, kWide>(P, S, item);
  }
  const uint32_t r = item / P.bl;
  const int64_t at = (r * P.seq_stride + static_cast<int64_t>(item - r * P.bl) * P.pos_stride) * kBytes;
  const uintptr_t row = reinterpret_cast<uintptr_t>(P.logits) + at;
  const u32x4_t* granules = reinterpret_cast<const u32x4_t*>(row & ~uintptr_t{15});
  const int off = static_cast<int>(row & 15) / kBytes, V = P.vocab;
  const int n_gran = (off + V + G - 1) / G;

  // a granule, what it holds beside the row as -inf
  auto whole = [&](u32x4_t v, int gi) {
    if (gi == 0 || gi == n_gran - 1) {
#pragma unroll
      for (int e = 0; e < G; ++e) {
        const int i = gi * G + e - off;
        if (i >= 0 && i < V) continue;
        if constexpr (kWide)
          v[e] = 0xff800000u;
        else
          v[e >> 1] = (v[e >> 1] & (e & 1 ? 0x0000ffffu : 0xffff0000u)) | (e & 1 ? 0xff800000u : 0x0000ff80u);
      }
    }
    return v;
  };
  auto element = [&](const u32x4_t& v, int e) {
    if constexpr (kWide) return __uint_as_float(v[e]);
    return e & 1 ? bf16hi(v[e >> 1]) : bf16lo(v[e >> 1]);
  };
  // f(granule, its first element's index) for every granule of this thread, the next one on its way
  auto each = [&](auto f) {
    if (tid >= n_gran) return;
    u32x4_t v = granules[tid];
    for (int gi = tid; gi < n_gran; gi += NT) {
      const u32x4_t next = granules[min(gi + NT, n_gran - 1)];
      f(whole(v, gi), gi * G - off);
      v = next;
    }
  };
  // f(key, bin) for every finite element of this thread, one at a time: for passes that are seldom made
  auto each_key = [&](auto f) {
    for (int i = tid; i < V; i += NT) {
      float x;
      if constexpr (kWide)
        x = reinterpret_cast<const float*>(row)[i];
      else
        x = bf16_to_f32(reinterpret_cast<const uint16_t*>(row)[i]);
      if (x > -INFINITY) f(x, key_of(x, i));
    }
  };

  const float T = P.temperature ? P.temperature[item] : P.temperature_all;
  const int k = P.top_k ? P.top_k[item] : P.top_k_all;
  const float top_p = P.top_p ? P.top_p[item] : P.top_p_all;
  const float min_p = P.min_p ? P.min_p[item] : P.min_p_all;
  const float u = P.u[item];
  if constexpr (!kWide) {
    if (sample_values<NT, NT == 512 ? 2 : 4>(P, S, granules, off, n_gran, Settings{T, k, top_p, min_p, u}, item)) return;
    __syncthreads();
  }
  for (int b = tid; b < kBins; b += NT) {
    S.mass[b] = 0;
    S.count[b] = 0;
  }
  if (tid == 0) S.bad = 0;

  // the largest and the least logit, and whether there is a NaN
  float mx = -INFINITY, mn = INFINITY;
  bool bad = false;
  if (tid < 2) {  // the ends' least
    const int gi = tid ? n_gran - 1 : 0;
    const u32x4_t v = granules[gi];
#pragma unroll
    for (int e = 0; e < G; ++e) {
      const int i = gi * G + e - off;
      if (i >= 0 && i < V) mn = fminf(mn, element(v, e));
    }
  }
  each([&](const u32x4_t& v, int i0) {
    float lo = INFINITY;
#pragma unroll
    for (int e = 0; e < G; e += 2) {
      const float x = element(v, e), y = element(v, e + 1);
      bad |= x != x || y != y;
      mx = max3(mx, x, y);
      lo = min3(lo, x, y);
    }
    if (i0 >= 0 && i0 + G <= V) mn = fminf(mn, lo);
  });
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    mx = fmaxf(mx, __shfl_xor(mx, d));
    mn = fminf(mn, __shfl_xor(mn, d));
  }
  if (lane == 0) {
    S.fmx[wave] = mx;
    S.fmn[wave] = mn;
  }
  __syncthreads();
  if (__any(bad) && lane == 0) atomicOr(&S.bad, 1u);
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    mx = fmaxf(mx, S.fmx[w]);
    mn = fminf(mn, S.fmn[w]);
  }
  if (tid == 0) S.n = 0xffffffffu;
  __syncthreads();
  if (S.bad || fabsf(mx) == INFINITY) {  // no distribution
    if (tid == 0) {
      P.token[item] = -1;
      P.logprob[item] = __builtin_nanf("");
    }
    return;
  }
  if (!(T > 0.f) || k == 1) {  // the first token
    uint32_t first = 0xffffffffu;
    each([&](const u32x4_t& v, int i0) {
#pragma unroll
      for (int e = 0; e < G; ++e)
        if (element(v, e) == mx) first = min(first, static_cast<uint32_t>(i0 + e));
    });
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) first = min(first, __shfl_xor(first, d));
    if (lane == 0) atomicMin(&S.n, first);
    __syncthreads();
    if (tid == 0) {
      P.token[item] = S.n;
      P.logprob[item] = 0.f;
    }
    return;
  }

  const double scale = kLog2e / static_cast<double>(T);
  // bins: the row's range, or 64 octaves of weight where that is less; the last one holds weights of 0 alone.
  // By halves: mx - x may be past fp32's range.
  const float half = 0.5f * mx;
  const float per_half = fminf(fmaxf((kBins - 1.5f) / __builtin_fmaf(-0.5f, mn, half), static_cast<float>((kBins - 1) / 32.0 * scale)), 1e30f);
  const double per_x = 0.5 * static_cast<double>(per_half);
  auto bin_of = [&](float x) {
    return static_cast<int>(fminf(__builtin_fmaf(-0.5f, x, half) * per_half, static_cast<float>(kBins - 1)));
  };
  auto t_of = [&](float x) { return (static_cast<double>(mx) - static_cast<double>(x)) * scale; };
  bool by_count = k > 0 && k < V;
  const bool by_min = min_p > 0.f;
  const double t_min = by_min ? -log2(static_cast<double>(fminf(min_p, 1.f))) : 0.0;
  // An element's weight, times 2^shift, in bins but the last: that at its bin's begin times a Taylor polynomial of what is
  // left, at most 64 octaves / kBins.  Weighing is what a row of fp32 costs: the vector unit is busy for three quarters
  // of a lone row's time.  Only temperatures below 1e-36 have wider bins; bf16 rows seldom come here.
  const double inv_T = 1.0 / static_cast<double>(T), width = inv_T / per_x;
  const bool narrow = kWide && width <= 64.0 * kLn2 / (kBins - 1) * 1.01;
  auto weigh = [&](float x, int b) -> uint64_t {
    const double far = static_cast<double>(x) - static_cast<double>(mx);  // may be past fp32's range
    if (!narrow) return weight_of(far * -scale, P.shift);
    const double a = __builtin_fma(far, inv_T, static_cast<double>(b) * width);
    double p = kBins < 2048 ? __builtin_fma(1.0 / 720, a, 1.0 / 120) : 1.0 / 120;  // off by 2e-13 at most
    p = __builtin_fma(p, a, 1.0 / 24);
    p = __builtin_fma(p, a, 1.0 / 6);
    p = __builtin_fma(p, a, 0.5);
    p = __builtin_fma(p, a, 1.0);
    p = __builtin_fma(p, a, 1.0);
    return __builtin_bit_cast(uint64_t, __builtin_fma(p, S.power[b], 0x1p52)) - (uint64_t{0x433} << 52);
  };

  // bins' sums and counts become inclusive prefix sums
  auto scan = [&](uint64_t* mass, uint32_t* count, bool counts) {
    constexpr int kPer = kBins / NT;
    uint64_t m[kPer], ms = 0;
    uint32_t c[kPer], cs = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      m[j] = ms += mass[tid * kPer + j];
      c[j] = cs += counts ? count[tid * kPer + j] : 0;
    }
    uint64_t mi = ms;
    uint32_t ci = cs;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint64_t ml = shfl_up64(mi, d);
      const uint32_t cl = __shfl_up(ci, d);
      if (lane >= d) {
        mi += ml;
        ci += cl;
      }
    }
    if (lane == 63) {
      S.part[wave] = mi;
      S.part2[wave] = ci;
    }
    __syncthreads();
    mi -= ms;
    ci -= cs;
    for (int w = 0; w < wave; ++w) {
      mi += S.part[w];
      ci += static_cast<uint32_t>(S.part2[w]);
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      mass[tid * kPer + j] = mi + m[j];
      if (counts) count[tid * kPer + j] = ci + c[j];
    }
    __syncthreads();
  };
  // the bin in which the target is met; S.bin, S.base and S.base_count tell, after a barrier
  auto find_bin = [&](const uint64_t* mass, const uint32_t* count, bool counts, Cross mode, uint64_t base, uint32_t base_count,
                      double target) {
    for (int b = tid; b < kBins; b += NT) {
      const uint64_t before = b ? mass[b - 1] : 0, with = mass[b];
      bool here;
      if (mode == kCount) {
        const uint32_t cb = base_count + (b ? count[b - 1] : 0), cw = base_count + count[b];
        here = cw >= target && cb < target;
      } else {
        const double db = static_cast<double>(base + before), dw = static_cast<double>(base + with);
        here = mode == kReach ? dw >= target && db < target : dw > target && db <= target;
      }
      if (here) {
        S.bin = b;
        S.base = base + before;
        S.base_count = base_count + (counts && b ? count[b - 1] : 0);
      }
    }
    __syncthreads();
  };

  // Weights are needed up to bin `cut`: that of the last element of top-k or, with neither top-k nor top-p, of min-p.
  int cut = kBins - 1;
  if (by_count) {
    uint32_t last = 0;  // elements of the last bin
    each([&](const u32x4_t& v, int) {
#pragma unroll
      for (int e = 0; e < G; ++e) {
        const float x = element(v, e);
        if (!(x > -INFINITY)) continue;
        const int b = bin_of(x);
        if (b < kBins - 1)
          atomicAdd(&S.count[b], 1u);
        else
          ++last;
      }
    });
    if (last) atomicAdd(&S.count[kBins - 1], last);
    __syncthreads();
    scan(S.mass, S.count, true);
    by_count = static_cast<uint32_t>(k) < S.count[kBins - 1];
    if (by_count) {
      find_bin(S.mass, S.count, true, kCount, 0, 0, k);
      cut = S.bin;
    }
  } else if (by_min && !(top_p < 1.f)) {
    cut = static_cast<int>(fmin(t_min / scale * per_x + 1.0, kBins - 1.0));  // one more for rounding
  }
  // Where the bins up to `cut` hold few elements (a small top-k, or min-p alone), all of them go to the list, and the three
  // sums are found there: no weights in bins, no further pass.
  if (by_count ? S.count[cut] <= kList : cut < kBins - 1) {
    if (tid == 0) S.n = 0;
    __syncthreads();
    each([&](const u32x4_t& v, int i0) {
#pragma unroll
      for (int e = 0; e < G; ++e) {
        const float x = element(v, e);
        if (!(x > -INFINITY) || bin_of(x) > cut) continue;
        const uint32_t to = atomicAdd(&S.n, 1u);
        if (to < kList) S.key[to] = key_of(x, i0 + e);
      }
    });
    __syncthreads();
    const int n = static_cast<int>(S.n);
    if (n <= kList) {
      for (int i = tid; i < n; i += NT) {  // in order
        const uint64_t key = S.key[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += S.key[j] > key;
        S.w[rank] = key;
      }
      __syncthreads();
      if (wave == 0) {  // inclusive sums of the weights, four a lane, into S.key
        uint64_t sum[kList / 64], all = 0;
#pragma unroll
        for (int j = 0; j < kList / 64; ++j) {
          const int i = lane * (kList / 64) + j;
          sum[j] = all += i < n ? weight_of(t_of(value_of(S.w[i])), P.shift) : 0;
        }
        uint64_t to = all;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const uint64_t left = shfl_up64(to, d);
          if (lane >= d) to += left;
        }
#pragma unroll
        for (int j = 0; j < kList / 64; ++j) S.key[lane * (kList / 64) + j] = to - all + sum[j];
      }
      __syncthreads();
      if (tid == 0) {
        // the first of [0, end) at which f holds; it holds from there on, and at end - 1
        auto first = [&](int end, auto f) {
          int lo = 0, hi = end - 1;
          while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (f(mid))
              hi = mid;
            else
              lo = mid + 1;
          }
          return lo;
        };
        int kept = by_count ? min(n, k) : n;
        uint64_t z = S.key[kept - 1];
        if (top_p < 1.f) {
          const double target = fmax(static_cast<double>(top_p) * static_cast<double>(z), 0.5);
          kept = first(kept, [&](int i) { return static_cast<double>(S.key[i]) >= target; }) + 1;
        }
        if (by_min) {
          const int out = first(n + 1, [&](int i) { return i >= n || t_of(value_of(S.w[i])) > t_min; });
          kept = min(kept, max(out, 1));
        }
        z = S.key[kept - 1];
        const double target = static_cast<double>(fminf(fmaxf(u, 0.f), 0x1.fffffep-1f)) * static_cast<double>(z);
        const uint64_t key = S.w[first(kept, [&](int i) { return static_cast<double>(S.key[i]) > target; })];
        P.token[item] = 0xffffffffu - static_cast<uint32_t>(key);
        P.logprob[item] = static_cast<float>(-t_of(value_of(key)) * kLn2 - log(__builtin_ldexp(static_cast<double>(z), -P.shift)));
      }
      return;
    }
  }
  // Searches read the row's elements of a bin again, from memory, unless mass2 holds them (until a bin is divided): all of
  // the bins up to `cut` where they fit, put there before they are weighed, else those of top-p's bin and of the ones
  // that the last search can end in, fetched in one pass for both.  (fp32 rows only: bf16 ones seldom come here.)
  bool held = kWide && by_count && S.count[cut] <= kBins;
  int held_to = held ? cut : -1, held_p = -1, held_lo = 0, held_hi = -1;  // bins up to held_to, held_p, held_lo to held_hi
  auto hold = [&](float x, int index) {
    const uint32_t to = atomicAdd(&S.n_held, 1u);
    if (to < kBins) S.mass2[to] = key_of(x, index);
  };
  if (tid == 0) S.n_held = 0;
  if constexpr (kWide)
    for (int b = tid; b <= cut; b += NT) S.power[b] = __builtin_ldexp(exp2_neg(b * width * kLog2e), P.shift);
  __syncthreads();  // the search for cut is over, too: S.bin may be used again

  uint64_t z_min = 0;  // the weight of what min-p keeps
  const int weighty = min(cut, kBins - 2);
  auto add = [&](float x, int b) {
    const uint64_t w = weigh(x, b);
    atomicAdd(reinterpret_cast<unsigned long long*>(&S.mass[b]), static_cast<unsigned long long>(w));
    if (by_min && t_of(x) <= t_min) z_min += w;
  };
  if (held) {
    each([&](const u32x4_t& v, int i0) {
#pragma unroll
      for (int e = 0; e < G; ++e) {
        const float x = element(v, e);
        if (bin_of(x) <= cut && x > -INFINITY) hold(x, i0 + e);
      }
    });
    __syncthreads();
    for (int i = tid; i < static_cast<int>(S.n_held); i += NT) {
      const float x = value_of(S.mass2[i]);
      const int b = bin_of(x);
      if (b <= weighty) add(x, b);
    }
  } else {
    each([&](const u32x4_t& v, int) {
#pragma unroll
      for (int e = 0; e < G; ++e) {
        const float x = element(v, e);
        const int b = bin_of(x);  // -inf is in the last
        if (b <= weighty) add(x, b);
      }
    });
  }
  if (by_min) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) z_min += shfl_xor64(z_min, d);
    if (lane == 0) S.z_min[wave] = z_min;
  }
  __syncthreads();
  if (by_min) {
    z_min = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) z_min += S.z_min[w];
  }
  scan(S.mass, S.count, false);

  // The element at which the target is met: its key in S.found, the inclusive sum in S.sum, after a barrier.
  auto cross = [&](Cross mode, double target) {
    find_bin(S.mass, S.count, by_count, mode, 0, 0, target);
    const int bin = S.bin;
    uint64_t base = S.base, klo = 0, khi = ~uint64_t{0};
    uint32_t base_count = S.base_count;
    constexpr int kLog = NT == 1024 ? 12 : NT == 512 ? 11 : 10;  // of kBins
    static_assert(1 << kLog == kBins, "an interval of keys fills the bins");
    for (;;) {  // at most 7 times: each further one leaves an interval of keys a thousandth as long, or less
      if (tid == 0) S.n = 0;
      __syncthreads();
      auto list = [&](uint64_t key) {
        const uint32_t to = atomicAdd(&S.n, 1u);
        if (to < kList) S.key[to] = key;
      };
      if (kWide && held && (bin <= held_to || bin == held_p || (bin >= held_lo && bin <= held_hi))) {
        for (int i = tid; i < static_cast<int>(S.n_held); i += NT) {
          const uint64_t key = S.mass2[i];
          if (bin_of(value_of(key)) == bin) list(key);
        }
      } else {
        each([&](const u32x4_t& v, int i0) {
#pragma unroll
          for (int e = 0; e < G; ++e) {
            const float x = element(v, e);
            if (!(x > -INFINITY) || bin_of(x) != bin) continue;
            const uint64_t key = key_of(x, i0 + e);
            if (key >= klo && key <= khi) list(key);
          }
        });
      }
      __syncthreads();
      const int n = static_cast<int>(S.n);
      if (n <= kList) {
        for (int i = tid; i < n; i += NT) S.w[i] = bin == kBins - 1 ? 0 : weigh(value_of(S.key[i]), bin);
        __syncthreads();
        for (int i = tid; i < n; i += NT) {
          const uint64_t key = S.key[i], w = S.w[i];
          uint64_t sum = base;
          uint32_t count = base_count;
          for (int j = 0; j < n; ++j) {
            const bool in = S.key[j] >= key;
            sum += in ? S.w[j] : 0;
            count += in;
          }
          const double with = static_cast<double>(sum), before = static_cast<double>(sum - w);
          const bool here = mode == kCount ? count == target
                            : mode == kReach ? with >= target && before < target
                                             : with > target && before <= target;
          if (here) {
            S.found = key;
            S.sum = sum;
          }
        }
        __syncthreads();
        return;
      }
      held = false;  // mass2 has another use now
      // the interval of the keys, then bins of it
      uint64_t lo = ~uint64_t{0}, hi = 0;
      each_key([&](float x, uint64_t key) {
        if (bin_of(x) != bin || key < klo || key > khi) return;
        lo = min(lo, key);
        hi = max(hi, key);
      });
      for (int d = 1; d < 64; d <<= 1) {
        lo = min(lo, shfl_xor64(lo, d));
        hi = max(hi, shfl_xor64(hi, d));
      }
      if (lane == 0) {
        S.part[wave] = lo;
        S.part2[wave] = hi;
      }
      for (int b = tid; b < kBins; b += NT) {
        S.mass2[b] = 0;
        S.count2[b] = 0;
      }
      __syncthreads();
      for (int w = 0; w < NT / 64; ++w) {
        lo = min(lo, S.part[w]);
        hi = max(hi, S.part2[w]);
      }
      klo = lo;
      khi = hi;
      const int bits = max(64 - __clzll(static_cast<long long>(khi - klo)) - kLog, 0);  // khi > klo: keys differ
      each_key([&](float x, uint64_t key) {
        if (bin_of(x) != bin || key < klo || key > khi) return;
        const int b = static_cast<int>((khi - key) >> bits);
        atomicAdd(reinterpret_cast<unsigned long long*>(&S.mass2[b]),
                  static_cast<unsigned long long>(bin == kBins - 1 ? 0 : weigh(x, bin)));
        atomicAdd(&S.count2[b], 1u);
      });
      __syncthreads();
      scan(S.mass2, S.count2, true);
      find_bin(S.mass2, S.count2, true, mode, base, base_count, target);
      base = S.base;
      base_count = S.base_count;
      const uint64_t top = khi - (static_cast<uint64_t>(S.bin) << bits);
      const uint64_t width = (uint64_t{1} << bits) - 1;
      klo = top - klo > width ? top - width : klo;
      khi = top;
      __syncthreads();  // S.bin has been read
    }
  };

  uint64_t z = S.mass[kBins - 1];
  // u is held to [0, 1 - 2^-24] (a NaN to 0)
  const double share = static_cast<double>(fminf(fmaxf(u, 0.f), 0x1.fffffep-1f));
  if (kWide && !by_count && top_p < 1.f) {
    find_bin(S.mass, S.count, false, kReach, 0, 0, fmax(static_cast<double>(top_p) * static_cast<double>(z), 0.5));
    held_p = S.bin;
    // what top-p keeps weighs at least S.base and at most S.mass[held_p]: the last search's target is between these shares
    const uint64_t least = by_min ? min(S.base, z_min) : S.base, most = by_min ? min(S.mass[held_p], z_min) : S.mass[held_p];
    __syncthreads();
    find_bin(S.mass, S.count, false, kExceed, 0, 0, share * static_cast<double>(least));
    held_lo = S.bin;
    __syncthreads();
    find_bin(S.mass, S.count, false, kExceed, 0, 0, share * static_cast<double>(most));
    held_hi = S.bin;
    each([&](const u32x4_t& v, int i0) {
#pragma unroll
      for (int e = 0; e < G; ++e) {
        const float x = element(v, e);
        const int b = bin_of(x);
        if (x > -INFINITY && (b == held_p || (b >= held_lo && b <= held_hi))) hold(x, i0 + e);
      }
    });
    held = true;
    __syncthreads();
  }
  if (S.n_held > kBins) held = false;
  for (int step = 0; step < 3; ++step) {
    Cross mode = kExceed;
    double target;
    if (step == 0) {
      if (!by_count) continue;
      mode = kCount;
      target = k;
    } else if (step == 1) {
      if (!(top_p < 1.f)) continue;
      mode = kReach;
      target = fmax(static_cast<double>(top_p) * static_cast<double>(z), 0.5);
    } else {
      if (by_min) z = min(z, z_min);
      target = share * static_cast<double>(z);
    }
    cross(mode, target);
    if (step < 2) {
      z = S.sum;
      __syncthreads();
    }
  }
  if (tid == 0) {
    const uint64_t key = S.found;
    P.token[item] = 0xffffffffu - static_cast<uint32_t>(key);
    P.logprob[item] = static_cast<float>(-t_of(value_of(key)) * kLn2 - log(__builtin_ldexp(static_cast<double>(z), -P.shift)));
  }
}

template <bool kWide, int NT>
void launch(const SampleParams& P, hipStream_t st) {
  hipLaunchKernelGGL((sample_kernel<kWide, NT>), dim3(P.items), dim3(NT), 0, st, P);
}

// Threads a row.  What a row does in turn (bins, sums, searches) is most of a short row's time, and more threads shorten it
// where a CU has a row or two; where it has more, small workgroups fill it better.  us with 256, 512 and 1024, top-k,
// top-p and min-p together, bf16 of 8194: one row 14.7, 11.3, 11.6; 256 rows 17.2, 13.5, 13.8; 512 18.4, 15.9, 25.8; 768
// 20.9, 25.9, 37.3; 4096 77, 103.  Longer rows, with 512 and 1024: 256 rows of 100003 bf16 37.0, 35.7; 300 46.5, 63.6; 1024 of
// 32000 46.8, 69.2.  fp32, temperature alone: 256 rows of 100003 98, 67; 300 107, 110 (settings of
// their own 110, 103, and 75 by cost); 600 183, 169; 300 of 50003 54, 61; 64 of 32000 28, 23; 1024 of 32000
// 81, 97.
template <bool kWide>
void launch_rows(SampleParams& P, hipStream_t st) {
  constexpr uint32_t kCUs = 256;
  if (P.vocab <= 10000) {
    if (P.items > 2 * kCUs)
      launch<kWide, 256>(P, st);
    else
      launch<kWide, 512>(P, st);
  } else if (P.items > kCUs && (!kWide || P.vocab <= 60000)) {
    launch<kWide, 512>(P, st);
  } else {
    P.by_cost = kWide && P.items > kCUs && P.items <= 1024 && (P.temperature != nullptr || P.top_k != nullptr);
    launch<kWide, 1024>(P, st);
  }
}

bool overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + b_bytes && y < x + a_bytes;
}

// Whether [b, b + b_bytes) shares a byte with a row of the logits.  Rows are gone through only where it lies among them.
bool overlaps_logits(const SampleParams& P, int64_t elem, const void* b, int64_t b_bytes) {
  const char* base = static_cast<const char*>(P.logits);
  const int64_t rows = P.items / P.bl, seq = P.seq_stride * elem, pos = P.pos_stride * elem, row_bytes = P.vocab * elem;
  const int64_t seq_end = (rows - 1) * seq, pos_end = (P.bl - 1) * pos;
  const int64_t lo = (seq_end < 0 ? seq_end : 0) + (pos_end < 0 ? pos_end : 0);
  const int64_t hi = (seq_end > 0 ? seq_end : 0) + (pos_end > 0 ? pos_end : 0) + row_bytes;
  if (!overlap(base + lo, hi - lo, b, b_bytes)) return false;
  for (int64_t r = 0; r < rows; ++r)
    for (int64_t i = 0; i < P.bl; ++i)
      if (overlap(base + r * seq + i * pos, row_bytes, b, b_bytes)) return true;
  return false;
}

}  // namespace
}  // namespace yapd

extern "C" int yapd_sample_tokens(const void* logits, int wide, int64_t seq_stride, int64_t pos_stride, int rows, int bl,
                                  int vocab, const float* uniform, const float* temperature, float temperature_all,
                                  const int32_t* top_k, int top_k_all, const float* top_p, float top_p_all,
                                  const float* min_p, float min_p_all, int64_t* token, float* logprob, void* stream) {
  YAPD_REQUIRE(rows >= 0 && bl >= 0, "sample_tokens: need rows and bl >= 0 (got %d, %d)", rows, bl);
  const int64_t items = static_cast<int64_t>(rows) * bl;
  YAPD_REQUIRE(items < (int64_t{1} << 22), "sample_tokens: rows * bl must be below 2^22");
  YAPD_REQUIRE(vocab >= 1 && vocab <= (1 << 24), "sample_tokens: need 1 <= vocab <= 2^24 (got %d)", vocab);
  YAPD_REQUIRE(temperature || temperature_all >= 0.f, "sample_tokens: temperature must be >= 0");
  YAPD_REQUIRE(top_p || top_p_all == top_p_all, "sample_tokens: top_p is NaN");
  YAPD_REQUIRE(min_p || min_p_all == min_p_all, "sample_tokens: min_p is NaN");
  if (items == 0) return YAPD_OK;
  YAPD_REQUIRE(logits && uniform && token && logprob, "sample_tokens: NULL pointer");
  YAPD_REQUIRE((reinterpret_cast<uintptr_t>(logits) & (wide ? 3u : 1u)) == 0, "sample_tokens: misaligned logits");
  int bits = 0;  // vocab <= 2^bits, so that all weights together stay below 2^63
  while ((int64_t{1} << bits) < vocab) ++bits;
  yapd::SampleParams P{logits, seq_stride, pos_stride, static_cast<uint32_t>(items), static_cast<uint32_t>(bl), vocab,
                             62 - bits < 51 ? 62 - bits : 51, uniform, temperature, temperature_all, top_k, top_k_all, top_p,
                             top_p_all, min_p, min_p_all, false, token, logprob};
  // a row's output is written while other rows are still read, and rows by cost read every row's settings
  const void* const outs[2] = {token, logprob};
  for (int o = 0; o < 2; ++o) {
    const int64_t bytes = items * (o == 0 ? 8 : 4);
    for (const void* in : {static_cast<const void*>(uniform), static_cast<const void*>(temperature),
                           static_cast<const void*>(top_k), static_cast<const void*>(top_p), static_cast<const void*>(min_p)})
      YAPD_REQUIRE(!in || !yapd::overlap(in, items * 4, outs[o], bytes),
                   "sample_tokens: token and logprob must not overlap uniform or the settings");
    YAPD_REQUIRE(!yapd::overlaps_logits(P, wide ? 4 : 2, outs[o], bytes),
                 "sample_tokens: token and logprob must not overlap the logits");
  }
  YAPD_REQUIRE(!yapd::overlap(token, items * 8, logprob, items * 4), "sample_tokens: token and logprob overlap");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (wide)
    yapd::launch_rows<true>(P, st);
  else
    yapd::launch_rows<false>(P, st);
  YAPD_LAUNCH_CHECK("sample_kernel launch");
  return YAPD_OK;
}
