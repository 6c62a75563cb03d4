// What the policy operators' kernels share: the types of logits, the penalties, the order of logits
// and the weights that a choice is drawn by.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "policy.cuh"

namespace mrn {

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_float(float v, float* o) { *o = v; }
__device__ __forceinline__ void from_float(float v, __half* o) { *o = __float2half_rn(v); }
__device__ __forceinline__ void from_float(float v, __nv_bfloat16* o) { *o = __float2bfloat16_rn(v); }

// A row's penalties.
struct Penalties {
  float repetition, presence, frequency;
  int seen;  // history entries to read
};

__device__ __forceinline__ Penalties row_penalties(const RuleParams& r, int row) {
  Penalties p{1.f, 0.f, 0.f, 0};
  if (!r.history) return p;
  if (r.repetition) p.repetition = r.repetition[row];
  if (r.presence) p.presence = r.presence[row];
  if (r.frequency) p.frequency = r.frequency[row];
  p.seen = r.history_len;
  if (r.history_lens) p.seen = min(max(r.history_lens[row], 0), r.history_len);
  return p;
}

// The logit of an action that the history holds `count` times. Every step is rounded to f32 by
// itself (no contraction), which is the operator's definition: the same bits on every path, so that
// two equal logits tie and the choice between them is the lower column's.
__device__ __forceinline__ float penalised(float x, int count, const Penalties& p) {
  if (count == 0) return x;
  x = x > 0.f ? __fdiv_rn(x, p.repetition) : __fmul_rn(x, p.repetition);
  return __fsub_rn(__fsub_rn(x, __fmul_rn(p.frequency, static_cast<float>(count))), p.presence);
}

// Counts of actions in shared memory: a hash table of N places, a power of two, with linear probing, at
// most half full, so that a probe always ends. Keys are -1 where a place is free.
template <int N>
struct ActionCounts {
  int keys[N];
  int counts[N];

  static __device__ __forceinline__ unsigned slot(int action) {
    return (static_cast<unsigned>(action) * 2654435761u) >> 16 & (N - 1);  // Knuth's multiplicative hash
  }
  __device__ __forceinline__ int insert(int action) {
    unsigned h = slot(action);
    for (;;) {
      const int was = atomicCAS(&keys[h], -1, action);
      if (was == -1 || was == action) return h;
      h = (h + 1) & (N - 1);
    }
  }
  __device__ __forceinline__ int find(int action) const {
    unsigned h = slot(action);
    for (;;) {
      const int k = keys[h];
      if (k == action) return h;
      if (k == -1) return -1;
      h = (h + 1) & (N - 1);
    }
  }
};

// Floats in an order that unsigned comparison keeps; the two zeros are one value.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ (static_cast<uint32_t>(static_cast<int>(u) >> 31) | 0x80000000u);
}

// The larger of two, NaN if one is.
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float warp_max_or_nan(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = max_or_nan(v, __shfl_xor_sync(~0u, v, o));
  return v;
}

__device__ __forceinline__ float power_of_two(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// exp((x - m) / t) for a finite m and t > 0, as a power of two of (x - m) times log2(e) / t. Neither factor
// may leave f32 where the product is of interest: above temperatures of 2^100 the logits are taken in units
// of 2^64, below 2^-100 in units of 2^-100; the first moves the exponent by less than 2^-100, the second is
// exact. In between a difference that overflows has a power of 0, and so has, below 2^-100, every logit
// but the largest where that is 2^20 or more: the next one is 2^-4 or more away.
struct Exponential {
  float unit, m, scale;
  __device__ __forceinline__ Exponential(float max, float t) {
    unit = t > 0x1p100f ? 0x1p-64f : t < 0x1p-100f && fabsf(max) < 0x1p20f ? 0x1p100f : 1.f;
    m = max * unit;
    // 0 at a temperature of +inf, but 0 times -inf is not 0
    scale = fmaxf(fminf(1.44269504088896341f / (t * unit), 3.4e38f), 1.5e-45f);
  }
  __device__ __forceinline__ float operator()(float x) const { return power_of_two(fmaf(x, unit, -m) * scale); }
};

__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// ---- the choice of an action -----------------------------------------------------------
// Weights are whole numbers, 2^40 for the largest logit: their sums are exact in any order, so the
// column that a uniform number falls on does not depend on how the row was split. The exponential
// is computed in f64: an error of 2^-24 in it would move the borders between columns by as much,
// and a row in a million would fall on another column than by the definition.
constexpr double kWeightOne = 1099511627776.0;  // 2^40; a row's 2^18 columns sum to at most 2^58

// 2^(i / 32).
static __device__ const double kPowers[32] = {
    0x1.0000000000000p+0, 0x1.059b0d3158574p+0, 0x1.0b5586cf9890fp+0, 0x1.11301d0125b51p+0,
    0x1.172b83c7d517bp+0, 0x1.1d4873168b9aap+0, 0x1.2387a6e756238p+0, 0x1.29e9df51fdee1p+0,
    0x1.306fe0a31b715p+0, 0x1.371a7373aa9cbp+0, 0x1.3dea64c123422p+0, 0x1.44e086061892dp+0,
    0x1.4bfdad5362a27p+0, 0x1.5342b569d4f82p+0, 0x1.5ab07dd485429p+0, 0x1.6247eb03a5585p+0,
    0x1.6a09e667f3bcdp+0, 0x1.71f75e8ec5f74p+0, 0x1.7a11473eb0187p+0, 0x1.82589994cce13p+0,
    0x1.8ace5422aa0dbp+0, 0x1.93737b0cdc5e5p+0, 0x1.9c49182a3f090p+0, 0x1.a5503b23e255dp+0,
    0x1.ae89f995ad3adp+0, 0x1.b7f76f2fb5e47p+0, 0x1.c199bdd85529cp+0, 0x1.cb720dcef9069p+0,
    0x1.d5818dcfba487p+0, 0x1.dfc97337b9b5fp+0, 0x1.ea4afa2a490dap+0, 0x1.f50765b6e4540p+0,
};

// 1 / v to a few units of the last place: the f32 reciprocal and two steps of Newton's iteration, which
// take a fraction of a division's time. v lies between 1e-30 and 1e30.
__device__ __forceinline__ double reciprocal(double v) {
  double r = 1.f / static_cast<float>(v);
  r = r * (2.0 - v * r);
  return r * (2.0 - v * r);
}

// The weight of a logit: with 32 z log2(e) = n + f for z = (x - m) / t, n whole and |f| <= 1/2, exp(z) is
// 2^(n / 32) exp(f ln 2 / 32), the first factor 2^(n >> 5) times one of 32 values, the second the first
// six terms of its series, the next one below 3e-15. About 15 operations in f64 where exp() takes
// several times as many.
struct Weights {
  double m, steps;  // the largest logit; 32 log2(e) / t
  bool infinite;    // the largest logit is +inf: the columns that hold it share the row
  float lowest;     // the smallest logit that may weigh anything
  __device__ __forceinline__ Weights(float max, float t) : m(max), infinite(max == INFINITY) {
    steps = 46.166241308446828 * (t > 1e-30f && t < 1e30f ? reciprocal(t) : 1.0 / static_cast<double>(t));
    // Below -41 ln 2 = -28.42 temperatures from the largest a weight rounds to 0. In f64 neither the product
    // nor the difference leaves the range, at any temperature, and f32 logits are the whole test: those from
    // the border rounded up on are those from the border on. -inf is never one of them.
    lowest = infinite ? INFINITY : fmaxf(__double2float_ru(m - 28.5 * static_cast<double>(t)), -3.402823466e38f);
  }
  // False only for logits that weigh 0.
  __device__ __forceinline__ bool maybe(float x) const { return x >= lowest; }
  __device__ __forceinline__ uint64_t operator()(float x) const {
    if (!maybe(x)) return 0;
    if (infinite) return x == INFINITY ? static_cast<uint64_t>(kWeightOne) : 0;
    constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number
    const double y = (static_cast<double>(x) - m) * steps;
    const double rounded = y + kRound;
    const int n = __double2loint(rounded);
    const double u = (y - (rounded - kRound)) * 0.021660849392498290;  // ln 2 / 32
    const double series = 1.0 + u * (1.0 + u * (0.5 + u * (1.0 / 6 + u * (1.0 / 24 + u * (1.0 / 120)))));
    const double power = __ldg(kPowers + (n & 31));  // times 2^(40 + (n >> 5)), through its exponent
    const double scaled = __hiloint2double(__double2hiint(power) + ((40 + (n >> 5)) << 20), __double2loint(power));
    constexpr double kWhole = 4503599627370496.0;  // 2^52: the sum's low bits are the rounded product
    return static_cast<uint64_t>(__double_as_longlong(scaled * series + kWhole)) & ((1ull << 52) - 1);
  }
};

// w / total, rounded once to f32 (up to a part in 2^40 of a step).
__device__ __forceinline__ float share_of(uint64_t w, uint64_t total) {
  return static_cast<float>(static_cast<double>(w) * reciprocal(static_cast<double>(total)));
}

// The whole number of weight units that a share of the mass needs.
__device__ __forceinline__ uint64_t needed_mass(float top_p, uint64_t mass) {
  const double want = ceil(static_cast<double>(top_p) * static_cast<double>(mass));
  return want < 1.0 ? 1 : min(static_cast<uint64_t>(want), mass);
}

__device__ __forceinline__ uint64_t drawn_unit(float uniform, uint64_t mass) {
  const double at = static_cast<double>(uniform) * static_cast<double>(mass);
  return at > 0.0 ? min(static_cast<uint64_t>(at), mass - 1) : 0;
}

__device__ __forceinline__ uint64_t warp_sum_u64(uint64_t v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// Exclusive sums over the lanes.
__device__ __forceinline__ uint64_t warp_exclusive_u64(uint64_t v, int lane) {
  uint64_t in = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t u = __shfl_up_sync(~0u, in, o);
    if (lane >= o) in += u;
  }
  return in - v;
}

// Sorts 32 G elements of a warp, largest first, in a bitonic network. Element i is lane i / G's
// e[i % G]: exchanges at a distance below G stay in a thread, the others are shuffles.
template <int G>
__device__ __forceinline__ void warp_sort(uint64_t (&e)[G], int lane) {
#pragma unroll
  for (int size = 2; size <= 32 * G; size <<= 1) {
#pragma unroll
    for (int d = size >> 1; d; d >>= 1) {
      if (d >= G) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const uint64_t o = __shfl_xor_sync(~0u, e[g], d / G);
          const int i = lane * G + g;
          const bool larger = ((i & d) == 0) == ((i & size) == 0 || size == 32 * G);
          e[g] = (e[g] > o) == larger ? e[g] : o;
        }
      } else {
#pragma unroll
        for (int g = 0; g < G; ++g)
          if (!(g & d)) {
            const int i = lane * G + g;
            const bool down = (i & size) == 0 || size == 32 * G;
            const uint64_t x = e[g], y = e[g | d];
            const bool swap = (x < y) == down;
            e[g] = swap ? y : x;
            e[g | d] = swap ? x : y;
          }
      }
    }
  }
}

struct Choice {
  int column;  // -1: nothing is left, or a NaN
  float prob;
};

__device__ __forceinline__ void write_choice(const ChooseParams& p, int row, Choice c) {
  p.column[row] = c.column;
  if (p.action) {
    const RuleParams& r = p.in.rules;
    p.action[row] = c.column < 0 || !r.columns ? c.column : r.columns[row * r.columns_stride + c.column];
  }
  if (p.prob) p.prob[row] = c.prob;
}

template <class F>
cudaError_t with_type(LogitType t, F&& f) {
  switch (t) {
    case LogitType::kF32: return f(float());
    case LogitType::kF16: return f(__half());
    case LogitType::kBf16: return f(__nv_bfloat16());
  }
  return cudaErrorInvalidValue;
}

// The kernels for rows of more than kNarrowWidth columns (policy_wide.cu).
cudaError_t launch_adjust_wide(const AdjustParams& p, cudaStream_t s);
cudaError_t launch_choose_wide(const ChooseParams& p, cudaStream_t s);
cudaError_t prepare_policy_wide();

}  // namespace mrn
