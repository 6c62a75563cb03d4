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

// Floats in an order that unsigned comparison keeps; the two zeros are one value.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ (static_cast<uint32_t>(static_cast<int>(u) >> 31) | 0x80000000u);
}

__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// ---- the choice of an action -----------------------------------------------------------
// Weights are whole numbers, 2^40 for the largest logit: their sums are exact in any order, so the
// column that a uniform number falls on does not depend on how the row was split. The exponential
// is computed in f64: an error of 2^-24 in it would move the borders between columns by as much,
// and a row in a million would fall on another column than by the definition.
constexpr double kWeightOne = 1099511627776.0;  // 2^40; a row's 2^18 columns sum to at most 2^58

struct Weights {
  double m, inv_t;
  bool infinite;  // the largest logit is +inf: the columns that hold it share the row
  float m32, inv_t32;
  __device__ __forceinline__ Weights(float max, float t)
      : m(max), inv_t(1.0 / static_cast<double>(t)), infinite(max == INFINITY), m32(max), inv_t32(1.f / t) {}
  // False only for logits that weigh 0: below -41 ln 2 = -28.42 the weight rounds to 0, and three
  // roundings in f32 move -28.5 by less than 1e-5.
  __device__ __forceinline__ bool maybe(float x) const { return !((x - m32) * inv_t32 < -28.5f) && x > -INFINITY; }
  __device__ __forceinline__ uint64_t operator()(float x) const {
    if (!maybe(x)) return 0;
    if (infinite) return x == INFINITY ? static_cast<uint64_t>(kWeightOne) : 0;
    return static_cast<uint64_t>(__double2ll_rn(exp((static_cast<double>(x) - m) * inv_t) * kWeightOne));
  }
};

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
