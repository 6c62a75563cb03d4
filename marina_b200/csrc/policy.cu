// The policy operators; see policy.cuh for the arguments.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernels.cuh"
#include "launch.h"
#include "policy.cuh"
#include "ptx.cuh"

namespace mrn {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kChunk = 4096;  // columns of a row held in shared memory at a time

// ---- slot tables ------------------------------------------------------------------------
__device__ __forceinline__ int clamped_length(const SlotTableParams& p, int row) {
  const int n = p.lengths[row];
  return n < 0 ? 0 : n > p.width ? p.width : n;
}

// starts[r] = lengths[0] + ... + lengths[r - 1]: one block walks the lengths 1024 at a time.
__global__ void __launch_bounds__(1024) slot_starts_kernel(SlotTableParams p) {
  __shared__ int warp_sum[32];
  grid_dep_wait();
  grid_dep_launch();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int base = 0;
  for (int r0 = 0; r0 < p.rows; r0 += 1024) {
    const int row = r0 + tid;
    int n = 0;
    if (row < p.rows) {
      n = clamped_length(p, row);
      if (n != p.lengths[row] && p.status) atomicCAS(p.status, 0, kErrBadLength);
    }
    int v = n;
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(~0u, v, o);
      if (lane >= o) v += u;
    }
    if (lane == 31) warp_sum[warp] = v;
    __syncthreads();
    if (warp == 0) {
      int w = warp_sum[lane];
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(~0u, w, o);
        if (lane >= o) w += u;
      }
      warp_sum[lane] = w;
    }
    __syncthreads();
    const int before = base + (warp ? warp_sum[warp - 1] : 0) + v - n;
    if (row < p.rows) p.starts[row] = before;
    base += warp_sum[31];
    __syncthreads();
  }
  if (tid == 0) {
    p.starts[p.rows] = base;
    if (base > p.count && p.status) atomicCAS(p.status, 0, kErrBadLength);
  }
}

// table[r, s] = entries[starts[r] + s], -1 behind the list; map[starts[r] + s] = r * width + s.
__global__ void __launch_bounds__(kThreads) slot_fill_kernel(SlotTableParams p) {
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (row >= p.rows) return;
  const int first = p.starts[row], n = clamped_length(p, row);
  const int64_t at = static_cast<int64_t>(row) * p.width;
  for (int s = lane; s < p.width; s += 32) {
    const bool listed = s < n && first + s < p.count;
    p.table[at + s] = listed ? p.entries[first + s] : -1;
    if (listed && p.map) p.map[first + s] = static_cast<int32_t>(at + s);
  }
}

// ---- adjusted logits ----------------------------------------------------------------------
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

// Adjusted logits of columns [c0, c0 + n) of a row into x[0, n). Thread t computes the columns
// t, t + kThreads, ... of the chunk; ends without a barrier.
template <class T>
__device__ void load_chunk(const LogitParams& p, const Penalties& pen, int row, int c0, int n, float* x) {
  const RuleParams& r = p.rules;
  const T* logits = static_cast<const T*>(p.logits) + row * p.stride + c0;
  const int32_t* history = r.history ? r.history + row * r.history_stride : nullptr;
  const int32_t* ids = r.bias_len ? r.bias_actions + row * r.bias_stride : nullptr;
  const float* values = r.bias_len ? r.bias_values + row * r.bias_stride : nullptr;
  const uint32_t* mask = r.mask ? r.mask + row * r.mask_stride : nullptr;
  if (r.columns) {
    const int32_t* columns = r.columns + row * r.columns_stride + c0;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const int a = columns[i];
      float v = -INFINITY;
      if (a >= r.actions && p.status) atomicCAS(p.status, 0, kErrBadAction);
      if (a >= 0 && a < r.actions && (!mask || (mask[a >> 5] >> (a & 31)) & 1)) {
        int count = 0;
        for (int h = 0; h < pen.seen; ++h) count += history[h] == a;
        v = penalised(as_float(logits[i]), count, pen);
        for (int e = 0; e < r.bias_len; ++e)
          if (ids[e] == a) v = __fadd_rn(v, values[e]);
      }
      x[i] = v;
    }
    return;
  }
  int* counts = reinterpret_cast<int*>(x);  // a cell holds its count until its logit replaces it
  if (history) {
    for (int i = threadIdx.x; i < n; i += kThreads) counts[i] = 0;
    __syncthreads();
    for (int h = threadIdx.x; h < pen.seen; h += kThreads) {
      const unsigned i = static_cast<unsigned>(history[h]) - static_cast<unsigned>(c0);
      if (history[h] >= 0 && i < static_cast<unsigned>(n)) atomicAdd(&counts[i], 1);
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const float v = as_float(logits[i]);
    x[i] = history ? penalised(v, counts[i], pen) : v;
  }
  // Each thread adds the entries of its own columns, in the list's order.
  for (int e = 0; e < r.bias_len; ++e) {
    const unsigned i = static_cast<unsigned>(ids[e]) - static_cast<unsigned>(c0);
    if (ids[e] >= 0 && i < static_cast<unsigned>(n) && i % kThreads == threadIdx.x) x[i] = __fadd_rn(x[i], values[e]);
  }
  if (mask)
    for (int i = threadIdx.x; i < n; i += kThreads)
      if (!((mask[(c0 + i) >> 5] >> ((c0 + i) & 31)) & 1)) x[i] = -INFINITY;
}

template <class V, class F>
__device__ V block_reduce(V v, F f, V* shared) {
  for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(~0u, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  v = shared[0];
  for (int w = 1; w < kWarps; ++w) v = f(v, shared[w]);
  return v;
}

// Floats in an order that unsigned comparison keeps; the two zeros are one value.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ (static_cast<uint32_t>(static_cast<int>(u) >> 31) | 0x80000000u);
}

// The row's largest logit and its lowest column as (order key, ~column); 0 where every column is
// masked. *nan: some column that is left holds NaN.
template <class T>
__device__ uint64_t row_maximum(const LogitParams& p, const Penalties& pen, int row, float* x, uint64_t* shared,
                                bool* nan) {
  uint64_t best = 0;
  int bad = 0;
  for (int c0 = 0; c0 < p.width; c0 += kChunk) {
    const int n = min(kChunk, p.width - c0);
    __syncthreads();
    load_chunk<T>(p, pen, row, c0, n, x);
    for (int i = threadIdx.x; i < n; i += kThreads) {
      if (x[i] != x[i]) bad = 1;
      else if (x[i] > -INFINITY) {
        const uint64_t k = static_cast<uint64_t>(order_key(x[i])) << 32 | ~static_cast<uint32_t>(c0 + i);
        if (k > best) best = k;
      }
    }
  }
  *nan = __syncthreads_or(bad);
  return block_reduce(best, [](uint64_t a, uint64_t b) { return a > b ? a : b; }, shared);
}

__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

template <class T>
__global__ void __launch_bounds__(kThreads) adjust_kernel(AdjustParams p) {
  __shared__ float x[kChunk];
  __shared__ uint64_t shared[kWarps];
  grid_dep_wait();
  grid_dep_launch();
  const int row = blockIdx.x, width = p.in.width;
  const Penalties pen = row_penalties(p.in.rules, row);
  const float t = p.in.temperature ? p.in.temperature[row] : 1.f;
  float m = 0.f, inv = 0.f;
  int first = -1;
  // exp((v - m) / t); a largest logit of +inf is shared by the columns that hold it
  auto relative = [&](float v) { return v == m ? 1.f : m == INFINITY ? v * 0.f : expf((v - m) / t); };
  if (p.priors) {
    bool nan;
    const uint64_t best = row_maximum<T>(p.in, pen, row, x, shared, &nan);
    m = best ? key_value(static_cast<uint32_t>(best >> 32)) : -INFINITY;
    first = best ? static_cast<int>(~static_cast<uint32_t>(best)) : -1;
    const bool bad = nan || t != t;
    float sum = bad ? NAN : 0.f;
    for (int c0 = 0; c0 < width; c0 += kChunk) {
      const int n = min(kChunk, width - c0);
      if (width > kChunk) {
        __syncthreads();
        load_chunk<T>(p.in, pen, row, c0, n, x);
      }
      for (int i = threadIdx.x; i < n; i += kThreads)
        if (x[i] > -INFINITY) sum += relative(x[i]);
    }
    sum = block_reduce(sum, [](float a, float b) { return a + b; }, reinterpret_cast<float*>(shared));
    inv = sum == 0.f ? 0.f : 1.f / sum;
  }
  for (int c0 = 0; c0 < width; c0 += kChunk) {
    const int n = min(kChunk, width - c0);
    if (width > kChunk || !p.priors) {
      __syncthreads();
      load_chunk<T>(p.in, pen, row, c0, n, x);
    }
    for (int i = threadIdx.x; i < n; i += kThreads) {
      if (p.out) from_float(x[i], static_cast<T*>(p.out) + row * p.out_stride + c0 + i);
      if (p.priors) {
        float e = 0.f;
        if (t <= 0.f && inv == inv) e = c0 + i == first ? 1.f : 0.f;
        else if (!(x[i] <= -INFINITY)) e = relative(x[i]) * inv;
        p.priors[row * p.priors_stride + c0 + i] = e;
      }
    }
  }
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
  __device__ __forceinline__ uint64_t operator()(float x) const {
    if (!(x > -INFINITY)) return 0;
    if (infinite) return x == INFINITY ? static_cast<uint64_t>(kWeightOne) : 0;
    return static_cast<uint64_t>(__double2ll_rn(exp((static_cast<double>(x) - m) * inv_t) * kWeightOne));
  }
};

template <class T>
__global__ void __launch_bounds__(kThreads) choose_kernel(ChooseParams p) {
  __shared__ float x[kChunk];
  __shared__ uint64_t shared[kWarps];
  __shared__ unsigned long long bins[256];
  __shared__ uint64_t scan[kThreads + 1];
  __shared__ int digit, chosen;
  __shared__ uint64_t passed;
  grid_dep_wait();
  grid_dep_launch();
  const int row = blockIdx.x, width = p.in.width, tid = threadIdx.x;
  const Penalties pen = row_penalties(p.in.rules, row);
  const float t = p.in.temperature ? p.in.temperature[row] : 1.f;
  auto add = [](uint64_t a, uint64_t b) { return a + b; };
  auto answer = [&](int column, float prob) {
    if (tid != 0) return;
    p.column[row] = column;
    if (p.action) {
      const RuleParams& r = p.in.rules;
      p.action[row] = column < 0 || !r.columns ? column : r.columns[row * r.columns_stride + column];
    }
    if (p.prob) p.prob[row] = prob;
  };

  bool nan;
  const uint64_t best = row_maximum<T>(p.in, pen, row, x, shared, &nan);
  if (nan || t != t) return answer(-1, NAN);
  if (!best) return answer(-1, 0.f);
  const int first = static_cast<int>(~static_cast<uint32_t>(best));
  if (t <= 0.f) return answer(first, 1.f);
  const float m = key_value(static_cast<uint32_t>(best >> 32));
  const Weights weight{static_cast<double>(m), 1.0 / static_cast<double>(t), m == INFINITY};

  // f(i, column, x) for every column, thread by thread; a row of one chunk is loaded already.
  auto each = [&](auto&& f) {
    for (int c0 = 0; c0 < width; c0 += kChunk) {
      const int n = min(kChunk, width - c0);
      if (width > kChunk) {
        __syncthreads();
        load_chunk<T>(p.in, pen, row, c0, n, x);
      }
      for (int i = tid; i < n; i += kThreads)
        if (x[i] > -INFINITY) f(x[i]);
    }
  };
  // The key at which the columns from the largest down reach `need` in the measure `of` (a count or
  // a weight), among those above `floor_key`; *above gets the measure of the larger keys.
  auto select = [&](uint64_t need, uint32_t floor_key, uint64_t* above, auto&& of) {
    uint32_t prefix = 0, known = 0;
    uint64_t over = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      bins[tid] = 0;
      __syncthreads();
      each([&](float v) {
        const uint32_t k = order_key(v);
        if (k > floor_key && (k & known) == prefix) atomicAdd(&bins[(k >> shift) & 255], static_cast<unsigned long long>(of(v)));
      });
      __syncthreads();
      if (tid == 0) {
        uint64_t sum = over;
        int d = 255;
        while (d > 0 && sum + bins[d] < need) sum += bins[d--];
        digit = d;
        passed = sum;
      }
      __syncthreads();
      prefix |= static_cast<uint32_t>(digit) << shift;
      known |= 255u << shift;
      over = passed;
    }
    *above = over;
    return prefix;
  };

  // Kept: the columns above key `cut`, and the first `ties` of those at it.
  uint32_t cut = 0;
  uint64_t ties = 0;
  const int k = p.top_k ? p.top_k[row] : 0;
  if (k > 0) {
    uint64_t live = 0;
    each([&](float) { ++live; });
    live = block_reduce(live, add, shared);
    if (live > static_cast<uint64_t>(k)) {
      uint64_t above;
      cut = select(static_cast<uint64_t>(k), 0, &above, [](float) { return 1; });
      ties = static_cast<uint64_t>(k) - above;
    }
  }
  uint64_t mass = 0;
  each([&](float v) {
    if (order_key(v) > cut) mass += weight(v);
  });
  mass = block_reduce(mass, add, shared);
  uint64_t at_cut = ties ? weight(key_value(cut)) : 0;
  uint64_t total = mass + ties * at_cut;
  const float top_p = p.top_p ? p.top_p[row] : 1.f;
  if (top_p < 1.f) {
    const double want = ceil(static_cast<double>(top_p) * static_cast<double>(total));
    const uint64_t need = want < 1.0 ? 1 : min(static_cast<uint64_t>(want), total);
    if (mass >= need) cut = select(need, cut, &mass, weight);
    at_cut = weight(key_value(cut));
    ties = (need - mass + at_cut - 1) / at_cut;
    total = mass + ties * at_cut;
  }
  if (!p.uniform) return answer(first, static_cast<float>(kWeightOne / static_cast<double>(total)));

  const double at = static_cast<double>(p.uniform[row]) * static_cast<double>(total);
  const uint64_t target = at > 0.0 ? min(static_cast<uint64_t>(at), total - 1) : 0;
  // Column order: each thread takes a run of the chunk's columns.
  constexpr int kRun = kChunk / kThreads;
  uint64_t before = 0, tied = 0;
  for (int c0 = 0; c0 < width; c0 += kChunk) {
    const int n = min(kChunk, width - c0);
    __syncthreads();
    if (width > kChunk) {
      load_chunk<T>(p.in, pen, row, c0, n, x);
      __syncthreads();
    }
    const int lo = min(tid * kRun, n), hi = min(lo + kRun, n);
    auto prefix_sum = [&](uint64_t v) {
      scan[tid + 1] = v;
      __syncthreads();
      if (tid == 0) {
        scan[0] = 0;
        for (int i = 0; i < kThreads; ++i) scan[i + 1] += scan[i];
      }
      __syncthreads();
    };
    uint64_t here = 0;
    for (int i = lo; i < hi; ++i) here += x[i] > -INFINITY && order_key(x[i]) == cut;
    prefix_sum(here);
    const uint64_t my_ties = tied + scan[tid];
    tied += scan[kThreads];
    __syncthreads();
    auto kept = [&](int i, uint64_t& rank) -> uint64_t {
      if (!(x[i] > -INFINITY)) return 0;
      const uint32_t key = order_key(x[i]);
      if (key > cut) return weight(x[i]);
      return key == cut && rank++ < ties ? at_cut : 0;
    };
    uint64_t rank = my_ties;
    here = 0;
    for (int i = lo; i < hi; ++i) here += kept(i, rank);
    prefix_sum(here);
    uint64_t sum = before + scan[tid];
    if (target >= sum && target < before + scan[tid + 1]) {
      rank = my_ties;
      for (int i = lo; i < hi; ++i) {
        const uint64_t w = kept(i, rank);
        if (target < sum + w) {
          chosen = c0 + i;
          passed = w;
          break;
        }
        sum += w;
      }
    }
    before += scan[kThreads];
    __syncthreads();
    if (before > target) {
      answer(chosen, static_cast<float>(static_cast<double>(passed) / static_cast<double>(total)));
      return;
    }
  }
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

}  // namespace

cudaError_t launch_slot_table(const SlotTableParams& p, cudaStream_t s) {
  cudaError_t e = launch_kernel(slot_starts_kernel, dim3(1), dim3(1024), 0, s, p);
  if (e != cudaSuccess || p.rows == 0) return e;
  return launch_kernel(slot_fill_kernel, dim3((p.rows + kWarps - 1) / kWarps), dim3(kThreads), 0, s, p);
}

cudaError_t launch_adjust(const AdjustParams& p, cudaStream_t s) {
  return with_type(p.in.type, [&](auto v) {
    return launch_kernel(adjust_kernel<decltype(v)>, dim3(p.in.rows), dim3(kThreads), 0, s, p);
  });
}

cudaError_t launch_choose(const ChooseParams& p, cudaStream_t s) {
  return with_type(p.in.type, [&](auto v) {
    return launch_kernel(choose_kernel<decltype(v)>, dim3(p.in.rows), dim3(kThreads), 0, s, p);
  });
}

cudaError_t prepare_policy() {
  cudaFuncAttributes a;
  cudaError_t e;
  if ((e = cudaFuncGetAttributes(&a, slot_starts_kernel)) != cudaSuccess) return e;
  if ((e = cudaFuncGetAttributes(&a, slot_fill_kernel)) != cudaSuccess) return e;
  for (LogitType t : {LogitType::kF32, LogitType::kF16, LogitType::kBf16}) {
    e = with_type(t, [&](auto v) {
      const cudaError_t r = cudaFuncGetAttributes(&a, adjust_kernel<decltype(v)>);
      return r != cudaSuccess ? r : cudaFuncGetAttributes(&a, choose_kernel<decltype(v)>);
    });
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace mrn
