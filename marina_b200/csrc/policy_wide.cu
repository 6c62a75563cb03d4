// The policy operators on rows of more than kNarrowWidth columns: a cluster of blocks takes a row,
// each block a contiguous segment of its columns, which it reads once, adjusts, and holds in shared
// memory until the row is done. Blocks of a row exchange maxima, sums and histograms through
// distributed shared memory.
#include <cooperative_groups.h>
#include <stdlib.h>

#include <utility>

#include "kernels.cuh"
#include "launch.h"
#include "policy.cuh"
#include "policy_rows.cuh"
#include "ptx.cuh"

namespace mrn {

namespace {

namespace cg = cooperative_groups;

constexpr int kMaxThreads = 512;
constexpr int kMaxWarps = kMaxThreads / 32;
constexpr int kMaxBlocks = 8;  // of a cluster; what every device schedules
constexpr int kMaxSegment = kPolicyMaxWidth / kMaxBlocks;

// This block's part of its row.
struct Part {
  int row, rank, blocks;
  int c0, n;  // columns [c0, c0 + n); c0 is a multiple of 32, n may be 0
};

__device__ __forceinline__ Part my_part(int blocks, int segment, int width) {
  Part q;
  q.blocks = blocks;
  q.row = blockIdx.x / blocks;
  q.rank = blockIdx.x - q.row * blocks;
  q.c0 = q.rank * segment;
  q.n = max(0, min(segment, width - q.c0));
  return q;
}

// A barrier of the row's blocks.
__device__ __forceinline__ void row_sync(const Part& q) {
  if (q.blocks > 1) cg::this_cluster().sync();
  else __syncthreads();
}

// Block `rank`'s copy of a shared variable.
template <class V>
__device__ __forceinline__ V* at_rank(V* v, const Part& q, int rank) {
  return q.blocks > 1 ? cg::this_cluster().map_shared_rank(v, rank) : v;
}

// f over one value per thread of the row; every thread gets the result. An Exchange serves one
// reduction of a launch: another block may still read `mine` after this returns.
template <class V>
struct Exchange {
  V warps[kMaxWarps];
  V mine;
};

template <class V, class F>
__device__ __forceinline__ V row_reduce(const Part& q, V v, F f, Exchange<V>& ex) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(~0u, v, o));
  if ((threadIdx.x & 31) == 0) ex.warps[threadIdx.x >> 5] = v;
  __syncthreads();
  v = ex.warps[0];
  const int warps = blockDim.x >> 5;
  for (int w = 1; w < warps; ++w) v = f(v, ex.warps[w]);
  if (q.blocks == 1) return v;
  if (threadIdx.x == 0) ex.mine = v;
  cg::this_cluster().sync();
  v = *at_rank(&ex.mine, q, 0);
  for (int r = 1; r < q.blocks; ++r) v = f(v, *at_rank(&ex.mine, q, r));
  return v;
}

// The adjusted logits of the block's columns into x[0, n). Thread t holds the columns t,
// t + blockDim.x, ... of the segment, and sees only its own until the next barrier.
template <class T>
__device__ __forceinline__ void load_part(const LogitParams& p, const Part& q, float* x) {
  const RuleParams& r = p.rules;
  const int n = q.n, c0 = q.c0, tid = threadIdx.x, threads = blockDim.x, row = q.row;
  const T* logits = static_cast<const T*>(p.logits) + row * p.stride + c0;
  const Penalties pen = row_penalties(r, row);
  const int32_t* history = r.history + row * r.history_stride;
  const int32_t* ids = r.bias_actions + row * r.bias_stride;
  const float* values = r.bias_values + row * r.bias_stride;
  const uint32_t* mask = r.mask ? r.mask + row * r.mask_stride : nullptr;
  if (r.columns) {
    // Slots of a wide row: each column counts its action in the history by itself.
    const int32_t* columns = r.columns + row * r.columns_stride + c0;
    for (int i = tid; i < n; i += threads) {
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
  if (pen.seen > 0) {
    for (int i = tid; i < n; i += threads) counts[i] = 0;
    __syncthreads();
    for (int h = tid; h < pen.seen; h += threads) {
      const int id = history[h];
      if (id >= c0 && id - c0 < n) atomicAdd(&counts[id - c0], 1);
    }
    __syncthreads();
  }
  constexpr int kAhead = 8;  // logits in flight per thread
  for (int i0 = tid; i0 < n; i0 += kAhead * threads) {
    float v[kAhead];
    uint32_t word[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u * threads;
      v[u] = i < n ? as_float(logits[i]) : 0.f;
      word[u] = mask && i < n ? mask[(c0 + i) >> 5] : ~0u;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u * threads;
      if (i < n) {
        if (pen.seen > 0) v[u] = penalised(v[u], counts[i], pen);
        x[i] = (word[u] >> ((c0 + i) & 31)) & 1 ? v[u] : -INFINITY;
      }
    }
  }
  if (r.bias_len) {
    // A column's entries are all added by the warp that the column belongs to, which goes through the
    // whole list in its order.
    __syncthreads();
    const int lane = tid & 31, warp = tid >> 5, warps = threads >> 5;
    for (int e0 = 0; e0 < r.bias_len; e0 += 32) {
      const int id = e0 + lane < r.bias_len ? ids[e0 + lane] : -1;
      bool mine = id >= c0 && id - c0 < n && (id - c0) % warps == warp;
      if (mine && mask) mine = (mask[id >> 5] >> (id & 31)) & 1;
      unsigned todo = __ballot_sync(~0u, mine);
      while (todo) {
        const int j = __ffs(todo) - 1;
        todo &= todo - 1;
        if (lane == j) x[id - c0] = __fadd_rn(x[id - c0], values[e0 + j]);
        __syncwarp();
      }
    }
    __syncthreads();
  }
}

// The row's largest logit and its lowest column as (order key, ~column): 0 where nothing is left,
// all ones where a column that is left holds NaN.
__device__ __forceinline__ uint64_t row_best(const Part& q, const float* x, Exchange<uint64_t>& ex) {
  uint64_t best = 0;
  for (int i = threadIdx.x; i < q.n; i += blockDim.x) {
    const float v = x[i];
    uint64_t k = 0;
    if (v != v) k = ~0ull;
    else if (v > -INFINITY) k = static_cast<uint64_t>(order_key(v)) << 32 | ~static_cast<uint32_t>(q.c0 + i);
    if (k > best) best = k;
  }
  return row_reduce(q, best, [](uint64_t a, uint64_t b) { return a > b ? a : b; }, ex);
}

template <class T>
__global__ void __launch_bounds__(kMaxThreads) adjust_wide_kernel(AdjustParams p, int blocks, int segment) {
  extern __shared__ __align__(16) float x[];
  __shared__ Exchange<uint64_t> ex_best;
  __shared__ Exchange<float> ex_sum;
  grid_dep_wait();
  grid_dep_launch();
  const Part q = my_part(blocks, segment, p.in.width);
  const int tid = threadIdx.x, threads = blockDim.x;
  load_part<T>(p.in, q, x);
  T* out = p.out ? static_cast<T*>(p.out) + q.row * p.out_stride + q.c0 : nullptr;
  if (!p.priors) {
    for (int i = tid; i < q.n; i += threads) from_float(x[i], out + i);
    return;
  }
  const uint64_t best = row_best(q, x, ex_best);
  const float t = p.in.temperature ? p.in.temperature[q.row] : 1.f;
  const bool nan = best == ~0ull || t != t;
  const float m = best ? key_value(static_cast<uint32_t>(best >> 32)) : -INFINITY;
  float sum = 0.f;
  for (int i = tid; i < q.n; i += threads) {
    const float v = x[i];
    if (out) from_float(v, out + i);
    float e;
    if (v == -INFINITY) e = 0.f;
    else if (nan) e = NAN;
    else if (t <= 0.f) e = static_cast<uint32_t>(q.c0 + i) == ~static_cast<uint32_t>(best) ? 1.f : 0.f;
    else e = v == m ? 1.f : m == INFINITY ? 0.f : expf((v - m) / t);
    x[i] = e;
    sum += e;
  }
  sum = row_reduce(q, sum, [](float a, float b) { return a + b; }, ex_sum);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  float* priors = p.priors + q.row * p.priors_stride + q.c0;
  for (int i = tid; i < q.n; i += threads) {
    const float e = x[i];
    priors[i] = e == 0.f ? 0.f : e * inv;  // a masked column's 0 stays one beside a NaN
  }
  if (q.blocks > 1) cg::this_cluster().sync();  // no block leaves while another reads from it
}

// ---- the choice ----------------------------------------------------------------------------
// Where a row is cut off (top_k, top_p), the last column that is kept is found by its element, (order
// key of the logit, ~column), so that equal logits are told apart by their columns: a histogram of
// counts and masses over the distance from the largest logit, kBins bins of 1/36 of a temperature
// that cover all weights above 0; then the elements of the bin that the border falls into, gathered in
// one block and sorted. Where a bin holds more than that block's list, the element is found digit by
// digit instead.
constexpr int kBins = 1024;
constexpr float kBinsPerUnit = 36.f;  // exp(-1024 / 36) < 2^-41: what lies below weighs 0

__host__ __device__ constexpr int list_capacity(int segment) { return segment <= 8192 ? 1024 : 4096; }

struct ChooseShared {
  Exchange<uint64_t> best, mass_k;
  uint64_t warp_sums[kMaxWarps];
  uint64_t scan[kMaxWarps + 1];
  uint64_t digits[256], digit_sums[256];
  uint64_t mass;         // kept by this block
  int digit;
  uint64_t passed;
  // written by the row's first block for the others
  int bin_k, bin_p;
  unsigned listed[2];    // elements of bin_k, bin_p
  uint64_t before, need; // mass of the bins above bin_p, mass to reach
  uint64_t total_k;
  uint64_t threshold;
};

// Dynamic shared memory of a block: the segment, then where rows may be cut off the list, this block's
// histogram and the row's (the same memory where a block has the row to itself).
struct ChooseMemory {
  float* x;
  uint64_t *list, *masses, *row_masses;
  uint32_t *counts, *row_counts;
  unsigned room;  // elements that the list holds
  __device__ ChooseMemory(unsigned char* base, int segment, int blocks) {
    room = list_capacity(segment);
    x = reinterpret_cast<float*>(base);
    list = reinterpret_cast<uint64_t*>(x + segment);
    masses = list + room;
    row_masses = blocks > 1 ? masses + kBins : masses;
    counts = reinterpret_cast<uint32_t*>(row_masses + kBins);
    row_counts = blocks > 1 ? counts + kBins : counts;
  }
  static size_t bytes(int segment, int blocks, bool cut) {
    const size_t histogram = kBins * (sizeof(uint64_t) + sizeof(uint32_t));
    return segment * sizeof(float) +
           (cut ? list_capacity(segment) * sizeof(uint64_t) + histogram * (blocks > 1 ? 2 : 1) : 0);
  }
};

__device__ __forceinline__ uint64_t element(float x, int column) {
  return static_cast<uint64_t>(order_key(x)) << 32 | ~static_cast<uint32_t>(column);
}

// Exclusive sums over the block's threads; *total: the sum of all.
__device__ __forceinline__ uint64_t block_exclusive_u64(uint64_t v, ChooseShared& sh, uint64_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  uint64_t in = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t u = __shfl_up_sync(~0u, in, o);
    if (lane >= o) in += u;
  }
  __syncthreads();
  if (lane == 31) sh.warp_sums[warp] = in;
  __syncthreads();
  uint64_t before = 0, all = 0;
  for (int w = 0; w < warps; ++w) {
    if (w < warp) before += sh.warp_sums[w];
    all += sh.warp_sums[w];
  }
  *total = all;
  return before + in - v;
}

// The bin at which the sums of `values` from bin 0 on reach `need` (<= their total), by one block:
// one thread calls found(bin, sum of the bins before).
template <class V, class F>
__device__ __forceinline__ void find_bin(const V* values, uint64_t need, ChooseShared& sh, F found) {
  const int per = kBins / blockDim.x, lo = threadIdx.x * per;
  uint64_t mine = 0, total;
  for (int b = lo; b < lo + per; ++b) mine += values[b];
  uint64_t before = block_exclusive_u64(mine, sh, &total);
  if (before < need && need <= before + mine) {
    int b = lo;
    while (before + values[b] < need) before += values[b++];
    found(b, before);
  }
}

// Sorts list[0, n), largest first, by one block. The list holds a power of two of at least n.
__device__ __forceinline__ void sort_list(uint64_t* list, int n) {
  int size2 = 2;
  while (size2 < n) size2 <<= 1;
  for (int i = n + threadIdx.x; i < size2; i += blockDim.x) list[i] = 0;
  for (int size = 2; size <= size2; size <<= 1)
    for (int d = size >> 1; d; d >>= 1) {
      __syncthreads();
      for (int j = threadIdx.x; j < size2 / 2; j += blockDim.x) {
        const int i = 2 * j - (j & (d - 1));
        const bool down = (i & size) == 0;
        const uint64_t a = list[i], b = list[i + d];
        if ((a < b) == down) list[i] = b, list[i + d] = a;
      }
    }
  __syncthreads();
}

struct Border {
  const Part& q;
  const ChooseMemory& mem;
  ChooseShared& sh;
  const Weights& weight;
  float m, per_bin;

  __device__ __forceinline__ int bin(float x) const {
    const float d = (m - x) * per_bin;  // falls as x rises, step by step under rounding too
    return d < static_cast<float>(kBins) ? static_cast<int>(d) : d != d ? 0 : kBins - 1;  // NaN: inf - inf, 0 * inf
  }

  // f(element, weight) for this block's columns that weigh anything.
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    for (int i = threadIdx.x; i < q.n; i += blockDim.x) {
      const float v = mem.x[i];
      const uint64_t w = weight(v);
      if (w) f(v, i, w);
    }
  }

  // The elements of a bin into the first block's list, in any order.
  __device__ __forceinline__ void gather(int wanted, int which) {
    unsigned* listed = at_rank(&sh.listed[which], q, 0);
    uint64_t* list = at_rank(mem.list, q, 0);
    const int lane = threadIdx.x & 31;
    for (int i0 = threadIdx.x - lane; i0 < q.n; i0 += blockDim.x) {
      const int i = i0 + lane;
      const float v = i < q.n ? mem.x[i] : -INFINITY;
      const bool in = v > -INFINITY && bin(v) == wanted && weight(v);
      const unsigned all = __ballot_sync(~0u, in);
      if (!all) continue;
      unsigned base = 0;
      if (lane == 0) base = atomicAdd(listed, static_cast<unsigned>(__popc(all)));
      base = __shfl_sync(~0u, base, 0) + __popc(all & ((1u << lane) - 1));
      if (in && base < mem.room) list[base] = element(v, q.c0 + i);
    }
  }
  __device__ __forceinline__ bool fits(int which) const {
    return *at_rank(&sh.listed[which], q, 0) <= mem.room;
  }

  // The element at which those from `floor` on, largest first, reach `need` in counts or in mass;
  // every block of the row finds it.
  __device__ uint64_t by_digits(uint64_t need, uint64_t floor, bool masses) {
    uint64_t prefix = 0, known = 0, over = 0;
    for (int shift = 56; shift >= 0; shift -= 8) {
      for (int b = threadIdx.x; b < 256; b += blockDim.x) sh.digits[b] = 0;
      __syncthreads();
      each([&](float v, int i, uint64_t w) {
        const uint64_t e = element(v, q.c0 + i);
        if (e >= floor && (e & known) == prefix)
          atomicAdd(reinterpret_cast<unsigned long long*>(&sh.digits[(e >> shift) & 255]),
                    static_cast<unsigned long long>(masses ? w : 1));
      });
      row_sync(q);
      for (int b = threadIdx.x; b < 256; b += blockDim.x) {
        uint64_t s = 0;
        for (int r = 0; r < q.blocks; ++r) s += at_rank(sh.digits, q, r)[b];
        sh.digit_sums[b] = s;
      }
      __syncthreads();
      if (threadIdx.x == 0) {
        uint64_t sum = over;
        int d = 255;
        while (d > 0 && sum + sh.digit_sums[d] < need) sum += sh.digit_sums[d--];
        sh.digit = d;
        sh.passed = sum;
      }
      row_sync(q);
      prefix |= static_cast<uint64_t>(sh.digit) << shift;
      known |= 255ull << shift;
      over = sh.passed;
      __syncthreads();
    }
    return prefix;
  }

  // The last element that the row keeps.
  __device__ uint64_t find(int k, float top_p) {
    const int tid = threadIdx.x, threads = blockDim.x;
    for (int b = tid; b < kBins; b += threads) mem.masses[b] = 0, mem.counts[b] = 0;
    if (tid == 0) sh.listed[0] = sh.listed[1] = 0;
    __syncthreads();
    each([&](float v, int, uint64_t w) {
      const int b = bin(v);
      atomicAdd(reinterpret_cast<unsigned long long*>(&mem.masses[b]), static_cast<unsigned long long>(w));
      if (k > 0) atomicAdd(&mem.counts[b], 1u);
    });
    row_sync(q);
    if (q.blocks > 1) {
      // each block adds up a share of the bins and hands it to the first
      const int share = kBins / q.blocks;
      uint64_t* row_masses = at_rank(mem.row_masses, q, 0);
      uint32_t* row_counts = at_rank(mem.row_counts, q, 0);
      for (int b = q.rank * share + tid; b < (q.rank + 1) * share; b += threads) {
        uint64_t s = 0;
        uint32_t c = 0;
        for (int r = 0; r < q.blocks; ++r) s += at_rank(mem.masses, q, r)[b], c += at_rank(mem.counts, q, r)[b];
        row_masses[b] = s, row_counts[b] = c;
      }
      row_sync(q);
    }
    const bool lead = q.rank == 0;
    uint64_t floor = 0;
    int bin_k = -1;
    bool listed = false;  // the first block's list holds bin_k, sorted
    if (lead) {
      uint64_t all = 0, mass = 0;
      for (int b = tid; b < kBins; b += threads) all += mem.row_counts[b], mass += mem.row_masses[b];
      uint64_t count, total;
      block_exclusive_u64(all, sh, &count);
      block_exclusive_u64(mass, sh, &total);
      if (tid == 0) sh.bin_k = -1, sh.total_k = total;
      __syncthreads();
      if (k > 0 && static_cast<uint64_t>(k) < count)
        find_bin(mem.row_counts, static_cast<uint64_t>(k), sh, [&](int b, uint64_t before) {
          sh.bin_k = b;
          sh.need = static_cast<uint64_t>(k) - before;
        });
    }
    if (k > 0) {
      row_sync(q);
      bin_k = *at_rank(&sh.bin_k, q, 0);
      if (bin_k >= 0) {
        gather(bin_k, 0);
        row_sync(q);
        listed = fits(0);
        if (listed) {
          if (lead) {
            const int n = static_cast<int>(sh.listed[0]), keep = static_cast<int>(sh.need);
            sort_list(mem.list, n);
            uint64_t mass = 0, total;
            for (int b = tid; b < bin_k; b += threads) mass += mem.row_masses[b];
            for (int i = tid; i < keep; i += threads) mass += weight(key_value(static_cast<uint32_t>(mem.list[i] >> 32)));
            block_exclusive_u64(mass, sh, &total);
            if (tid == 0) sh.threshold = mem.list[keep - 1], sh.total_k = total;
          }
          row_sync(q);
          floor = *at_rank(&sh.threshold, q, 0);
        } else {
          floor = by_digits(static_cast<uint64_t>(k), 0, false);
          uint64_t mass = 0;
          each([&](float v, int i, uint64_t w) {
            if (element(v, q.c0 + i) >= floor) mass += w;
          });
          mass = row_reduce(q, mass, [](uint64_t a, uint64_t b) { return a + b; }, sh.mass_k);
          if (lead && tid == 0) sh.total_k = mass;
          __syncthreads();
        }
      }
    }
    if (!(top_p < 1.f)) return floor;
    if (lead) {
      __syncthreads();
      const uint64_t need = needed_mass(top_p, sh.total_k);
      find_bin(mem.row_masses, need, sh, [&](int b, uint64_t before) {
        sh.bin_p = b;
        sh.before = before;
      });
      if (tid == 0) sh.need = need;
    }
    row_sync(q);
    const int bin_p = *at_rank(&sh.bin_p, q, 0);
    if (bin_p != bin_k || !listed) {
      gather(bin_p, 1);
      row_sync(q);
      if (!fits(1)) return by_digits(*at_rank(&sh.need, q, 0), floor, true);
      if (lead) sort_list(mem.list, static_cast<int>(sh.listed[1]));
    }
    if (lead) {
      __syncthreads();
      const int n = static_cast<int>(sh.listed[bin_p != bin_k || !listed]);
      const int per = (n + threads - 1) / threads, lo = min(tid * per, n), hi = min(lo + per, n);
      uint64_t mine = 0, total;
      for (int i = lo; i < hi; ++i) mine += weight(key_value(static_cast<uint32_t>(mem.list[i] >> 32)));
      uint64_t ahead = sh.before + block_exclusive_u64(mine, sh, &total);
      if (ahead < sh.need && sh.need <= ahead + mine)
        for (int i = lo; i < hi; ++i) {
          ahead += weight(key_value(static_cast<uint32_t>(mem.list[i] >> 32)));
          if (ahead >= sh.need) {
            sh.threshold = mem.list[i];
            break;
          }
        }
    }
    row_sync(q);
    return *at_rank(&sh.threshold, q, 0);
  }
};

template <class T>
__global__ void __launch_bounds__(kMaxThreads) choose_wide_kernel(ChooseParams p, int blocks, int segment) {
  extern __shared__ __align__(16) unsigned char dynamic[];
  __shared__ ChooseShared sh;
  grid_dep_wait();
  grid_dep_launch();
  const Part q = my_part(blocks, segment, p.in.width);
  const ChooseMemory mem(dynamic, segment, blocks);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5, row = q.row;
  load_part<T>(p.in, q, mem.x);
  const uint64_t best = row_best(q, mem.x, sh.best);
  const float t = p.in.temperature ? p.in.temperature[row] : 1.f;
  const int first = static_cast<int>(~static_cast<uint32_t>(best));
  if (best == 0 || best == ~0ull || t != t || t <= 0.f) {
    if (q.rank == 0 && tid == 0) {
      if (best == ~0ull || (best && t != t)) write_choice(p, row, Choice{-1, NAN});
      else if (best == 0) write_choice(p, row, Choice{-1, t != t ? NAN : 0.f});
      else write_choice(p, row, Choice{first, 1.f});
    }
    row_sync(q);
    return;
  }
  const float m = key_value(static_cast<uint32_t>(best >> 32));
  const Weights weight(m, t);
  const int k = p.top_k ? p.top_k[row] : 0;
  const float top_p = p.top_p ? p.top_p[row] : 1.f;
  uint64_t last = 0;
  if (k > 0 || top_p < 1.f) last = Border{q, mem, sh, weight, m, kBinsPerUnit / t}.find(k, top_p);
  else __syncthreads();  // the draw reads other threads' columns

  // Column order: each warp takes a run of the block's columns.
  const int run = ((q.n + warps - 1) / warps + 31) & ~31;
  const int lo = min(warp * run, q.n), hi = min(lo + run, q.n);
  auto kept = [&](int i) -> uint64_t {
    const float v = mem.x[i];
    return v > -INFINITY && element(v, q.c0 + i) >= last ? weight(v) : 0;
  };
  uint64_t mass = 0;
  for (int i = lo + lane; i < hi; i += 32) mass += kept(i);
#pragma unroll
  for (int o = 16; o; o >>= 1) mass += __shfl_xor_sync(~0u, mass, o);
  if (lane == 0) sh.scan[warp] = mass;
  __syncthreads();
  if (tid == 0) {
    uint64_t sum = 0;
    for (int w = 0; w < warps; ++w) {
      const uint64_t here = sh.scan[w];
      sh.scan[w] = sum;
      sum += here;
    }
    sh.scan[warps] = sum;
    sh.mass = sum;
  }
  row_sync(q);
  uint64_t total = 0, ahead = 0;
  for (int r = 0; r < q.blocks; ++r) {
    const uint64_t here = *at_rank(&sh.mass, q, r);
    if (r < q.rank) ahead += here;
    total += here;
  }
  if (!p.uniform) {
    if (q.rank == 0 && tid == 0) write_choice(p, row, Choice{first, static_cast<float>(kWeightOne / static_cast<double>(total))});
  } else {
    const uint64_t unit = drawn_unit(p.uniform[row], total);
    ahead += sh.scan[warp];
    const uint64_t end = ahead + sh.scan[warp + 1] - sh.scan[warp];
    if (unit >= ahead && unit < end) {
      for (int i0 = lo; i0 < hi; i0 += 32) {
        const uint64_t w = i0 + lane < hi ? kept(i0 + lane) : 0;
        uint64_t in = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint64_t u = __shfl_up_sync(~0u, in, o);
          if (lane >= o) in += u;
        }
        const bool here = w && unit >= ahead + in - w && unit < ahead + in;
        if (here)
          write_choice(p, row, Choice{q.c0 + i0 + lane, static_cast<float>(static_cast<double>(w) / static_cast<double>(total))});
        ahead += __shfl_sync(~0u, in, 31);
        if (__any_sync(~0u, here)) break;
      }
    }
  }
  if (q.blocks > 1) cg::this_cluster().sync();  // no block leaves while another reads from it
}

struct Shape {
  int blocks, segment, threads;
};

// Blocks per row: enough for segments of 8192 columns, and more where the rows alone would leave
// multiprocessors idle, as long as a segment keeps 1024 columns.
Shape wide_shape(const LogitParams& p) {
  const int rows = p.rows, width = p.width, sms = p.sms;
  int blocks = 1;
  while (blocks < kMaxBlocks && (width > blocks * 8192 || (static_cast<int64_t>(rows) * blocks < sms && width >= blocks * 2048)))
    blocks *= 2;
#ifdef MRN_TUNE
  if (getenv("MRN_B")) blocks = atoi(getenv("MRN_B"));
#endif
  Shape s;
  s.blocks = blocks;
  s.segment = ((width + blocks - 1) / blocks + 31) & ~31;
  s.threads = s.segment <= 2048 ? 256 : 512;
#ifdef MRN_TUNE
  if (getenv("MRN_T")) s.threads = atoi(getenv("MRN_T"));
#endif
  return s;
}

template <typename... Params, typename... Args>
cudaError_t launch_rows(void (*kernel)(Params...), int rows, const Shape& shape, size_t smem, cudaStream_t stream,
                        Args&&... args) {
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * shape.blocks);
  cfg.blockDim = dim3(shape.threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = static_cast<unsigned int>(pdl_attribute(attr));
  if (shape.blocks > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = shape.blocks;
    attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

}  // namespace

cudaError_t launch_adjust_wide(const AdjustParams& p, cudaStream_t s) {
  const Shape shape = wide_shape(p.in);
  return with_type(p.in.type, [&](auto v) {
    return launch_rows(adjust_wide_kernel<decltype(v)>, p.in.rows, shape, shape.segment * sizeof(float), s, p, shape.blocks,
                       shape.segment);
  });
}

cudaError_t launch_choose_wide(const ChooseParams& p, cudaStream_t s) {
  const Shape shape = wide_shape(p.in);
  const size_t smem = ChooseMemory::bytes(shape.segment, shape.blocks, p.top_k || p.top_p);
  return with_type(p.in.type, [&](auto v) {
    return launch_rows(choose_wide_kernel<decltype(v)>, p.in.rows, shape, smem, s, p, shape.blocks, shape.segment);
  });
}

cudaError_t prepare_policy_wide() {
  for (LogitType t : {LogitType::kF32, LogitType::kF16, LogitType::kBf16}) {
    const cudaError_t e = with_type(t, [&](auto v) {
      const cudaError_t r = cudaFuncSetAttribute(adjust_wide_kernel<decltype(v)>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 static_cast<int>(kMaxSegment * sizeof(float)));
      if (r != cudaSuccess) return r;
      return cudaFuncSetAttribute(choose_wide_kernel<decltype(v)>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  static_cast<int>(ChooseMemory::bytes(kMaxSegment, kMaxBlocks, true)));
    });
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace mrn
