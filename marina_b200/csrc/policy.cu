// The policy operators; see policy.cuh for the arguments.
#include <type_traits>

#include "kernels.cuh"
#include "launch.h"
#include "policy.cuh"
#include "policy_rows.cuh"
#include "ptx.cuh"
#include "rows.cuh"

namespace mrn {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// ---- slot tables ------------------------------------------------------------------------
__device__ __forceinline__ int clamped_length(const SlotTableParams& p, int row) {
  const int n = p.lengths[row];
  return n < 0 ? 0 : n > p.width ? p.width : n;
}

// Exclusive sums of one value per thread in thread order, for a block of up to 32 warps;
// *total gets the sum of all. `sums` is shared memory of 32.
__device__ __forceinline__ int block_exclusive(int v, int* sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int in = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(~0u, in, o);
    if (lane >= o) in += u;
  }
  __syncthreads();
  if (lane == 31) sums[warp] = in;
  __syncthreads();
  const int w = lane < warps ? sums[lane] : 0;
  *total = __reduce_add_sync(~0u, w);
  return __reduce_add_sync(~0u, lane < warp ? w : 0) + in - v;
}

__device__ __forceinline__ void flag_length(const SlotTableParams& p) {
  if (p.status) atomicCAS(p.status, 0, kErrBadLength);
}

// ROWS rows of the table and the map, by one warp: table[r, s] = entries[first + s] for s < n, -1 behind;
// map[first + s] = r * width + s. The rows' entries are asked for together. QUADS: rows are 16-byte
// aligned, four slots to a store.
template <bool QUADS, int ROWS>
__device__ __forceinline__ void fill_rows(const SlotTableParams& p, const int (&row)[ROWS], const int (&first)[ROWS],
                                          const int (&n)[ROWS], int lane) {
  // Columns are counted without a sign: a row may have 2^31 - 1 of them, and the last step goes past that.
  const unsigned width = static_cast<unsigned>(p.width);
  unsigned listed[ROWS];  // 0 where the entries ended before, or there is no such row
#pragma unroll
  for (int i = 0; i < ROWS; ++i) listed[i] = static_cast<unsigned>(max(0, min(n[i], p.count - first[i])));
  if (QUADS) {
    for (unsigned s = 4 * lane; s < width; s += 128) {
      int4 v[ROWS];
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int32_t* from = p.entries + first[i] + s;
        v[i].x = s < listed[i] ? __ldg(from) : -1;
        v[i].y = s + 1 < listed[i] ? __ldg(from + 1) : -1;
        v[i].z = s + 2 < listed[i] ? __ldg(from + 2) : -1;
        v[i].w = s + 3 < listed[i] ? __ldg(from + 3) : -1;
      }
#pragma unroll
      for (int i = 0; i < ROWS; ++i)
        if (row[i] < p.rows) {
          int4* to = reinterpret_cast<int4*>(p.table + row[i] * p.width + s);
          if (ROWS > 1) __stcs(to, v[i]);  // a large table does not stay in L2 anyway (65.2 -> 63.5 us)
          else *to = v[i];
        }
    }
  } else {
    for (unsigned s = lane; s < width; s += 32) {
      int v[ROWS];
#pragma unroll
      for (int i = 0; i < ROWS; ++i) v[i] = s < listed[i] ? __ldg(p.entries + first[i] + s) : -1;
#pragma unroll
      for (int i = 0; i < ROWS; ++i)
        if (row[i] < p.rows) p.table[row[i] * p.width + s] = v[i];
    }
  }
  if (p.map) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
      for (unsigned s = lane; s < listed[i]; s += 32)
        p.map[first[i] + s] = row[i] * p.width + static_cast<int>(s);
  }
}

// Bound by HBM where there are many rows (262144 rows of 224: 64.2 us, 4.9 TB/s of the 6.57 measured for a
// copy), by the launch where there are few (4096 rows: 4.1 us). A warp takes a row whatever its width, so that
// rows of other widths than a multiple of four store four bytes a lane, and rows of less than 128 slots leave lanes
// idle.
//
// Few rows: one launch. Block b lays out the rows [b * per, (b + 1) * per), per <= 32, and finds where
// they start by adding up every length before them: reading up to 64 KB that all blocks share in L2
// takes less time than two more launches. 16384 rows: 7.3 us in one, 9.5 us in three; 32768: 12.3 and
// 11.3 us.
constexpr int kSlotsOneLaunch = 16384;

template <bool QUADS>
__global__ void __launch_bounds__(kThreads) slot_table_kernel(SlotTableParams p, int per) {
  __shared__ int sums[32];
  __shared__ int first[33];
  grid_dep_wait();
  grid_dep_launch();
  const int tid = threadIdx.x, lane = tid & 31;
  const int r0 = blockIdx.x * per, r1 = min(r0 + per, p.rows);
  int before = 0;
  for (int r = tid; r < r0; r += kThreads) before += clamped_length(p, r);
  int total;
  block_exclusive(before, sums, &total);
  if (tid < 32) {
    const int row = r0 + lane;
    const int n = row < r1 ? clamped_length(p, row) : 0;
    if (row < r1 && n != p.lengths[row]) flag_length(p);
    int in = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(~0u, in, o);
      if (lane >= o) in += u;
    }
    first[lane] = total + in - n;
    if (lane == 31) first[32] = total + in;
    if (row < r1) p.starts[row] = total + in - n;
    if (lane == 31 && r1 == p.rows) {
      p.starts[p.rows] = total + in;
      if (total + in > p.count) flag_length(p);
    }
  }
  __syncthreads();
  for (int r = tid >> 5; r0 + r < r1; r += kWarps)
    fill_rows<QUADS, 1>(p, {r0 + r}, {first[r]}, {first[r + 1] - first[r]}, lane);
}

// Many rows, in three launches. The first adds up the lengths of each chunk of rows, the second turns
// these sums into the chunks' starts, and the third lays the chunks out, a block each. A chunk's sum
// waits in `starts` itself, behind its first row: nobody but that chunk's block reads or writes it later.
constexpr int kChunkRows = 64;

__device__ __forceinline__ int32_t* chunk_sum(const SlotTableParams& p, int64_t chunk) {
  return p.starts + chunk * kChunkRows + 1;
}

__global__ void __launch_bounds__(kThreads) slot_sums_kernel(SlotTableParams p, int64_t chunks) {
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x & 31;
  const int64_t chunk = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (chunk >= chunks) return;
  int sum = 0;
#pragma unroll
  for (int i = 0; i < kChunkRows / 32; ++i) {
    const int64_t row = chunk * kChunkRows + 32 * i + lane;
    if (row < p.rows) {
      const int n = clamped_length(p, static_cast<int>(row));
      if (n != p.lengths[row]) flag_length(p);
      sum += n;
    }
  }
  sum = __reduce_add_sync(~0u, sum);
  if (lane == 0) *chunk_sum(p, chunk) = sum;
}

__global__ void __launch_bounds__(1024) slot_starts_kernel(SlotTableParams p, int64_t chunks) {
  __shared__ int sums[32];
  grid_dep_wait();
  grid_dep_launch();
  constexpr int kRun = 4;  // chunks of a thread
  int base = 0, total;
  for (int64_t c0 = 0; c0 < chunks; c0 += 1024 * kRun) {
    const int64_t c = c0 + static_cast<int64_t>(threadIdx.x) * kRun;
    int v[kRun], sum = 0;
#pragma unroll
    for (int i = 0; i < kRun; ++i) v[i] = c + i < chunks ? *chunk_sum(p, c + i) : 0;
#pragma unroll
    for (int i = 0; i < kRun; ++i) sum += v[i];
    int at = base + block_exclusive(sum, sums, &total);
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      if (c + i < chunks) *chunk_sum(p, c + i) = at;
      at += v[i];
    }
    base += total;
  }
  if (threadIdx.x == 0 && base > p.count) flag_length(p);
}

template <bool QUADS>
__global__ void __launch_bounds__(kThreads) slot_fill_kernel(SlotTableParams p) {
  __shared__ int first[kChunkRows + 1];
  grid_dep_wait();
  grid_dep_launch();
  const int tid = threadIdx.x, lane = tid & 31;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * kChunkRows;
  const int rows = static_cast<int>(min(static_cast<int64_t>(kChunkRows), p.rows - r0));
  if (tid < 32) {
    int at = *chunk_sum(p, blockIdx.x);
    __syncwarp();  // read before it is overwritten
#pragma unroll
    for (int i = 0; i < kChunkRows / 32; ++i) {
      const int r = 32 * i + lane;
      const int n = r < rows ? clamped_length(p, static_cast<int>(r0 + r)) : 0;
      int in = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(~0u, in, o);
        if (lane >= o) in += u;
      }
      first[r] = at + in - n;
      if (r < rows) p.starts[r0 + r] = at + in - n;
      at += __shfl_sync(~0u, in, 31);
    }
    if (lane == 0) {
      first[kChunkRows] = at;
      if (r0 + rows == p.rows) p.starts[p.rows] = at;
    }
  }
  __syncthreads();
  constexpr int kTogether = 4;  // rows of a warp: 65.2 us for 262144 rows of 224; one at a time 67.8, eight 75.1
  for (int r = tid >> 5; r < rows; r += kTogether * kWarps) {
    int row[kTogether], from[kTogether], n[kTogether];
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      const int q = r + i * kWarps;
      row[i] = q < rows ? static_cast<int>(r0) + q : p.rows;  // behind the last: not written
      from[i] = q < rows ? first[q] : 0;
      n[i] = q < rows ? first[q + 1] - first[q] : 0;
    }
    fill_rows<QUADS, kTogether>(p, row, from, n, lane);
  }
}

// ---- narrow rows: one warp each ------------------------------------------------------------
// A row of up to 512 columns (a slot row has 224) stays in the registers of one warp, column
// 32 k + lane in v[k]: nothing but warp shuffles between its steps, and every global read of the row
// in flight at once. K * 32 is the widest row of an instantiation.
// Bound by the latency of a row's steps: 8192 rows of 224 slots without lists adjust in 5.9 us (5.2 TB/s,
// inputs in L2), with 40 entries and 8 biases in 12.8 us: rows of more than 64 moves pay for all 256 columns,
// and the few with every slot filled come last. The choice takes 28 us; its first stall is for instructions
// (four unrolled sorts, of which neighbouring warps run different ones), then come f64 weights.
constexpr int kNarrowWarps = 4;
constexpr int kCompared = 128;  // longest lists that are compared with a row's columns entry by entry

// A warp's shared memory: a table from action to count (for slots), or a count for each column; then, for
// the choice, the columns that are left.
template <int K>
struct alignas(16) NarrowShared {
  union {
    ActionCounts<64 * K> table;  // twice the columns, a power of two
    struct {
      uint64_t kept[32 * K];  // weight of the i-th column that is left, 0 once it is cut off
      float x[32 * K];
      int column[32 * K];
    };
  };
};

// Adjusted logits of a row. Returns the k whose columns are not all masked or empty, a bit each: lists of
// moves fill the first slots only, and what follows can pass over the rest.
template <class T, int K, bool SLOTS>
__device__ __forceinline__ unsigned load_narrow(const LogitParams& p, int row, int lane, NarrowShared<K>& sh, float (&v)[K]) {
  const RuleParams& r = p.rules;
  const T* logits = static_cast<const T*>(p.logits) + row * p.stride;
  const Penalties pen = row_penalties(r, row);
  const uint32_t* mask = r.mask ? r.mask + row * r.mask_stride : nullptr;
  const int32_t* history = r.history + row * r.history_stride;
  const int32_t* ids = r.bias_actions + row * r.bias_stride;
  const float* values = r.bias_values + row * r.bias_stride;
  const int biases = r.bias_len;
  // Everything that the row reads first is asked for at once: the first of both lists, whether the row
  // has that many entries or not, slots and logits.
  constexpr int kAhead = 2;  // history entries of a lane
  int seen[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u) seen[u] = r.history && lane + 32 * u < r.history_len ? history[lane + 32 * u] : -1;
  int id = lane < biases ? ids[lane] : -1;
  float value = lane < biases ? values[lane] : 0.f;
  int a[K], at[K];  // the column's action, -1 where it is masked or empty; its count's place
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = 32 * k + lane;
    a[k] = -1;
    v[k] = 0.f;
    if (c < p.width) {
      a[k] = SLOTS ? r.columns[row * r.columns_stride + c] : c;
      v[k] = as_float(logits[c]);
    }
  }
  unsigned used = 0;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (SLOTS && a[k] >= r.actions) {
      if (p.status) atomicCAS(p.status, 0, kErrBadAction);
      a[k] = -1;
    }
    at[k] = 32 * k + lane;
    if (mask && a[k] >= 0 && !((mask[a[k] >> 5] >> (a[k] & 31)) & 1)) a[k] = -1;
    if (__any_sync(~0u, a[k] >= 0)) used |= 1u << k;
  }
  if (SLOTS && pen.seen <= kCompared && biases <= kCompared) {
    // Short lists: every entry is shown to the columns of every lane, of which rows of up to 64 moves
    // have two. Measured on 8192 rows of 224 slots, 40 entries and 8 biases: 12.6 us, and 15.3 us with the
    // hash table, whose insertions take 7 us in the longest rows.
    auto compare = [&](auto columns) {
      constexpr int C = decltype(columns)::value;
      if (pen.seen > 0) {
        int c[C] = {};
        for (int e0 = 0; e0 < pen.seen; e0 += 32) {
          const int mine = e0 == 0 ? seen[0] : e0 == 32 ? seen[1] : e0 + lane < pen.seen ? history[e0 + lane] : -1;
          const int count = min(32, pen.seen - e0);
          for (int e = 0; e < count; ++e) {
            const int action = __shfl_sync(~0u, mine, e);
#pragma unroll
            for (int k = 0; k < C; ++k) c[k] += action == a[k];
          }
        }
#pragma unroll
        for (int k = 0; k < C; ++k)
          if (a[k] >= 0) v[k] = penalised(v[k], c[k], pen);
      }
      for (int e0 = 0; e0 < biases; e0 += 32) {
        if (e0) {
          id = e0 + lane < biases ? ids[e0 + lane] : -1;
          value = e0 + lane < biases ? values[e0 + lane] : 0.f;
        }
        const int count = min(32, biases - e0);
        for (int e = 0; e < count; ++e) {
          const int action = __shfl_sync(~0u, id, e);
          const float add = __shfl_sync(~0u, value, e);
#pragma unroll
          for (int k = 0; k < C; ++k)
            if (action == a[k]) v[k] = __fadd_rn(v[k], add);
        }
      }
    };
    if (used < 4) compare(std::integral_constant<int, 2>());
    else compare(std::integral_constant<int, K>());
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (a[k] < 0) v[k] = -INFINITY;
    return used;
  }
  if (pen.seen > 0 || (SLOTS && biases)) {
    if (SLOTS) {
#pragma unroll
      for (int i = 0; i < K / 2; ++i) {
        reinterpret_cast<int4*>(sh.table.keys)[32 * i + lane] = make_int4(-1, -1, -1, -1);
        reinterpret_cast<int4*>(sh.table.counts)[32 * i + lane] = make_int4(0, 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) sh.table.counts[32 * k + lane] = 0;
    }
    __syncwarp();
    if (SLOTS) {
#pragma unroll
      for (int k = 0; k < K; ++k)
        if ((used >> k) & 1 && a[k] >= 0) at[k] = sh.table.insert(a[k]);
      __syncwarp();
    }
    auto count = [&](int action) {
      const int h = action < 0 ? -1 : SLOTS ? sh.table.find(action) : action < p.width ? action : -1;
      if (h >= 0) atomicAdd(&sh.table.counts[h], 1);
    };
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (lane + 32 * u < pen.seen) count(seen[u]);
    for (int e = lane + 32 * kAhead; e < pen.seen; e += 32) count(history[e]);
    __syncwarp();
    if (pen.seen > 0) {
#pragma unroll
      for (int k = 0; k < K; ++k)
        if ((used >> k) & 1 && a[k] >= 0) v[k] = penalised(v[k], sh.table.counts[at[k]], pen);
    }
  }
  // Biases in the list's order: every lane looks one entry up, and the ones that name a column are
  // added one after the other.
  for (int e0 = 0; e0 < biases; e0 += 32) {
    if (e0) {
      id = e0 + lane < biases ? ids[e0 + lane] : -1;
      value = e0 + lane < biases ? values[e0 + lane] : 0.f;
    }
    const int h = id < 0 ? -1 : SLOTS ? sh.table.find(id) : id < p.width ? id : -1;
    unsigned todo = __ballot_sync(~0u, h >= 0);
    while (todo) {
      const int j = __ffs(todo) - 1;
      todo &= todo - 1;
      const int place = __shfl_sync(~0u, h, j);
      const float add = __shfl_sync(~0u, value, j);
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (at[k] == place && a[k] >= 0) v[k] = __fadd_rn(v[k], add);
    }
  }
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (a[k] < 0) v[k] = -INFINITY;
  return used;
}

template <class T, int K, bool SLOTS>
__global__ void __launch_bounds__(kNarrowWarps * 32) adjust_narrow_kernel(AdjustParams p) {
  __shared__ NarrowShared<K> shared[kNarrowWarps];
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.x * kNarrowWarps + warp;
  if (row >= p.in.rows) return;
  const int width = p.in.width;
  float v[K];
  const unsigned used = load_narrow<T, K, SLOTS>(p.in, row, lane, shared[warp], v);
  if (p.out) {
    T* out = static_cast<T*>(p.out) + row * p.out_stride;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (32 * k + lane < width) from_float(v[k], out + 32 * k + lane);
  }
  if (!p.priors) return;
  const float t = p.in.temperature ? p.in.temperature[row] : 1.f;
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < K; ++k)
    if ((used >> k) & 1) m = max_or_nan(m, v[k]);
  m = warp_max_or_nan(m);
  float* priors = p.priors + row * p.priors_stride;
  float sum = 0.f, inv;
  if (m > -INFINITY && m < INFINITY && t > 0.f) {
    const Exponential exponential(m, t);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float e = 0.f;
      if ((used >> k) & 1) e = exponential(v[k]);
      v[k] = e;
      sum += e;
    }
    inv = 1.f / warp_sum(sum);
  } else {
    // Nothing left: 0. A NaN, in the row or as t: NaN wherever something is left. Else the largest
    // logit's lowest column, or the columns at +inf.
    const bool nan = m != m || t != t;
    int first = -1;
    if (!nan && t <= 0.f) {
      first = kPolicyMaxWidth;
#pragma unroll
      for (int k = K - 1; k >= 0; --k)
        if (v[k] == m) first = 32 * k + lane;
      first = __reduce_min_sync(~0u, first);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const bool there = v[k] == m && (t > 0.f || 32 * k + lane == first);
      v[k] = v[k] == -INFINITY ? 0.f : nan ? NAN : there ? 1.f : 0.f;
      if (!nan) sum += v[k];
    }
    sum = warp_sum(sum);
    inv = sum == 0.f ? 1.f : 1.f / sum;
  }
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (32 * k + lane < width) priors[32 * k + lane] = v[k] * inv;
}

// Draws from the `left` <= 32 G columns in sh.x, which are in column order. With a cut-off they are
// sorted by (logit, lower column), and a weight is computed once for each column.
template <int G, int K>
__device__ __forceinline__ Choice draw_narrow(const ChooseParams& p, int row, int lane, NarrowShared<K>& sh, int left,
                                              const Weights& weight) {
  const int k = p.top_k ? p.top_k[row] : 0;
  const float top_p = p.top_p ? p.top_p[row] : 1.f;
  uint64_t kept[G];
  uint64_t total;
  if ((k > 0 && k < left) || top_p < 1.f) {
    uint64_t e[G];  // order key, then the complement of the place: larger is earlier
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int i = lane * G + g;
      e[g] = i < left ? static_cast<uint64_t>(order_key(sh.x[i])) << 32 | ~static_cast<uint32_t>(i) : 0;
    }
    warp_sort<G>(e, lane);
    const int most = k > 0 ? min(k, left) : left;
    uint64_t mine = 0;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      kept[g] = lane * G + g < most ? weight(key_value(static_cast<uint32_t>(e[g] >> 32))) : 0;
      mine += kept[g];
    }
    uint64_t ahead = warp_exclusive_u64(mine, lane);
    total = __shfl_sync(~0u, ahead + mine, 31);
    if (top_p < 1.f) {
      const uint64_t need = needed_mass(top_p, total);
      mine = 0;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const uint64_t w = kept[g];
        if (ahead >= need) kept[g] = 0;
        ahead += w;
        mine += kept[g];
      }
      total = warp_sum_u64(mine);
    }
    // back to column order
#pragma unroll
    for (int g = 0; g < G; ++g)
      if (lane * G + g < left) sh.kept[~static_cast<uint32_t>(e[g])] = kept[g];
    __syncwarp();
#pragma unroll
    for (int g = 0; g < G; ++g) kept[g] = lane * G + g < left ? sh.kept[lane * G + g] : 0;
  } else {
    uint64_t mine = 0;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      kept[g] = lane * G + g < left ? weight(sh.x[lane * G + g]) : 0;
      mine += kept[g];
    }
    total = warp_sum_u64(mine);
  }
  if (!p.uniform) return Choice{-1, share_of(static_cast<uint64_t>(kWeightOne), total)};  // the largest's
  const uint64_t unit = drawn_unit(p.uniform[row], total);
  uint64_t mine = 0;
#pragma unroll
  for (int g = 0; g < G; ++g) mine += kept[g];
  uint64_t ahead = warp_exclusive_u64(mine, lane);
  int place = -1;
  uint64_t w = 0;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    if (place < 0 && unit >= ahead && unit < ahead + kept[g]) place = lane * G + g, w = kept[g];
    ahead += kept[g];
  }
  const int owner = __ffs(__ballot_sync(~0u, place >= 0)) - 1;
  place = __shfl_sync(~0u, place, owner);
  w = __shfl_sync(~0u, w, owner);
  return Choice{sh.column[place], share_of(w, total)};
}

template <class T, int K, bool SLOTS>
__global__ void __launch_bounds__(kNarrowWarps * 32) choose_narrow_kernel(ChooseParams p) {
  __shared__ NarrowShared<K> shared[kNarrowWarps];
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.x * kNarrowWarps + warp;
  if (row >= p.in.rows) return;
  NarrowShared<K>& sh = shared[warp];
  float v[K];
  const unsigned used = load_narrow<T, K, SLOTS>(p.in, row, lane, sh, v);
  __syncwarp();
  const float t = p.in.temperature ? p.in.temperature[row] : 1.f;
  float m = -INFINITY;
  int left = 0;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (!((used >> k) & 1)) continue;
    m = max_or_nan(m, v[k]);
    const unsigned here = __ballot_sync(~0u, v[k] > -INFINITY);
    if (v[k] > -INFINITY) {
      const int i = left + __popc(here & ((1u << lane) - 1));
      sh.x[i] = v[k], sh.column[i] = 32 * k + lane;
    }
    left += __popc(here);
  }
  m = warp_max_or_nan(m);
  const bool nan = m != m || t != t;
  __syncwarp();
  Choice c{-1, nan ? NAN : 0.f};
  if (!nan && left) {
    if (t <= 0.f || !p.uniform) {
      int first = kPolicyMaxWidth;
#pragma unroll
      for (int k = K - 1; k >= 0; --k)
        if (v[k] == m) first = 32 * k + lane;
      c.column = __reduce_min_sync(~0u, first);
      c.prob = 1.f;
    }
    if (t > 0.f) {
      const Weights weight(m, t);
      Choice d;
      if (K == 1 || left <= 32) d = draw_narrow<1, K>(p, row, lane, sh, left, weight);
      else if (K == 2 || left <= 64) d = draw_narrow<2, K>(p, row, lane, sh, left, weight);
      else if (K == 4 || left <= 128) d = draw_narrow<4, K>(p, row, lane, sh, left, weight);
      else if (K == 8 || left <= 256) d = draw_narrow<8, K>(p, row, lane, sh, left, weight);
      else d = draw_narrow<16, K>(p, row, lane, sh, left, weight);
      if (!p.uniform) d.column = c.column;
      c = d;
    }
  }
  if (lane == 0) write_choice(p, row, c);
}

template <int N>
using Int = std::integral_constant<int, N>;

// Widest row of the one-warp kernels, whatever the number of rows. By one warp and by a block of 128
// threads, us without lists: 4096 rows of 512 adjust in 5.3 and 20.5, under a mask in 7.5 and 22.6, and
// choose by top_p in 54.0 and 91.7, under a mask in 15.2 and 43.8. One row: 2.5 and 4.0, 3.5 and 4.1; 20.5
// and 13.2, 5.9 and 9.4: only the choice from a few rows without a mask would be faster by a block (16 rows:
// 21.1 and 20.0).
constexpr int kNarrowWidth = 512;

dim3 narrow_grid(int rows) { return dim3((rows + kNarrowWarps - 1) / kNarrowWarps); }

// f(type, columns / 32, whether columns are slots) for the narrow kernels' instantiations.
template <class F>
cudaError_t with_narrow(const LogitParams& p, F&& f) {
  return with_type(p.type, [&](auto v) {
    auto with_width = [&](auto slots) {
      if (p.width <= 64) return f(v, Int<2>(), slots);
      if (p.width <= 256) return f(v, Int<8>(), slots);
      return f(v, Int<16>(), slots);
    };
    return p.rules.columns ? with_width(std::true_type()) : with_width(std::false_type());
  });
}

}  // namespace

cudaError_t launch_slot_table(const SlotTableParams& p, cudaStream_t s) {
  const bool quads = p.width % 4 == 0 && reinterpret_cast<uintptr_t>(p.table) % 16 == 0;
  if (p.rows <= kSlotsOneLaunch) {
    const int per = p.rows <= 2048 ? 4 : p.rows <= 8192 ? 8 : 32;
    const int blocks = p.rows ? (p.rows + per - 1) / per : 1;
    return launch_kernel(quads ? slot_table_kernel<true> : slot_table_kernel<false>, dim3(blocks), dim3(kThreads), 0, s, p,
                         per);
  }
  const int64_t chunks = (static_cast<int64_t>(p.rows) + kChunkRows - 1) / kChunkRows;
  cudaError_t e = launch_kernel(slot_sums_kernel, dim3(static_cast<unsigned>((chunks + kWarps - 1) / kWarps)), dim3(kThreads), 0,
                                s, p, chunks);
  if (e != cudaSuccess) return e;
  const PdlScope pdl(true);  // each waits for the one before it to finish before it reads anything
  if ((e = launch_kernel(slot_starts_kernel, dim3(1), dim3(1024), 0, s, p, chunks)) != cudaSuccess) return e;
  return launch_kernel(quads ? slot_fill_kernel<true> : slot_fill_kernel<false>, dim3(static_cast<unsigned>(chunks)),
                       dim3(kThreads), 0, s, p);
}

cudaError_t launch_adjust(const AdjustParams& p, cudaStream_t s) {
  if (p.in.width > kNarrowWidth) return launch_adjust_wide(p, s);
  return with_narrow(p.in, [&](auto v, auto k, auto slots) {
    return launch_kernel(adjust_narrow_kernel<decltype(v), k.value, slots.value>, narrow_grid(p.in.rows),
                         dim3(kNarrowWarps * 32), 0, s, p);
  });
}

cudaError_t launch_choose(const ChooseParams& p, cudaStream_t s) {
  if (p.in.width > kNarrowWidth) return launch_choose_wide(p, s);
  return with_narrow(p.in, [&](auto v, auto k, auto slots) {
    return launch_kernel(choose_narrow_kernel<decltype(v), k.value, slots.value>, narrow_grid(p.in.rows),
                         dim3(kNarrowWarps * 32), 0, s, p);
  });
}

cudaError_t prepare_policy() {
  cudaFuncAttributes a;
  cudaError_t e;
  if ((e = cudaFuncGetAttributes(&a, slot_sums_kernel)) != cudaSuccess) return e;
  if ((e = cudaFuncGetAttributes(&a, slot_starts_kernel)) != cudaSuccess) return e;
  if ((e = cudaFuncGetAttributes(&a, slot_fill_kernel<true>)) != cudaSuccess) return e;
  if ((e = cudaFuncGetAttributes(&a, slot_fill_kernel<false>)) != cudaSuccess) return e;
  if ((e = cudaFuncGetAttributes(&a, slot_table_kernel<true>)) != cudaSuccess) return e;
  if ((e = cudaFuncGetAttributes(&a, slot_table_kernel<false>)) != cudaSuccess) return e;
  for (LogitType t : {LogitType::kF32, LogitType::kF16, LogitType::kBf16})
    for (int width : {64, 256, 512})
      for (bool slots : {false, true}) {
        LogitParams in{};
        const int32_t some = 0;
        in.type = t, in.width = width, in.rules.columns = slots ? &some : nullptr;
        e = with_narrow(in, [&](auto v, auto k, auto sl) {
          const cudaError_t r = cudaFuncGetAttributes(&a, adjust_narrow_kernel<decltype(v), k.value, sl.value>);
          return r != cudaSuccess ? r : cudaFuncGetAttributes(&a, choose_narrow_kernel<decltype(v), k.value, sl.value>);
        });
        if (e != cudaSuccess) return e;
      }
  return prepare_policy_wide();
}

}  // namespace mrn
