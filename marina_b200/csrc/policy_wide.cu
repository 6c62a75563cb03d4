// The policy operators on rows of more than kNarrowWidth columns: a cluster of blocks takes a row,
// each block a contiguous segment of its columns, which it reads once into registers. Blocks of a row
// exchange maxima, sums and histograms through distributed shared memory.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>
#include <utility>

#include "kernels.cuh"
#include "launch.h"
#include "policy.cuh"
#include "policy_rows.cuh"
#include "ptx.cuh"
#include "rows.cuh"

namespace mrn {

namespace {

namespace cg = cooperative_groups;

constexpr int kMaxThreads = 1024;
constexpr int kMaxWarps = kMaxThreads / 32;
constexpr int kMaxBlocks = 8;  // of a cluster; what every device schedules
constexpr int kMaxSegment = kPolicyMaxWidth / kMaxBlocks;
constexpr int kQuads = 8;  // columns a thread holds, over four
static_assert(4 * kQuads <= 32, "a bit for each column of a thread");
constexpr int kListed = 512;  // entries of a bias list held at a time
constexpr int kSpan = 128;  // columns that a warp takes at a time, four to a lane

// This block's part of its row.
struct Part {
  int row, rank, blocks;
  int c0, n;  // columns [c0, c0 + n); c0 is a multiple of kSpan, n may be 0
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

// The registers of a row: thread t holds kQuads times four columns. Span k of a warp is the block's columns
// from kSpan * (warp + warps * k) on; with QUADS, where every row starts on a boundary of four elements,
// lane l holds columns 4 l + j of it, read four at a time; otherwise the columns 32 j + l, each read
// of the warp one contiguous piece.
template <bool QUADS>
__device__ __forceinline__ int span_column(int j) {
  const int lane = threadIdx.x & 31;
  return QUADS ? 4 * lane + j : 32 * j + lane;
}

__device__ __forceinline__ int span_base(int k) {
  const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  return kSpan * (warp + warps * k);
}

template <class T>
struct Quad {
  T v[4];
};

// The four columns that a lane holds of the span at `base`, -inf behind the n of the block's part.
template <bool QUADS, class T>
__device__ __forceinline__ void load_span(const T* from, int base, int n, float (&x)[4]) {
  if (QUADS && base + span_column<QUADS>(3) < n) {
    using Vector = typename std::conditional<sizeof(T) == 4, float4, uint2>::type;
    const Vector raw = __ldcs(reinterpret_cast<const Vector*>(from + base + span_column<QUADS>(0)));
    const Quad<T>& q = reinterpret_cast<const Quad<T>&>(raw);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = as_float(q.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = base + span_column<QUADS>(j);
      x[j] = i < n ? as_float(from[i]) : -INFINITY;
    }
  }
}

template <bool QUADS, class T>
__device__ __forceinline__ void store_span(T* to, int base, int n, const float (&x)[4]) {
  if (QUADS && base + span_column<QUADS>(3) < n) {
    using Vector = typename std::conditional<sizeof(T) == 4, float4, uint2>::type;
    Vector raw;
    Quad<T>& q = reinterpret_cast<Quad<T>&>(raw);
#pragma unroll
    for (int j = 0; j < 4; ++j) from_float(x[j], &q.v[j]);
    *reinterpret_cast<Vector*>(to + base + span_column<QUADS>(0)) = raw;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = base + span_column<QUADS>(j);
      if (i < n) from_float(x[j], to + i);
    }
  }
}

// Slots of a wide row, kTile of them at a time: a table of the actions that they name, which each entry of
// the row's lists is looked up in once.
constexpr int kTile = 2048;
constexpr int kChunk = 1024;  // bias entries looked up at a time
constexpr uint16_t kNoPlace = 0xffff;

struct alignas(16) SlotTile {
  ActionCounts<2 * kTile> table;
  uint16_t at[kTile];  // each slot's place in the table, kNoPlace where it is masked or empty
  int found[kChunk];   // each bias entry's place, -1 where no slot of the tile has its action
  int found_in[kChunk / 32];  // of 32 entries each
  struct {
    int place;
    float value;
  } hits[kChunk];  // the entries that were found, in the list's order
};
static_assert(2 * kTile < kNoPlace && kChunk == 32 * 32, "places in 16 bits, a warp's lanes for the groups of a chunk");

// Whether a row's lists are looked up in such a table. Shorter ones are compared with each slot entry by
// entry, which leaves room for more blocks on a multiprocessor: at 192 entries, 4096 rows of 700 slots choose
// in 178 us so and in 183 by the table (147 and 185 at 128 entries), 64 rows of 4096 adjust in 73 and 40.
__host__ __device__ constexpr bool long_lists(int history, int biases) { return history + biases > 192; }

// The adjusted logits of a block's slots into cells[0, q.n), where the row's lists are long. An entry costs
// one look-up for each tile of slots, so that a row takes its columns / kTile passes over its lists, not
// one for each column: 2 rows of 4096 slots with 65536 entries in both lists take 3.4 ms, compared column
// by column 86 ms. Bound by latency: a segment has one thread to 32 slots. `action` gives the action of a slot, -1
// where it is masked or empty.
template <class T, class F>
__device__ __forceinline__ void look_up_lists(const LogitParams& p, const Part& q, const Penalties& pen, const F& action,
                                              float* cells, SlotTile& tile) {
  const RuleParams& r = p.rules;
  const int n = q.n, tid = threadIdx.x, threads = blockDim.x, row = q.row;
  const int lane = tid & 31, warp = tid >> 5, warps = threads >> 5;
  const T* logits = static_cast<const T*>(p.logits) + row * p.stride + q.c0;
  const int32_t* history = r.history + row * r.history_stride;
  const int32_t* ids = r.bias_actions + row * r.bias_stride;
  const float* values = r.bias_values + row * r.bias_stride;
  for (int t0 = 0; t0 < n; t0 += kTile) {
    const int m = min(kTile, n - t0);
    __syncthreads();  // the tile before has been read
    for (int i = tid; i < kTile / 2; i += threads) {
      reinterpret_cast<int4*>(tile.table.keys)[i] = make_int4(-1, -1, -1, -1);
      reinterpret_cast<int4*>(tile.table.counts)[i] = make_int4(0, 0, 0, 0);
    }
    __syncthreads();
    for (int i = tid; i < m; i += threads) {
      const int a = action(t0 + i);
      tile.at[i] = a < 0 ? kNoPlace : static_cast<uint16_t>(tile.table.insert(a));
    }
    __syncthreads();
    for (int h = tid; h < pen.seen; h += threads) {
      const int a = history[h], place = a < 0 ? -1 : tile.table.find(a);
      if (place >= 0) atomicAdd(&tile.table.counts[place], 1);
    }
    __syncthreads();
    // Slot i is its thread's from here on.
    for (int i = tid; i < m; i += threads)
      cells[t0 + i] = tile.at[i] == kNoPlace ? -INFINITY
                                             : penalised(as_float(logits[t0 + i]), tile.table.counts[tile.at[i]], pen);
    for (int e0 = 0; e0 < r.bias_len; e0 += kChunk) {
      for (int g = warp; g < kChunk / 32; g += warps) {
        const int e = e0 + 32 * g + lane;
        const int id = e < r.bias_len ? ids[e] : -1, place = id < 0 ? -1 : tile.table.find(id);
        const unsigned here = __ballot_sync(~0u, place >= 0);
        tile.found[32 * g + lane] = place;
        if (lane == 0) tile.found_in[g] = __popc(here);
      }
      __syncthreads();
      const int in_group = tile.found_in[lane];
      const int hits = __reduce_add_sync(~0u, in_group);
      for (int g = warp; g < kChunk / 32; g += warps) {
        const int before = __reduce_add_sync(~0u, lane < g ? in_group : 0);
        const int place = tile.found[32 * g + lane];
        const unsigned here = __ballot_sync(~0u, place >= 0);
        if (place >= 0)
          tile.hits[before + __popc(here & ((1u << lane) - 1))] = {place, values[e0 + 32 * g + lane]};
      }
      __syncthreads();
      if (hits) {
        constexpr int kTogether = 4;  // slots of a thread: 3.4 ms in the case above, 5.9 ms one at a time
        for (int i0 = tid; i0 < m; i0 += kTogether * threads) {
          int place[kTogether];
          float v[kTogether];
#pragma unroll
          for (int u = 0; u < kTogether; ++u) {
            const int i = i0 + u * threads;
            place[u] = i < m ? tile.at[i] : kNoPlace;
            v[u] = i < m ? cells[t0 + i] : 0.f;
          }
          for (int h = 0; h < hits; ++h) {
            const int at = tile.hits[h].place;
            const float value = tile.hits[h].value;
#pragma unroll
            for (int u = 0; u < kTogether; ++u)
              if (at == place[u]) v[u] = __fadd_rn(v[u], value);
          }
#pragma unroll
          for (int u = 0; u < kTogether; ++u)
            if (i0 + u * threads < m) cells[t0 + i0 + u * threads] = v[u];
        }
      }
    }
  }
}

// The adjusted logits of the block's columns, -inf behind the last. `cells` is shared memory for the
// segment's columns, needed where the rows have a history or slots; LOOK_UP: rows of slots that may have
// long lists, with a SlotTile behind the cells.
template <class T, bool QUADS, bool LOOK_UP>
__device__ __forceinline__ void load_part(const LogitParams& p, const Part& q, int segment, float* cells,
                                          float (&x)[kQuads][4]) {
  const RuleParams& r = p.rules;
  const int n = q.n, c0 = q.c0, tid = threadIdx.x, threads = blockDim.x, row = q.row;
  const T* logits = static_cast<const T*>(p.logits) + row * p.stride + c0;
  const uint32_t* mask = r.mask ? r.mask + row * r.mask_stride : nullptr;
  const Penalties pen = row_penalties(r, row);
  const int32_t* history = r.history + row * r.history_stride;
  const int32_t* ids = r.bias_actions + row * r.bias_stride;
  const float* values = r.bias_values + row * r.bias_stride;
  if (LOOK_UP || r.columns) {
    const int32_t* columns = r.columns + row * r.columns_stride + c0;
    auto action = [&](int i) {  // -1 where the slot is masked or empty
      const int a = columns[i];
      if (a >= r.actions && p.status) atomicCAS(p.status, 0, kErrBadAction);
      return a >= 0 && a < r.actions && (!mask || (mask[a >> 5] >> (a & 31)) & 1) ? a : -1;
    };
    if (LOOK_UP && long_lists(pen.seen, r.bias_len)) {
      look_up_lists<T>(p, q, pen, action, cells, *reinterpret_cast<SlotTile*>(cells + segment));
    } else {
      for (int i = tid; i < n; i += threads) {
        const int a = action(i);
        float v = -INFINITY;
        if (a >= 0) {
          int count = 0;
          for (int h = 0; h < pen.seen; ++h) count += history[h] == a;
          v = penalised(as_float(logits[i]), count, pen);
          for (int e = 0; e < r.bias_len; ++e)
            if (ids[e] == a) v = __fadd_rn(v, values[e]);
        }
        cells[i] = v;
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kQuads; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = span_base(k) + span_column<QUADS>(j);
        x[k][j] = i < n ? cells[i] : -INFINITY;
      }
    __syncthreads();
    return;
  }
  // Everything that the row reads first is asked for at once: the history's first entries, whether the
  // row has that many or not, the logits, the first of the bias list, and the mask, of which lane
  // 4 k + j keeps the word for columns 32 j .. 32 j + 31 of span k.
  const int lane = tid & 31, warp = tid >> 5, warps = threads >> 5;
  int* counts = reinterpret_cast<int*>(cells);
  constexpr int kAhead = 2;  // history entries of a thread
  int seen[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u) seen[u] = r.history && tid + u * threads < r.history_len ? history[tid + u * threads] : -1;
#pragma unroll
  for (int k = 0; k < kQuads; ++k) load_span<QUADS>(logits, span_base(k), n, x[k]);
  const int biased = lane < r.bias_len ? ids[lane] : -1;
  uint32_t words = ~0u;
  if (mask) {
    const int i = kSpan * (warp + warps * (lane >> 2)) + 32 * (lane & 3);
    words = i < n ? __ldg(mask + ((c0 + i) >> 5)) : 0u;
  }
  if (r.history) {
    for (int i = tid; 4 * i < n; i += threads) reinterpret_cast<int4*>(counts)[i] = make_int4(0, 0, 0, 0);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (seen[u] >= c0 && seen[u] - c0 < n && tid + u * threads < pen.seen) atomicAdd(&counts[seen[u] - c0], 1);
    for (int h0 = tid + kAhead * threads; h0 < pen.seen; h0 += kAhead * threads) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) seen[u] = h0 + u * threads < pen.seen ? history[h0 + u * threads] : -1;
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (seen[u] >= c0 && seen[u] - c0 < n) atomicAdd(&counts[seen[u] - c0], 1);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kQuads; ++k) {
      const int i = span_base(k) + span_column<QUADS>(0);
      if (QUADS) {
        if (i < n) {
          const int4 c = *reinterpret_cast<const int4*>(counts + i);  // a cell behind n holds 0
          if (c.x | c.y | c.z | c.w) {
            x[k][0] = penalised(x[k][0], c.x, pen);
            x[k][1] = penalised(x[k][1], c.y, pen);
            x[k][2] = penalised(x[k][2], c.z, pen);
            x[k][3] = penalised(x[k][3], c.w, pen);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (i + 32 * j < n) x[k][j] = penalised(x[k][j], counts[i + 32 * j], pen);
      }
    }
  }
  if (mask) {
#pragma unroll
    for (int k = 0; k < kQuads; ++k) {
      uint32_t word = QUADS ? __shfl_sync(~0u, words, 4 * k + (lane >> 3)) : 0u;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!QUADS) word = __shfl_sync(~0u, words, 4 * k + j);
        if (!((word >> (span_column<QUADS>(j) & 31)) & 1)) x[k][j] = -INFINITY;
      }
    }
  }
  // A column's bias entries are all added by the warp that holds the column, which goes through the
  // whole list in its order, 32 entries at a time.
  auto add_listed = [&](unsigned id, int e) {
    const unsigned i = id - static_cast<unsigned>(c0);  // a negative id is far behind n
    const int span = static_cast<int>(i / kSpan);
    bool mine = i < static_cast<unsigned>(n) && span % warps == warp;
    if (mine && mask) mine = (mask[(c0 + i) >> 5] >> ((c0 + i) & 31)) & 1;
    unsigned todo = __ballot_sync(~0u, mine);
    if (!todo) return;
    const float value = mine ? values[e] : 0.f;
    const int in = static_cast<int>(i % kSpan);
    // where the column is: its register, and its lane in the upper bits
    const int place = 4 * (span / warps) + (QUADS ? in % 4 : in / 32) + ((QUADS ? in / 4 : in % 32) << 16);
    while (todo) {
      const int from = __ffs(todo) - 1;
      todo &= todo - 1;
      const int to = __shfl_sync(~0u, place, from);
      const float add = __shfl_sync(~0u, value, from);
      const int slot = to >> 16 == lane ? to & 0xffff : -1;
#pragma unroll
      for (int k = 0; k < kQuads; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (slot == 4 * k + j) x[k][j] = __fadd_rn(x[k][j], add);
    }
  };
  if (r.bias_len <= 32) {
    if (r.bias_len) add_listed(static_cast<unsigned>(biased), lane);
    return;
  }
  __shared__ int listed[kListed];
  for (int l0 = 0; l0 < r.bias_len; l0 += kListed) {
    const int length = min(kListed, r.bias_len - l0);
    __syncthreads();
    for (int e = tid; e < length; e += threads) listed[e] = ids[l0 + e];
    __syncthreads();
#pragma unroll 1
    for (int e = lane; e - lane < length; e += 32) add_listed(e < length ? static_cast<unsigned>(listed[e]) : ~0u, l0 + e);
  }
}

// The order key of the row's largest logit: 0 where nothing is left, all ones where a column that is
// left holds NaN.
__device__ __forceinline__ uint32_t row_best(const Part& q, const float (&x)[kQuads][4], Exchange<uint32_t>& ex, float& m) {
  m = -INFINITY;  // of this thread
#pragma unroll
  for (int k = 0; k < kQuads; ++k)
#pragma unroll
    for (int j = 0; j < 4; ++j) m = max_or_nan(m, x[k][j]);
  const uint32_t key = m != m ? ~0u : m == -INFINITY ? 0u : order_key(m);
  return row_reduce(q, key, [](uint32_t a, uint32_t b) { return a > b ? a : b; }, ex);
}

// The lowest column that holds m.
template <bool QUADS>
__device__ __forceinline__ int row_first(const Part& q, const float (&x)[kQuads][4], float m, Exchange<int>& ex) {
  int first = kPolicyMaxWidth;
#pragma unroll
  for (int k = kQuads - 1; k >= 0; --k)
#pragma unroll
    for (int j = 3; j >= 0; --j)
      if (x[k][j] == m) first = min(first, q.c0 + span_base(k) + span_column<QUADS>(j));
  return row_reduce(q, first, [](int a, int b) { return a < b ? a : b; }, ex);
}

// Bound by HBM: a logit is read once, stays in a register through maximum, exponential and sum, and
// leaves as its adjusted value and its prior. 4096 rows of 4672 f32 without lists take 38.4 us (6.0 TB/s of
// the 6.57 measured for a copy), with a history of 40 entries and 16 biases 46.7 us (5.0 TB/s): what a list
// names is looked up in shared memory between two barriers, and the row's other columns wait. 100 rows of
// 100003 f16 under a mask: 12.5 us without lists, 37.0 us with histories of 4096 and 300 biases: each of a
// row's eight blocks goes through the whole history, and each of its warps through the whole bias list.
template <class T, bool QUADS, bool LOOK_UP>
__global__ void __launch_bounds__(kMaxThreads) adjust_wide_kernel(AdjustParams p, int blocks, int segment) {
  extern __shared__ __align__(16) float cells[];
  __shared__ Exchange<uint32_t> ex_best;
  __shared__ Exchange<int> ex_first;
  __shared__ Exchange<float> ex_sum;
  grid_dep_wait();
  grid_dep_launch();
  const Part q = my_part(blocks, segment, p.in.width);
  float x[kQuads][4];
  load_part<T, QUADS, LOOK_UP>(p.in, q, segment, cells, x);
  if (p.out) {
    T* out = static_cast<T*>(p.out) + q.row * p.out_stride + q.c0;
#pragma unroll
    for (int k = 0; k < kQuads; ++k) store_span<QUADS>(out, span_base(k), q.n, x[k]);
  }
  if (!p.priors) return;
  const float t = p.in.temperature ? p.in.temperature[q.row] : 1.f;
  float mine;
  const uint32_t best = row_best(q, x, ex_best, mine);
  const float m = key_value(best);
  float sum = 0.f, inv;
  auto total = [&]() { return row_reduce(q, sum, [](float a, float b) { return a + b; }, ex_sum); };
  if (best && best != ~0u && t > 0.f && m != INFINITY) {
    const Exponential exponential(m, t);
#pragma unroll
    for (int k = 0; k < kQuads; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[k][j] = exponential(x[k][j]);
        sum += x[k][j];
      }
    inv = 1.f / total();
  } else {
    // Nothing left: 0. A NaN, in the row or as t: NaN wherever something is left. Else the largest
    // logit's lowest column, or the columns at +inf.
    const bool nan = best == ~0u || t != t;
    const int first = !nan && best && t <= 0.f ? row_first<QUADS>(q, x, m, ex_first) : -1;
#pragma unroll
    for (int k = 0; k < kQuads; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool there = x[k][j] == m && (t > 0.f || q.c0 + span_base(k) + span_column<QUADS>(j) == first);
        x[k][j] = x[k][j] == -INFINITY ? 0.f : nan ? NAN : there ? 1.f : 0.f;
        if (!nan) sum += x[k][j];
      }
    sum = total();
    inv = sum == 0.f ? 1.f : 1.f / sum;
  }
  float* priors = p.priors + q.row * p.priors_stride + q.c0;
#pragma unroll
  for (int k = 0; k < kQuads; ++k) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[k][j] *= inv;
    store_span<QUADS>(priors, span_base(k), q.n, x[k]);
  }
  if (q.blocks > 1) cg::this_cluster().sync();  // no block leaves while another reads from it
}

// ---- the choice ----------------------------------------------------------------------------
// Where a row is cut off (top_k, top_p), a histogram over the distance from the largest logit, kBins
// bins of 1/18 of a temperature that cover all weights above 0, says how far down the border lies.
// Where no more than kFew columns lie above the end of its bin, they are gathered in the row's first
// block, and one warp sorts them, cuts them off and draws: for a small top_k the histogram counts each
// thread's largest logit only, which puts the border a little too low. Otherwise the last column that is kept is
// found by its element, (order key of the logit, ~column), so that equal logits are told apart by
// their columns: among the elements of the border's bin, gathered and sorted, or digit by digit where
// even the bin holds more than the list; and the draw goes over the whole row again.
constexpr int kBins = 512;
constexpr float kBinsPerUnit = 18.f;  // exp(-512 / 18) < 2^-41: what lies below weighs 0
// Measured with and without the short way, for the few and for its list: 54.5 and 75.8 us for 2048 rows of
// 4672, 15.8 and 46.8 us for one row of 131072, 114 and 127 us for 64 rows of 150001.
constexpr int kFew = 256;

__host__ __device__ constexpr int list_capacity(int segment) { return segment <= 8192 ? 1024 : 4096; }

struct ChooseShared {
  int spans[kMaxSegment / kSpan + 1];  // columns that may weigh anything before each span
  Exchange<uint32_t> best;
  Exchange<int> first;
  Exchange<uint64_t> mass_k;
  uint64_t warp_sums[kMaxWarps];
  uint64_t scan[kMaxWarps + 1];
  uint64_t digits[256], digit_sums[256];
  uint64_t mass;         // kept by this block
  int digit;
  uint64_t passed;
  // written by the row's first block for the others
  int border, above;     // the border's bin; columns that lie in it or above
  int bin_k, bin_p;
  unsigned listed[4];    // elements gathered from above the border; from bin_k; from bin_p; from above few_k()'s border
  uint64_t before, need; // mass of the bins above bin_p, mass to reach
  uint64_t total_k;
  uint64_t threshold;
};

// Dynamic shared memory of a block: the segment, then where rows may be cut off the list, this block's
// histogram and the row's (the same memory where a block has the row to itself).
struct ChooseMemory {
  float* x;
  uint16_t* places;  // of the columns that may weigh anything, in their order, if they are half the segment or fewer
  uint64_t *list, *masses, *row_masses;
  uint32_t *counts, *row_counts;
  unsigned room;  // elements that the list holds
  int left;       // places, -1 where there were too many
  __device__ ChooseMemory(unsigned char* base, int segment, int blocks) {
    room = list_capacity(segment);
    x = reinterpret_cast<float*>(base);
    places = reinterpret_cast<uint16_t*>(x + segment);
    list = reinterpret_cast<uint64_t*>(places + segment / 2);
    masses = list + room;
    row_masses = blocks > 1 ? masses + kBins : masses;
    counts = reinterpret_cast<uint32_t*>(row_masses + kBins);
    row_counts = blocks > 1 ? counts + kBins : counts;
  }
  static size_t bytes(int segment, int blocks, bool cut) {
    const size_t histogram = kBins * (sizeof(uint64_t) + sizeof(uint32_t));
    return segment * sizeof(float) + segment / 2 * sizeof(uint16_t) +
           (cut ? list_capacity(segment) * sizeof(uint64_t) + histogram * (blocks > 1 ? 2 : 1) : 0);
  }
};

__device__ __forceinline__ uint64_t element(float x, int column) {
  return static_cast<uint64_t>(order_key(x)) << 32 | ~static_cast<uint32_t>(column);
}

// *cell += w, as two 32-bit additions: shared memory adds those by itself, 64-bit ones in a loop.
__device__ __forceinline__ void add_mass(uint64_t* cell, uint64_t w) {
  uint32_t* half = reinterpret_cast<uint32_t*>(cell);
  const uint32_t low = static_cast<uint32_t>(w), was = atomicAdd(half, low);
  const uint32_t high = static_cast<uint32_t>(w >> 32) + (was + low < was ? 1u : 0u);
  if (high) atomicAdd(half + 1, high);
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

// Sums over a row's histogram, by one warp: of groups of 32 bins first, all of them at once.
template <class V>
struct BinSums {
  static constexpr int kGroups = kBins / 32;
  const V* values;
  V sums[kGroups];

  __device__ __forceinline__ explicit BinSums(const V* bins) : values(bins) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) sums[g] = values[32 * g + lane];
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      if constexpr (sizeof(V) == 4) sums[g] = __reduce_add_sync(~0u, sums[g]);
      else sums[g] = warp_sum_u64(sums[g]);
    }
  }
  __device__ __forceinline__ uint64_t total() const {
    uint64_t sum = 0;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) sum += sums[g];
    return sum;
  }
  // The bin at which the sums from bin 0 on reach `need`, and the sum of the bins before it; -1, and the
  // sum of all, where they never do.
  __device__ __forceinline__ int reach(uint64_t need, uint64_t* before) const {
    uint64_t ahead = 0;
    int group = -1;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      if (group < 0) {
        if (ahead + sums[g] >= need) group = g;
        else ahead += sums[g];
      }
    }
    *before = ahead;
    if (group < 0) return -1;
    const int lane = threadIdx.x & 31;
    const uint64_t here = values[32 * group + lane];
    const uint64_t mine = ahead + warp_exclusive_u64(here, lane);
    const int first = __ffs(__ballot_sync(~0u, mine + here >= need)) - 1;
    *before = __shfl_sync(~0u, mine, first);
    return 32 * group + first;
  }
};

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

// The element at rank `need` - 1 of list[0, n), counted from the largest, or the one at which the
// weights reach `need`, into *found, by one block.
template <class W>
__device__ __forceinline__ void reach_in_list(uint64_t* list, int n, bool masses, uint64_t need, const W& weight,
                                              ChooseShared& sh, uint64_t* found) {
  const int threads = blockDim.x;
  if (n > kFew) {
    sort_list(list, n);
    const int per = (n + threads - 1) / threads;
    const int lo = min(static_cast<int>(threadIdx.x) * per, n), hi = min(lo + per, n);
    auto of = [&](int i) { return masses ? weight(key_value(static_cast<uint32_t>(list[i] >> 32))) : 1; };
    uint64_t mine = 0, total;
    for (int i = lo; i < hi; ++i) mine += of(i);
    uint64_t ahead = block_exclusive_u64(mine, sh, &total);
    if (ahead < need && need <= ahead + mine)
      for (int i = lo; i < hi; ++i) {
        ahead += of(i);
        if (ahead >= need) {
          *found = list[i];
          break;
        }
      }
  } else {
    // A short list is not sorted: every element adds up what lies ahead of it.
    for (int i = threadIdx.x; i < n; i += threads)
      sh.digits[i] = masses ? weight(key_value(static_cast<uint32_t>(list[i] >> 32))) : 1;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += threads) {
      const uint64_t e = list[i];
      uint64_t ahead = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j)
        if (list[j] > e) ahead += sh.digits[j];
      if (ahead < need && need <= ahead + sh.digits[i]) *found = e;
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

  // f(logit, column of the block) for this block's columns that may weigh anything.
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    if (mem.left >= 0) {
      for (int u = threadIdx.x; u < mem.left; u += blockDim.x) f(mem.x[mem.places[u]], mem.places[u]);
      return;
    }
    for (int i = 4 * threadIdx.x; i < q.n; i += 4 * blockDim.x) {
      const float4 v = *reinterpret_cast<const float4*>(mem.x + i);  // -inf from n on
      if (weight.maybe(v.x)) f(v.x, i);
      if (weight.maybe(v.y)) f(v.y, i + 1);
      if (weight.maybe(v.z)) f(v.z, i + 2);
      if (weight.maybe(v.w)) f(v.w, i + 3);
    }
  }

  // The elements of the bins from `lo` to `hi` into the first block's list, in any order.
  __device__ __forceinline__ void gather(int lo, int hi, int which) {
    unsigned* listed = at_rank(&sh.listed[which], q, 0);
    uint64_t* list = at_rank(mem.list, q, 0);
    // Most columns lie below the bins by any rounding.
    const float low = hi == kBins - 1 ? -INFINITY : m - (static_cast<float>(hi + 1) / per_bin) * 1.0001f - fabsf(m) * 1e-6f;
    auto add = [&](float v, int i) {
      const int b = bin(v);
      if (b < lo || b > hi || !weight.maybe(v)) return;
      const cg::coalesced_group here = cg::coalesced_threads();
      unsigned at = 0;
      if (here.thread_rank() == 0) at = atomicAdd(listed, here.size());
      at = here.shfl(at, 0) + here.thread_rank();
      if (at < mem.room) list[at] = element(v, q.c0 + i);
    };
    if (mem.left >= 0) {
      for (int u = threadIdx.x; u < mem.left; u += blockDim.x) add(mem.x[mem.places[u]], mem.places[u]);
      return;
    }
    for (int i = 4 * threadIdx.x; i < q.n; i += 4 * blockDim.x) {
      const float4 v = *reinterpret_cast<const float4*>(mem.x + i);
      if (fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) < low) continue;
      add(v.x, i);
      add(v.y, i + 1);
      add(v.z, i + 2);
      add(v.w, i + 3);
    }
  }

  // The element at which those from `floor` on, largest first, reach `need` in counts or in mass;
  // every block of the row finds it.
  __device__ uint64_t by_digits(uint64_t need, uint64_t floor, bool masses) {
    uint64_t prefix = 0, known = 0, over = 0;
    for (int shift = 56; shift >= 0; shift -= 8) {
      for (int b = threadIdx.x; b < 256; b += blockDim.x) sh.digits[b] = 0;
      __syncthreads();
      each([&](float v, int i) {
        const uint64_t e = element(v, q.c0 + i);
        if (e >= floor && (e & known) == prefix) add_mass(&sh.digits[(e >> shift) & 255], masses ? weight(v) : 1);
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

  // The blocks' histograms added up over the row, in the first block.
  __device__ __forceinline__ void add_up(bool counts, bool masses) const {
    row_sync(q);
    if (q.blocks == 1) return;
    // each block adds up a share of the bins and hands it to the first
    const int share = kBins / q.blocks;
    uint64_t* row_masses = at_rank(mem.row_masses, q, 0);
    uint32_t* row_counts = at_rank(mem.row_counts, q, 0);
    for (int b = q.rank * share + threadIdx.x; b < (q.rank + 1) * share; b += blockDim.x) {
      uint64_t s = 0;
      uint32_t c = 0;
      for (int r = 0; r < q.blocks; ++r) {
        if (masses) s += at_rank(mem.masses, q, r)[b];
        if (counts) c += at_rank(mem.counts, q, r)[b];
      }
      if (masses) row_masses[b] = s;
      if (counts) row_counts[b] = c;
    }
    row_sync(q);
  }

  __device__ __forceinline__ void clear(bool counts, bool masses) const {
    for (int b = threadIdx.x; b < kBins; b += blockDim.x) {
      if (counts) mem.counts[b] = 0;
      if (masses) mem.masses[b] = 0;
    }
    __syncthreads();
  }

  __device__ __forceinline__ void histogram(bool counts, bool masses) const {
    clear(counts, masses);
    each([&](float v, int) {
      const int b = bin(v);
      if (counts) atomicAdd(&mem.counts[b], 1u);
      if (masses) add_mass(&mem.masses[b], weight(v));
    });
    add_up(counts, masses);
  }

  // Whether no more than kFew columns lie above the end of the border's bin for a small k; the first
  // block's list then holds them. `mine` is the thread's largest logit: k of the row's threads have one
  // above the border, so that k of its columns lie there.
  __device__ __forceinline__ bool few_k(float mine, int k) {
    if (k > kFew / 2 || 2 * k > static_cast<int>(blockDim.x) * q.blocks) return false;
    clear(true, false);
    if (weight.maybe(mine)) atomicAdd(&mem.counts[bin(mine)], 1u);
    add_up(true, false);
    if (q.rank == 0 && threadIdx.x < 32) {
      uint64_t before;
      const int b = BinSums<uint32_t>(mem.row_counts).reach(static_cast<uint64_t>(k), &before);
      if (threadIdx.x == 0) sh.border = b < 0 ? kBins - 1 : b;
    }
    row_sync(q);
    gather(0, *at_rank(&sh.border, q, 0), 3);
    row_sync(q);
    return *at_rank(&sh.listed[3], q, 0) <= kFew;
  }

  // Histogram and border. True where few columns lie above the border's end, which the first block's
  // list then holds; sh.total_k is the row's mass where k <= 0.
  __device__ bool few(int k, float top_p) {
    histogram(true, k <= 0);
    if (q.rank == 0 && threadIdx.x < 32) {
      uint64_t before = 0, total = 0;
      int bin_k = -1, border;
      uint64_t above, ahead = 0, need = 0;
      if (k > 0) {
        bin_k = BinSums<uint32_t>(mem.row_counts).reach(static_cast<uint64_t>(k), &before);
        border = bin_k < 0 ? kBins - 1 : bin_k;
        above = bin_k < 0 ? before : before + mem.row_counts[bin_k];
      } else {
        const BinSums<uint64_t> masses(mem.row_masses);
        total = masses.total();
        need = needed_mass(top_p, total);
        border = masses.reach(need, &ahead);
        above = 0;
        for (int b = threadIdx.x; b <= border; b += 32) above += mem.row_counts[b];
        above = warp_sum_u64(above);
      }
      if (threadIdx.x == 0) {
        sh.bin_k = bin_k, sh.border = border, sh.above = static_cast<int>(above);
        // of bin_k, or of bin_p
        sh.need = k > 0 ? static_cast<uint64_t>(k) - before : need;
        sh.bin_p = border, sh.before = ahead, sh.total_k = total;
      }
    }
    row_sync(q);
    if (*at_rank(&sh.above, q, 0) > kFew) return false;
    gather(0, *at_rank(&sh.border, q, 0), 0);
    row_sync(q);
    return true;
  }

  // The last element that the row keeps, after few() said no.
  __device__ uint64_t find(int k, float top_p) {
    const int tid = threadIdx.x, threads = blockDim.x;
    const bool lead = q.rank == 0;
    uint64_t floor = 0;
    bool listed = false;  // the first block's list holds bin_k
    const int bin_k = *at_rank(&sh.bin_k, q, 0);
    if (k > 0) {
      histogram(false, true);
      if (lead) {
        if (tid < 32) {
          const uint64_t total = BinSums<uint64_t>(mem.row_masses).total();
          if (tid == 0) sh.total_k = total;
        }
        __syncthreads();
      }
      if (bin_k >= 0) {
        gather(bin_k, bin_k, 1);
        row_sync(q);
        listed = *at_rank(&sh.listed[1], q, 0) <= mem.room;
        if (listed) {
          if (lead) {
            const int n = static_cast<int>(sh.listed[1]);
            reach_in_list(mem.list, n, false, sh.need, weight, sh, &sh.threshold);
            uint64_t mass = 0, total;
            for (int b = tid; b < bin_k; b += threads) mass += mem.row_masses[b];
            for (int i = tid; i < n; i += threads)
              if (mem.list[i] >= sh.threshold) mass += weight(key_value(static_cast<uint32_t>(mem.list[i] >> 32)));
            block_exclusive_u64(mass, sh, &total);
            if (tid == 0) sh.total_k = total;
          }
          row_sync(q);
          floor = *at_rank(&sh.threshold, q, 0);
        } else {
          floor = by_digits(static_cast<uint64_t>(k), 0, false);
          uint64_t mass = 0;
          each([&](float v, int i) {
            if (element(v, q.c0 + i) >= floor) mass += weight(v);
          });
          mass = row_reduce(q, mass, [](uint64_t a, uint64_t b) { return a + b; }, sh.mass_k);
          if (lead && tid == 0) sh.total_k = mass;
          __syncthreads();
        }
      }
    }
    if (!(top_p < 1.f)) return floor;
    if (k > 0) {
      if (lead) {
        __syncthreads();
        if (tid < 32) {
          const uint64_t need = needed_mass(top_p, sh.total_k);
          uint64_t before;
          const int b = BinSums<uint64_t>(mem.row_masses).reach(need, &before);
          if (tid == 0) sh.bin_p = b, sh.before = before, sh.need = need;
        }
      }
      row_sync(q);
    }
    const int bin_p = *at_rank(&sh.bin_p, q, 0);
    const bool again = bin_p != bin_k || !listed;
    if (again) {
      gather(bin_p, bin_p, 2);
      row_sync(q);
      if (*at_rank(&sh.listed[2], q, 0) > mem.room) return by_digits(*at_rank(&sh.need, q, 0), floor, true);
    }
    if (lead) {
      __syncthreads();
      reach_in_list(mem.list, static_cast<int>(sh.listed[again ? 2 : 1]), true, sh.need - sh.before, weight, sh, &sh.threshold);
    }
    row_sync(q);
    return *at_rank(&sh.threshold, q, 0);
  }
};

// The places of the block's columns that may weigh anything, in column order, and how many they are;
// -1 where they are more than half the segment. A row under a grammar mask has few, which the passes
// that follow then go through without the gaps.
__device__ __forceinline__ int compact(const Part& q, const float* x, const Weights& weight, int segment,
                                       uint16_t* places, ChooseShared& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, spans = segment / kSpan;
  for (int s = warp; s < spans; s += warps) {
    const float4 v = reinterpret_cast<const float4*>(x + s * kSpan)[lane];
    const int count = weight.maybe(v.x) + weight.maybe(v.y) + weight.maybe(v.z) + weight.maybe(v.w);
    const int all = __reduce_add_sync(~0u, count);
    if (lane == 0) sh.spans[s] = all;
  }
  __syncthreads();
  if (warp == 0) {
    const int per = (spans + 31) / 32, lo = min(lane * per, spans), hi = min(lo + per, spans);
    int sum = 0;
    for (int i = lo; i < hi; ++i) sum += sh.spans[i];
    int ahead = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(~0u, ahead, o);
      if (lane >= o) ahead += u;
    }
    if (lane == 31) sh.spans[spans] = ahead;
    ahead -= sum;
    for (int i = lo; i < hi; ++i) {
      const int here = sh.spans[i];
      sh.spans[i] = ahead;
      ahead += here;
    }
  }
  __syncthreads();
  const int left = sh.spans[spans];
  if (left > segment / 2) return -1;
  const unsigned below = (1u << lane) - 1;
  for (int s = warp; s < spans; s += warps) {
    const float4 v = reinterpret_cast<const float4*>(x + s * kSpan)[lane];
    const bool in[4] = {weight.maybe(v.x), weight.maybe(v.y), weight.maybe(v.z), weight.maybe(v.w)};
    int at = sh.spans[s];
#pragma unroll
    for (int j = 0; j < 4; ++j) at += __popc(__ballot_sync(~0u, in[j]) & below);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (in[j]) places[at++] = static_cast<uint16_t>(s * kSpan + 4 * lane + j);
  }
  __syncthreads();
  return left;
}

// Cuts off and draws from the n <= 32 G elements of a list, by one warp; `total` is the row's mass
// where k <= 0, and `kept` shared memory for 32 G weights.
template <int G>
__device__ __forceinline__ Choice draw_sorted(const uint64_t* list, int n, int k, float top_p, uint64_t total,
                                           const float* uniform, const Weights& weight, uint64_t* kept) {
  const int lane = threadIdx.x & 31;
  uint64_t e[G], w[G];
#pragma unroll
  for (int g = 0; g < G; ++g) e[g] = lane * G + g < n ? list[lane * G + g] : 0;
  warp_sort<G>(e, lane);
  const int most = k > 0 ? min(k, n) : n;
  uint64_t mine = 0;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    w[g] = lane * G + g < most ? weight(key_value(static_cast<uint32_t>(e[g] >> 32))) : 0;
    mine += w[g];
  }
  uint64_t ahead = warp_exclusive_u64(mine, lane);
  if (k > 0) total = __shfl_sync(~0u, ahead + mine, 31);
  if (top_p < 1.f) {
    const uint64_t need = needed_mass(top_p, total);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const uint64_t here = w[g];
      if (ahead >= need) w[g] = 0;
      ahead += here;
    }
  }
  // in the order of the columns
  mine = 0;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    mine += w[g];
    kept[lane * G + g] = w[g];
    e[g] = w[g] ? e[g] << 32 | static_cast<uint32_t>(lane * G + g) : 0;
  }
  total = warp_sum_u64(mine);
  if (!uniform) return Choice{-1, share_of(static_cast<uint64_t>(kWeightOne), total)};  // the largest's
  const uint64_t unit = drawn_unit(*uniform, total);
  warp_sort<G>(e, lane);
  __syncwarp();
  mine = 0;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    w[g] = e[g] ? kept[static_cast<uint32_t>(e[g])] : 0;
    mine += w[g];
  }
  ahead = warp_exclusive_u64(mine, lane);
  int column = -1;
  uint64_t drawn = 0;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    if (unit >= ahead && unit < ahead + w[g]) column = static_cast<int>(~static_cast<uint32_t>(e[g] >> 32)), drawn = w[g];
    ahead += w[g];
  }
  const int owner = __ffs(__ballot_sync(~0u, column >= 0)) - 1;
  return Choice{__shfl_sync(~0u, column, owner),
                share_of(__shfl_sync(~0u, drawn, owner), total)};
}

// Cuts off and draws from the n <= kFew elements of a list, by one block; `total` is the row's mass where
// k <= 0. Nothing is sorted: each element counts what lies ahead of it, first by logit and then by
// column, which takes n steps of two short loops on all threads at once.
__device__ __forceinline__ void draw_few(const ChooseParams& p, int row, const uint64_t* list, int n, int k, float top_p,
                                         uint64_t total, float uniform, int first, const Weights& weight,
                                         ChooseShared& sh) {
  const int tid = threadIdx.x, threads = blockDim.x;
  if (n <= 64) {
    // The shortest lists: one warp, without a barrier.
    if (tid >= 32) return;
    const float* u = p.uniform ? &uniform : nullptr;
    Choice c = n <= 32 ? draw_sorted<1>(list, n, k, top_p, total, u, weight, sh.digits)
                       : draw_sorted<2>(list, n, k, top_p, total, u, weight, sh.digits);
    if (!u) c.column = first;
    if (tid == 0) write_choice(p, row, c);
    return;
  }
  uint64_t* w = sh.digits;
  for (int i = tid; i < n; i += threads) w[i] = weight(key_value(static_cast<uint32_t>(list[i] >> 32)));
  __syncthreads();
  uint64_t mass = 0;
  uint64_t* ahead = sh.digit_sums;
  for (int i = tid; i < n; i += threads) {
    const uint64_t e = list[i];
    uint64_t sum = 0;
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j)
      if (list[j] > e) ++rank, sum += w[j];
    const bool in = k <= 0 || rank < k;
    ahead[i] = in ? sum : ~0ull;
    if (in) mass += w[i];
  }
  if (k > 0) block_exclusive_u64(mass, sh, &total);
  const uint64_t need = top_p < 1.f ? needed_mass(top_p, total) : ~0ull;
  mass = 0;
  __syncthreads();
  for (int i = tid; i < n; i += threads) {
    if (ahead[i] >= need) w[i] = 0;
    mass += w[i];
  }
  block_exclusive_u64(mass, sh, &total);
  if (!p.uniform) {
    if (tid == 0) write_choice(p, row, Choice{first, share_of(static_cast<uint64_t>(kWeightOne), total)});
    return;
  }
  const uint64_t unit = drawn_unit(uniform, total);
  for (int i = tid; i < n; i += threads) {
    const uint32_t place = static_cast<uint32_t>(list[i]);  // ~column
    uint64_t before = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j)
      if (static_cast<uint32_t>(list[j]) > place) before += w[j];
    if (unit >= before && unit < before + w[i])
      write_choice(p, row, Choice{static_cast<int>(~place), share_of(w[i], total)});
  }
}

// Bound by the latency of its steps, each a pass over shared memory between barriers, and by instruction
// fetches (ncu: no_instruction and barrier are the first stalls): loops over shared memory are faster here
// than the same work unrolled over registers, whose code does not stay in the cache. Blocks of up to 1024
// threads leave it 64 registers, of which it spills 680 to 750 bytes a thread, blocks of 160 too. 2048 rows of
// 4672 f32 under a mask, top_k and top_p: 54.8 us; one row of 131072 bf16, top_k and top_p: 15.5 us; 64 rows of
// 150001 bf16 under a mask, top_p alone: 115 us, for which one block of 608 threads and 147 KB of shared memory fits a
// multiprocessor, in 3.5 waves.
template <class T, bool QUADS, bool LOOK_UP>
__global__ void __launch_bounds__(kMaxThreads) choose_wide_kernel(ChooseParams p, int blocks, int segment) {
  extern __shared__ __align__(16) unsigned char dynamic[];
  __shared__ ChooseShared sh;
  if (threadIdx.x < 4) sh.listed[threadIdx.x] = 0;
  grid_dep_wait();
  grid_dep_launch();
  const Part q = my_part(blocks, segment, p.in.width);
  ChooseMemory mem(dynamic, segment, blocks);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5, row = q.row;
  const float t = p.in.temperature ? p.in.temperature[row] : 1.f;
  const int k = p.top_k ? p.top_k[row] : 0;
  const float top_p = p.top_p ? p.top_p[row] : 1.f;
  const float uniform = p.uniform ? p.uniform[row] : 0.f;
  float x[kQuads][4], mine;
  load_part<T, QUADS, LOOK_UP>(p.in, q, segment, mem.x, x);
  const uint32_t best = row_best(q, x, sh.best, mine);
  const float m = key_value(best);
  const int first = best && best != ~0u && (t <= 0.f || !p.uniform) ? row_first<QUADS>(q, x, m, sh.first) : -1;
  if (best == 0 || best == ~0u || !(t > 0.f)) {
    if (q.rank == 0 && tid == 0) {
      const bool nan = best == ~0u || t != t;
      write_choice(p, row, nan ? Choice{-1, NAN} : best ? Choice{first, 1.f} : Choice{-1, 0.f});
    }
    row_sync(q);  // no block leaves while another reads from it
    return;
  }
  const Weights weight(m, t);
#pragma unroll
  for (int k = 0; k < kQuads; ++k)
    if (span_base(k) < segment) store_span<QUADS>(mem.x, span_base(k), segment, x[k]);
  mem.left = -1;
  __syncthreads();
  uint64_t last = 0;
  // Where every weight is needed first, or again, the row is gone through without its gaps.
  if (k <= 0) mem.left = compact(q, mem.x, weight, segment, mem.places, sh);
  if (k > 0 || top_p < 1.f) {
    Border border{q, mem, sh, weight, m, kBinsPerUnit / t};
    // Under a mask the threads' maxima say little about the few columns that are left: all are counted.
    // Rows of 4672 of which one column in 16 is left: 54.5 us per 2048 so and 61.3 by the maxima; one row
    // of 131072 without a mask: 19.8 and 15.8 us.
    const bool small = k > 0 && !p.in.rules.mask && border.few_k(mine, k);
    if (!small && k > 0) mem.left = compact(q, mem.x, weight, segment, mem.places, sh);
    if (small || border.few(k, top_p)) {
      // The first block draws out of its own memory, but it may not leave while another still reads from
      // it how many columns were gathered.
      if (q.blocks > 1) cg::this_cluster().barrier_arrive();
      if (q.rank == 0)
        draw_few(p, row, mem.list, static_cast<int>(sh.listed[small ? 3 : 0]), k, top_p, sh.total_k, uniform, first, weight, sh);
      if (q.blocks > 1) cg::this_cluster().barrier_wait();
      return;
    }
    last = border.find(k, top_p);
  }

  // Column order: each warp takes a run of the block's columns.
  const int columns = mem.left >= 0 ? mem.left : q.n;
  const int run = ((columns + warps - 1) / warps + 31) & ~31;
  const int lo = min(warp * run, columns), hi = min(lo + run, columns);
  auto place = [&](int u) { return mem.left >= 0 ? static_cast<int>(mem.places[u]) : u; };
  auto kept = [&](int i) -> uint64_t {
    const float v = mem.x[i];
    return weight.maybe(v) && element(v, q.c0 + i) >= last ? weight(v) : 0;
  };
  uint64_t mass = 0;
  for (int u = lo + lane; u < hi; u += 32) mass += kept(place(u));
  mass = warp_sum_u64(mass);
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
    if (q.rank == 0 && tid == 0) write_choice(p, row, Choice{first, share_of(static_cast<uint64_t>(kWeightOne), total)});
  } else {
    const uint64_t unit = drawn_unit(uniform, total);
    ahead += sh.scan[warp];
    const uint64_t end = ahead + sh.scan[warp + 1] - sh.scan[warp];
    if (unit >= ahead && unit < end) {
      for (int u0 = lo; u0 < hi; u0 += 32) {
        const int i = u0 + lane < hi ? place(u0 + lane) : 0;
        const uint64_t w = u0 + lane < hi ? kept(i) : 0;
        const uint64_t before = ahead + warp_exclusive_u64(w, lane);
        const bool here = w && unit >= before && unit < before + w;
        if (here)
          write_choice(p, row, Choice{q.c0 + i, share_of(w, total)});
        ahead = __shfl_sync(~0u, before + w, 31);
        if (__any_sync(~0u, here)) break;
      }
    }
  }
  if (q.blocks > 1) cg::this_cluster().sync();  // no block leaves while another reads from it
}

constexpr int kWholeRow = 16384;

struct Shape {
  int blocks, segment, threads;
};

// Blocks per row, and threads: as many as hold the segment. A row of up to 16384 columns is one block's,
// wider ones have four or eight blocks of 4097 to 8192 columns, or eight of up to 32768. The rule looks at
// the width alone and is one for both operators, which does not suit all of them (us by 1 / 2 / 4 / 8 blocks, logits
// without lists, the choice by top_p alone):
//                     adjust                      choose
//   1 x 4672           3.6 / 5.2 / 5.5 / 5.9      32.4 / 24.1 / 20.4 / 18.5
//   512 x 4672         5.7 / 8.2 / 14.9 / 29.7    40.3 / 56.5 / 70.7 / 101.0
//   1 x 16000          5.8 / 5.7 / 5.5 / 5.9      36.8 / 40.5 / 37.0 / 25.2
//   512 x 16000       16.6 / 20.0 / 20.2 / 31.9  116.3 / 103.8 / 143.9 / 164.9
//   1 x 60000            - / 10.7 / 7.6 / 6.4        - / 44.2 / 45.0 / 41.2
//   128 x 60000          - / 22.8 / 22.4 / 21.7      - / 106.1 / 149.0 / 116.7
//   1 x 100000           -  /  -  / 9.9 / 7.7        -  /  -  / 48.4 / 43.5
//   128 x 100000         -  /  -  / 44.9 / 44.3      -  /  -  / 191.4 / 328.8
// Adjust is within 7 % of its best everywhere. The choice is not: a single row of one block would be faster on
// eight, and many rows of 100000 on four, as a segment above 8192 columns takes a list of 32 KB
// (list_capacity) and leaves room for one block on a multiprocessor.
Shape wide_shape(const LogitParams& p) {
  const int width = p.width;
  int blocks = 1;
  while (width > kWholeRow && blocks < kMaxBlocks && width > blocks * 8192) blocks *= 2;
  Shape s;
  s.blocks = blocks;
  s.segment = ((width + blocks - 1) / blocks + kSpan - 1) / kSpan * kSpan;
  s.threads = (s.segment + kQuads * kSpan - 1) / (kQuads * kSpan) * 32;
  if (s.threads < 128) s.threads = 128;
  return s;
}

bool may_look_up(const LogitParams& p) { return p.rules.columns && long_lists(p.rules.history_len, p.rules.bias_len); }

// f(type, whether four columns are read at once, whether lists may be looked up) for the instantiations.
// Columns are read so where each row of logits and of the outputs starts on a boundary of four elements.
// The look-up has kernels of its own, as its code costs the others registers (4096 rows of 4672, adjust:
// 51.5 us with it and 48.7 without), and they read column by column, as they go through shared memory first.
template <class F>
cudaError_t with_wide(const LogitParams& p, bool quads, F&& f) {
  return with_type(p.type, [&](auto v) {
    if (may_look_up(p)) return f(v, std::false_type(), std::true_type());
    return quads ? f(v, std::true_type(), std::false_type()) : f(v, std::false_type(), std::false_type());
  });
}

bool quad_rows(const void* base, int64_t stride, int size) {
  return reinterpret_cast<uintptr_t>(base) % (4 * size) == 0 && stride % 4 == 0;
}

bool quad_rows(const LogitParams& p) { return quad_rows(p.logits, p.stride, p.type == LogitType::kF32 ? 4 : 2); }

// Shared memory that load_part uses.
size_t load_bytes(const LogitParams& p, int segment) {
  return segment * sizeof(float) + (may_look_up(p) ? sizeof(SlotTile) : 0);
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
  const bool quads = quad_rows(p.in) && (!p.out || quad_rows(p.out, p.out_stride, p.in.type == LogitType::kF32 ? 4 : 2)) &&
                     (!p.priors || quad_rows(p.priors, p.priors_stride, 4));
  const size_t smem = p.in.rules.history || p.in.rules.columns ? load_bytes(p.in, shape.segment) : 0;
  return with_wide(p.in, quads, [&](auto v, auto q, auto look_up) {
    return launch_rows(adjust_wide_kernel<decltype(v), q.value, look_up.value>, p.in.rows, shape, smem, s, p, shape.blocks,
                       shape.segment);
  });
}

cudaError_t launch_choose_wide(const ChooseParams& p, cudaStream_t s) {
  const Shape shape = wide_shape(p.in);
  const size_t smem = std::max(ChooseMemory::bytes(shape.segment, shape.blocks, p.top_k || p.top_p),
                               load_bytes(p.in, shape.segment));
  return with_wide(p.in, quad_rows(p.in), [&](auto v, auto q, auto look_up) {
    return launch_rows(choose_wide_kernel<decltype(v), q.value, look_up.value>, p.in.rows, shape, smem, s, p, shape.blocks,
                       shape.segment);
  });
}

cudaError_t prepare_policy_wide() {
  for (LogitType t : {LogitType::kF32, LogitType::kF16, LogitType::kBf16})
    for (int form : {0, 1, 2}) {  // one column at a time, four, long lists of slots
      LogitParams in{};
      const int32_t some = 0;
      in.type = t, in.rules.columns = form == 2 ? &some : nullptr, in.rules.history_len = 1 << 20;
      const cudaError_t e = with_wide(in, form == 1, [&](auto v, auto q, auto look_up) {
        const cudaError_t r = cudaFuncSetAttribute(adjust_wide_kernel<decltype(v), q.value, look_up.value>,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   static_cast<int>(kMaxSegment * sizeof(float) + sizeof(SlotTile)));
        if (r != cudaSuccess) return r;
        return cudaFuncSetAttribute(choose_wide_kernel<decltype(v), q.value, look_up.value>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    static_cast<int>(std::max(ChooseMemory::bytes(kMaxSegment, kMaxBlocks, true),
                                                              kMaxSegment * sizeof(float) + sizeof(SlotTile))));
      });
      if (e != cudaSuccess) return e;
    }
  return cudaSuccess;
}

}  // namespace mrn
