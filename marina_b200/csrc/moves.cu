// The forward pass on move lists as a search holds them (one behind the other, with their lengths)
// instead of padded slot rows: mrn_evaluate_moves and mrn_choose_moves. The lists cross the bus once,
// about thirty actions a position instead of 224 slots, together with the rules of the call; the slot
// rows are built on the GPU (mrn_slot_table), the pass leaves raw slot logits, and the policy operators
// turn those into priors or into one move per position.
#include <string.h>

#include "../../include/marina_b200.h"
#include "kernels.cuh"
#include "launch.h"
#include "policy.cuh"
#include "policy_api.h"
#include "ptx.cuh"
#include "runtime.h"

namespace {

#define CK(call)                                                                                   \
  do {                                                                                             \
    const cudaError_t e_ = (call);                                                                 \
    if (e_ != cudaSuccess) {                                                                       \
      cudaGetLastError();                                                                          \
      return c->fail(MRN_ERR_CUDA, "%s: %s", #call, cudaGetErrorString(e_));                       \
    }                                                                                              \
  } while (0)

// out[t] = in[map[t]]: the priors of the lists' moves out of the slot rows.
__global__ void __launch_bounds__(256) gather_slots_kernel(const float* __restrict__ in, const int32_t* __restrict__ map,
                                                           float* __restrict__ out, int count) {
  mrn::grid_dep_wait();
  mrn::grid_dep_launch();
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t < count) out[t] = in[map[t]];
}

// One call's small arrays side by side, in pinned host memory and at the same offsets on the device.
struct Arena {
  size_t bytes = 0;
  size_t add(size_t b) {
    const size_t at = bytes;
    bytes += (b + 15) & ~size_t(15);
    return at;
  }
};

int grow(mrn_ctx* c, size_t bytes) {
  if (bytes <= c->moves_bytes) return MRN_OK;
  const size_t size = bytes + bytes / 2;  // calls of slowly rising sizes do not allocate each time
  CK(cudaStreamSynchronize(c->stream));
  if (c->moves_dev) cudaFree(c->moves_dev);
  if (c->moves_host) cudaFreeHost(c->moves_host);
  c->moves_dev = c->moves_host = nullptr;
  c->moves_bytes = 0;
  CK(cudaMalloc(&c->moves_dev, size));
  CK(cudaMallocHost(&c->moves_host, size));
  c->moves_bytes = size;
  return MRN_OK;
}

// `rows` rows of `len` 4-byte elements at `stride`, packed.
void pack_rows(void* to, const void* from, int rows, int64_t len, int64_t stride) {
  const uint8_t* src = static_cast<const uint8_t*>(from);
  if (stride == len || rows == 1) {
    memcpy(to, src, static_cast<size_t>(rows) * len * 4);
    return;
  }
  for (int r = 0; r < rows; ++r) memcpy(static_cast<uint8_t*>(to) + r * len * 4, src + r * stride * 4, len * 4);
}

struct MovesCall {
  int n;
  const uint8_t* boards;
  const int32_t *lengths, *actions;
  const mrn_rules* rules;
  const float* temperature;
  // mrn_evaluate_moves
  float* priors = nullptr;
  // mrn_choose_moves
  const int32_t* top_k = nullptr;
  const float *top_p = nullptr, *uniform = nullptr;
  int32_t* move = nullptr;
  float* prob = nullptr;
  float* wdl = nullptr;
};

int run_moves(mrn_ctx* c, const MovesCall& m) {
  const int n = m.n;
  if (n < 0) return c->fail(MRN_ERR_ARGUMENT, "n = %d", n);
  if (n > c->max_batch) return c->fail(MRN_ERR_BATCH_TOO_LARGE, "batch of %d positions exceeds max_batch %d", n, c->max_batch);
  if (n == 0) return MRN_OK;
  if (!m.boards || !m.lengths || !m.wdl || (!m.priors && !m.move)) return c->fail(MRN_ERR_ARGUMENT, "NULL buffer");
  int64_t total = 0;
  for (int i = 0; i < n; ++i) {
    if (m.lengths[i] < 0) return c->fail(MRN_ERR_ARGUMENT, "position %d: a list of %d moves", i, m.lengths[i]);
    if (m.lengths[i] > MRN_MAX_LEGAL)
      return c->fail(MRN_ERR_TOO_MANY_MOVES, "position %d with %d legal moves exceeds MAX_LEGAL %d", i, m.lengths[i], MRN_MAX_LEGAL);
    total += m.lengths[i];
  }
  if (total && !m.actions) return c->fail(MRN_ERR_ARGUMENT, "NULL buffer");
  if (static_cast<int64_t>(n) * MRN_MAX_LEGAL > INT32_MAX)
    return c->fail(MRN_ERR_BATCH_TOO_LARGE, "%d positions in one call", n);
  const mrn_rules* r = m.rules;
  mrn::RuleParams rules;
  int rc;
  if (r && r->columns) return c->fail(MRN_ERR_ARGUMENT, "rules: the moves are the columns; leave columns NULL");
  if (r && r->actions != MRN_ACTIONS) return c->fail(MRN_ERR_ARGUMENT, "rules: actions %d, not %d", r->actions, MRN_ACTIONS);
  if ((rc = mrn::rule_params(c, n, MRN_MAX_LEGAL, r, &rules))) return rc;
  rules.actions = MRN_ACTIONS;

  // The arena: inputs first, then what comes back.
  Arena a;
  const int count = static_cast<int>(total), words = (MRN_ACTIONS + 31) / 32;
  auto rows_of = [&](int64_t stride) { return stride ? n : 1; };
  const int mask_rows = rows_of(rules.mask_stride), bias_rows = rows_of(rules.bias_stride), history_rows = rows_of(rules.history_stride);
  const size_t lengths_at = a.add(size_t(n) * 4), entries_at = a.add(size_t(count) * 4);
  const size_t mask_at = rules.mask ? a.add(size_t(mask_rows) * words * 4) : 0;
  const size_t bias_ids_at = a.add(size_t(bias_rows) * rules.bias_len * 4), bias_values_at = a.add(size_t(bias_rows) * rules.bias_len * 4);
  const size_t history_at = a.add(size_t(history_rows) * rules.history_len * 4);
  struct PerRow {
    const void* from;
    size_t at;
    const void* on_device;
  } per_row[] = {{rules.history_lens, 0, nullptr}, {rules.repetition, 0, nullptr}, {rules.presence, 0, nullptr},
                 {rules.frequency, 0, nullptr},    {m.temperature, 0, nullptr},    {m.top_k, 0, nullptr},
                 {m.top_p, 0, nullptr},            {m.uniform, 0, nullptr}};
  for (PerRow& q : per_row)
    if (q.from) q.at = a.add(size_t(n) * 4);
  const size_t input_bytes = a.bytes;
  const size_t out_at = a.add(m.move ? size_t(n) * 4 : size_t(count) * 4), prob_at = m.move ? a.add(size_t(n) * 4) : 0;
  const size_t output_end = a.bytes;
  const size_t starts_at = a.add((size_t(n) + 1) * 4), map_at = a.add(size_t(count) * 4);

  CK(cudaSetDevice(c->device));
  mrn::Bucket* b = nullptr;
  if ((rc = mrn::slot_logits_bucket(c, n, &b)) || (rc = grow(c, a.bytes))) return rc;
  uint8_t *host = c->moves_host, *dev = c->moves_dev;
  memcpy(c->h_boards, m.boards, size_t(n) * MRN_BOARD_BYTES);
  memcpy(host + lengths_at, m.lengths, size_t(n) * 4);
  if (count) memcpy(host + entries_at, m.actions, size_t(count) * 4);
  if (rules.mask) {
    pack_rows(host + mask_at, rules.mask, mask_rows, words, rules.mask_stride);
    rules.mask = reinterpret_cast<const uint32_t*>(dev + mask_at);
    rules.mask_stride = mask_rows > 1 ? words : 0;
  }
  if (rules.bias_len) {
    pack_rows(host + bias_ids_at, rules.bias_actions, bias_rows, rules.bias_len, rules.bias_stride);
    pack_rows(host + bias_values_at, rules.bias_values, bias_rows, rules.bias_len, rules.bias_stride);
    rules.bias_actions = reinterpret_cast<const int32_t*>(dev + bias_ids_at);
    rules.bias_values = reinterpret_cast<const float*>(dev + bias_values_at);
    rules.bias_stride = bias_rows > 1 ? rules.bias_len : 0;
  }
  if (rules.history_len) {
    pack_rows(host + history_at, rules.history, history_rows, rules.history_len, rules.history_stride);
    rules.history = reinterpret_cast<const int32_t*>(dev + history_at);
    rules.history_stride = history_rows > 1 ? rules.history_len : 0;
  }
  for (PerRow& q : per_row)
    if (q.from) {
      memcpy(host + q.at, q.from, size_t(n) * 4);
      q.on_device = dev + q.at;
    }
  rules.history_lens = static_cast<const int32_t*>(per_row[0].on_device);
  rules.repetition = static_cast<const float*>(per_row[1].on_device);
  rules.presence = static_cast<const float*>(per_row[2].on_device);
  rules.frequency = static_cast<const float*>(per_row[3].on_device);
  rules.columns = c->legal, rules.columns_stride = MRN_MAX_LEGAL;

  const int P = b->positions;
  cudaStream_t s = c->stream;
  if ((rc = mrn::begin_pass(c, s))) return rc;
  CK(cudaMemcpyAsync(c->boards, c->h_boards, size_t(n) * MRN_BOARD_BYTES, cudaMemcpyHostToDevice, s));
  CK(cudaMemcpyAsync(dev, host, input_bytes, cudaMemcpyHostToDevice, s));
  if (P > n) {
    CK(cudaMemsetAsync(c->boards + size_t(n) * MRN_BOARD_BYTES, 0, size_t(P - n) * MRN_BOARD_BYTES, s));
    CK(cudaMemsetAsync(c->legal + size_t(n) * MRN_MAX_LEGAL, 0xff, size_t(P - n) * MRN_MAX_LEGAL * 4, s));
  }
  int32_t* map = reinterpret_cast<int32_t*>(dev + map_at);
  const mrn::SlotTableParams table{n, MRN_MAX_LEGAL, reinterpret_cast<int32_t*>(dev + lengths_at), count,
                                   reinterpret_cast<int32_t*>(dev + entries_at), reinterpret_cast<int32_t*>(dev + starts_at),
                                   c->legal, map, c->status};
  CK(mrn::launch_slot_table(table, s));
  CK(cudaGraphLaunch(b->slot_graph, s));
  const mrn::LogitParams in{c->slot_logits, mrn::LogitType::kF32, MRN_MAX_LEGAL, n, MRN_MAX_LEGAL, rules,
                            static_cast<const float*>(per_row[4].on_device), c->status};
  if (m.move) {
    const mrn::ChooseParams choose{in, static_cast<const int32_t*>(per_row[5].on_device),
                                   static_cast<const float*>(per_row[6].on_device),
                                   static_cast<const float*>(per_row[7].on_device), reinterpret_cast<int32_t*>(dev + out_at),
                                   nullptr, reinterpret_cast<float*>(dev + prob_at)};
    CK(mrn::launch_choose(choose, s));
  } else {
    const mrn::AdjustParams adjust{in, nullptr, 0, c->priors, MRN_MAX_LEGAL};
    CK(mrn::launch_adjust(adjust, s));
    if (count)
      CK(mrn::launch_kernel(gather_slots_kernel, dim3((count + 255) / 256), dim3(256), 0, s,
                            static_cast<const float*>(c->priors), static_cast<const int32_t*>(map),
                            reinterpret_cast<float*>(dev + out_at), count));
  }
  if (output_end > out_at) CK(cudaMemcpyAsync(host + out_at, dev + out_at, output_end - out_at, cudaMemcpyDeviceToHost, s));
  CK(cudaMemcpyAsync(c->h_wdl, c->wdl, size_t(n) * 3 * 4, cudaMemcpyDeviceToHost, s));
  CK(cudaMemcpyAsync(c->h_status, c->status, 4, cudaMemcpyDeviceToHost, s));
  if ((rc = mrn::end_pass(c, s))) return rc;
  // As in mrn_evaluate, the inputs are checked while the GPU runs: the kernels take any of them.
  int invalid = mrn::check_boards(c, n, m.boards);
  for (int64_t t = 0, p = 0, left = m.lengths[0]; t < total && !invalid; ++t) {
    while (left == 0) left = m.lengths[++p];
    --left;
    if (m.actions[t] < 0 || m.actions[t] >= MRN_ACTIONS)
      invalid = c->fail(MRN_ERR_ACTION, "position %lld: action %d outside [0, %d)", (long long)p, m.actions[t], MRN_ACTIONS);
  }
  CK(cudaStreamSynchronize(s));
  const int word = *c->h_status;
  if (word) {
    CK(cudaMemsetAsync(c->status, 0, 4, s));
    CK(cudaStreamSynchronize(s));
  }
  if (invalid) return invalid;
  if (word) return mrn::status_error(c, word);
  if (m.move) {
    memcpy(m.move, host + out_at, size_t(n) * 4);
    if (m.prob) memcpy(m.prob, host + prob_at, size_t(n) * 4);
  } else if (count) {
    memcpy(m.priors, host + out_at, size_t(count) * 4);
  }
  memcpy(m.wdl, c->h_wdl, size_t(n) * 3 * 4);
  return MRN_OK;
}

}  // namespace

extern "C" {

MRN_API int mrn_evaluate_moves(mrn_ctx* c, int n, const uint8_t* boards, const int32_t* lengths, const int32_t* actions,
                               const mrn_rules* rules, const float* temperature, float* priors, float* wdl) {
  if (!c) return MRN_ERR_ARGUMENT;
  std::lock_guard<std::mutex> lock(c->mu);
  if (n > 0 && !priors) return c->fail(MRN_ERR_ARGUMENT, "NULL buffer");
  MovesCall m{n, boards, lengths, actions, rules, temperature};
  m.priors = priors, m.wdl = wdl;
  return run_moves(c, m);
}

MRN_API int mrn_choose_moves(mrn_ctx* c, int n, const uint8_t* boards, const int32_t* lengths, const int32_t* actions,
                             const mrn_rules* rules, const float* temperature, const int32_t* top_k, const float* top_p,
                             const float* uniform, int32_t* move, float* prob, float* wdl) {
  if (!c) return MRN_ERR_ARGUMENT;
  std::lock_guard<std::mutex> lock(c->mu);
  if (n > 0 && !move) return c->fail(MRN_ERR_ARGUMENT, "NULL buffer");
  MovesCall m{n, boards, lengths, actions, rules, temperature};
  m.top_k = top_k, m.top_p = top_p, m.uniform = uniform, m.move = move, m.prob = prob, m.wdl = wdl;
  return run_moves(c, m);
}

}  // extern "C"
