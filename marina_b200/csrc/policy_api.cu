// C entry points of the policy operators (include/marina_b200.h): the checks of their arguments,
// and the launches of policy.cu.
#include <limits.h>

#include "../../include/marina_b200.h"
#include "policy.cuh"
#include "policy_api.h"
#include "runtime.h"

namespace mrn {

static_assert(MRN_MAX_WIDTH == kPolicyMaxWidth && MRN_MAX_ROWS == kPolicyMaxRows, "the header's limits are the kernels'");

namespace {

bool misaligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }

// Rows of `bytes` bytes, `stride` bytes apart.
struct Block {
  const void* base;
  int64_t stride, bytes;
  int rows;
};

// Whether two blocks share a byte. Blocks of one stride whose rows lie side by side (two column
// ranges of one matrix) do not.
bool overlap(const Block& a, const Block& b) {
  if (!a.base || !b.base) return false;
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a.base), pb = reinterpret_cast<uintptr_t>(b.base);
  const uintptr_t ea = pa + (a.rows - 1) * a.stride + a.bytes, eb = pb + (b.rows - 1) * b.stride + b.bytes;
  if (pa >= eb || pb >= ea) return false;
  if (a.stride != b.stride || a.stride == 0) return true;
  const int64_t apart = static_cast<int64_t>(pb > pa ? pb - pa : pa - pb) % a.stride;
  const int64_t low = pb > pa ? a.bytes : b.bytes, high = pb > pa ? b.bytes : a.bytes;
  return apart < low || a.stride - apart < high;
}

}  // namespace

int rule_params(mrn_ctx* c, int rows, int width, const mrn_rules* r, RuleParams* out) {
  *out = RuleParams{};
  out->actions = width;
  if (!r) return MRN_OK;
  if (r->actions < 1) return c->fail(MRN_ERR_ARGUMENT, "rules: actions %d < 1", r->actions);
  if (!r->columns && r->actions < width)
    return c->fail(MRN_ERR_ARGUMENT, "rules: %d actions for %d columns that are actions in order", r->actions, width);
  if (r->columns && (r->columns_stride < 0 || (r->columns_stride > 0 && r->columns_stride < width)))
    return c->fail(MRN_ERR_ARGUMENT, "rules: columns_stride %lld for rows of %d", (long long)r->columns_stride, width);
  const int64_t words = (static_cast<int64_t>(r->actions) + 31) / 32;
  if (r->mask && (r->mask_stride < 0 || (r->mask_stride > 0 && r->mask_stride < words)))
    return c->fail(MRN_ERR_ARGUMENT, "rules: mask_stride %lld for rows of %lld words", (long long)r->mask_stride,
                   (long long)words);
  if (r->bias_len < 0 || r->history_len < 0)
    return c->fail(MRN_ERR_ARGUMENT, "rules: a negative length (bias_len %d, history_len %d)", r->bias_len, r->history_len);
  if (r->bias_len > MRN_MAX_LIST || r->history_len > MRN_MAX_LIST)
    return c->fail(MRN_ERR_ARGUMENT, "rules: a list longer than %d (bias_len %d, history_len %d)", MRN_MAX_LIST, r->bias_len,
                   r->history_len);
  if (r->bias_len && (!r->bias_actions || !r->bias_values))
    return c->fail(MRN_ERR_ARGUMENT, "rules: bias_len %d without bias_actions and bias_values", r->bias_len);
  if (r->bias_len && (r->bias_stride < 0 || (r->bias_stride > 0 && r->bias_stride < r->bias_len)))
    return c->fail(MRN_ERR_ARGUMENT, "rules: bias_stride %lld for lists of %d", (long long)r->bias_stride, r->bias_len);
  if (r->history_len && !r->history) return c->fail(MRN_ERR_ARGUMENT, "rules: history_len %d without history", r->history_len);
  if (r->history_len && (r->history_stride < 0 || (r->history_stride > 0 && r->history_stride < r->history_len)))
    return c->fail(MRN_ERR_ARGUMENT, "rules: history_stride %lld for lists of %d", (long long)r->history_stride,
                   r->history_len);
  for (const void* p : {(const void*)r->columns, (const void*)r->mask, (const void*)r->bias_actions,
                        (const void*)r->bias_values, (const void*)r->history, (const void*)r->history_lens,
                        (const void*)r->repetition, (const void*)r->presence, (const void*)r->frequency})
    if (misaligned(p, 4)) return c->fail(MRN_ERR_ARGUMENT, "rules: a pointer is not aligned to 4 bytes");
  out->actions = r->actions;
  out->columns = r->columns, out->columns_stride = r->columns_stride;
  out->mask = r->mask, out->mask_stride = r->mask_stride;
  if (r->bias_len) {
    out->bias_actions = r->bias_actions, out->bias_values = r->bias_values;
    out->bias_len = r->bias_len, out->bias_stride = r->bias_stride;
  }
  if (r->history_len) {
    out->history = r->history, out->history_lens = r->history_lens;
    out->history_len = r->history_len, out->history_stride = r->history_stride;
    out->repetition = r->repetition, out->presence = r->presence, out->frequency = r->frequency;
  }
  return MRN_OK;
}

namespace {

int logit_params(mrn_ctx* c, int rows, int width, const void* logits, int type, int64_t stride, const mrn_rules* rules,
                 const float* temperature, LogitParams* out) {
  if (rows < 0 || rows > kPolicyMaxRows) return c->fail(MRN_ERR_ARGUMENT, "rows = %d (0..%d)", rows, kPolicyMaxRows);
  if (width < 1 || width > MRN_MAX_WIDTH) return c->fail(MRN_ERR_ARGUMENT, "width %d (1..%d)", width, MRN_MAX_WIDTH);
  if (type < MRN_TYPE_F32 || type > MRN_TYPE_BF16) return c->fail(MRN_ERR_ARGUMENT, "unknown type %d", type);
  if (stride < 0 || (stride > 0 && stride < width))
    return c->fail(MRN_ERR_ARGUMENT, "stride %lld for rows of %d", (long long)stride, width);
  if (!logits && rows) return c->fail(MRN_ERR_ARGUMENT, "logits is NULL");
  if (misaligned(logits, type == MRN_TYPE_F32 ? 4 : 2) || misaligned(temperature, 4))
    return c->fail(MRN_ERR_ARGUMENT, "logits or temperature is not aligned to its elements");
  out->logits = logits, out->type = static_cast<LogitType>(type), out->stride = stride;
  out->rows = rows, out->width = width, out->temperature = temperature, out->status = c->status;
  return rule_params(c, rows, width, rules, &out->rules);
}

int launched(mrn_ctx* c, cudaError_t e, const char* what) {
  if (e == cudaSuccess) return MRN_OK;
  cudaGetLastError();
  return c->fail(MRN_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

// Makes a context's device current, and the caller's again at the end.
struct DeviceScope {
  int before = -1;
  cudaError_t error;
  explicit DeviceScope(int device) {
    error = cudaGetDevice(&before);
    if (error == cudaSuccess && before != device) error = cudaSetDevice(device);
    else before = -1;
  }
  ~DeviceScope() {
    if (before >= 0) cudaSetDevice(before);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
};

// What a call reads of the context never changes, so that one on a stream of the caller's need not wait for a
// synchronous pass, which holds the context's lock until it is done. The context's own stream may be in
// capture under that lock (a batch size's first pass): a call on it has to wait.
struct OwnStreamLock {
  std::unique_lock<std::mutex> held;
  OwnStreamLock(mrn_ctx* c, void* stream) : held(c->mu, std::defer_lock) {
    if (!stream) held.lock();
  }
};

cudaStream_t stream_of(const mrn_ctx* c, void* stream) { return stream ? static_cast<cudaStream_t>(stream) : c->stream; }

}  // namespace

}  // namespace mrn

extern "C" {

MRN_API int mrn_slot_table(mrn_ctx* c, int rows, int width, const int32_t* lengths, int count, const int32_t* entries,
                           int32_t* starts, int32_t* table, int32_t* map, void* stream) {
  if (!c) return MRN_ERR_ARGUMENT;
  const mrn::OwnStreamLock lock(c, stream);
  if (rows < 0 || width < 1 || count < 0)
    return c->fail(MRN_ERR_ARGUMENT, "slot table: rows %d, width %d, count %d", rows, width, count);
  if (static_cast<int64_t>(rows) * width > INT_MAX)
    return c->fail(MRN_ERR_ARGUMENT, "slot table: %d rows of %d slots are more than 2^31 - 1", rows, width);
  if (!starts || (rows && (!lengths || !table)) || (count && !entries)) return c->fail(MRN_ERR_ARGUMENT, "NULL buffer");
  for (const void* p : {(const void*)lengths, (const void*)entries, (const void*)starts, (const void*)table, (const void*)map})
    if (mrn::misaligned(p, 4)) return c->fail(MRN_ERR_ARGUMENT, "slot table: a pointer is not aligned to 4 bytes");
  auto block = [](const void* p, int64_t elements) { return mrn::Block{elements ? p : nullptr, 0, elements * 4, 1}; };
  const mrn::Block in[] = {block(lengths, rows), block(entries, count)};
  const mrn::Block out[] = {block(starts, int64_t(rows) + 1), block(table, int64_t(rows) * width), block(map, count)};
  for (int i = 0; i < 3; ++i) {
    for (const mrn::Block& b : in)
      if (mrn::overlap(out[i], b)) return c->fail(MRN_ERR_ARGUMENT, "slot table: an output overlaps an input");
    for (int j = 0; j < i; ++j)
      if (mrn::overlap(out[i], out[j])) return c->fail(MRN_ERR_ARGUMENT, "slot table: two outputs overlap");
  }
  const mrn::DeviceScope device(c->device);
  if (device.error != cudaSuccess) return mrn::launched(c, device.error, "cudaSetDevice");
  const mrn::SlotTableParams p{rows, width, lengths, count, entries, starts, table, map, c->status};
  return mrn::launched(c, mrn::launch_slot_table(p, mrn::stream_of(c, stream)), "slot table");
}

MRN_API int mrn_adjust_logits(mrn_ctx* c, int rows, int width, const void* logits, int type, int64_t stride,
                              const mrn_rules* rules, const float* temperature, void* out, int64_t out_stride,
                              float* priors, int64_t priors_stride, void* stream) {
  if (!c) return MRN_ERR_ARGUMENT;
  const mrn::OwnStreamLock lock(c, stream);
  mrn::AdjustParams p{};
  const int rc = mrn::logit_params(c, rows, width, logits, type, stride, rules, temperature, &p.in);
  if (rc) return rc;
  if (!out && !priors) return c->fail(MRN_ERR_ARGUMENT, "adjust: neither out nor priors");
  const int size = type == MRN_TYPE_F32 ? 4 : 2;
  if (mrn::misaligned(out, size) || mrn::misaligned(priors, 4))
    return c->fail(MRN_ERR_ARGUMENT, "adjust: an output is not aligned to its elements");
  if ((out && out_stride < width && rows > 1) || (priors && priors_stride < width && rows > 1) || out_stride < 0 ||
      priors_stride < 0)
    return c->fail(MRN_ERR_ARGUMENT, "adjust: out_stride %lld, priors_stride %lld for rows of %d", (long long)out_stride,
                   (long long)priors_stride, width);
  if (rows == 0) return MRN_OK;
  const mrn::Block in{logits, stride * size, int64_t(width) * size, rows}, o{out, out_stride * size, int64_t(width) * size, rows},
      q{priors, priors_stride * 4, int64_t(width) * 4, rows};
  const bool in_place = out == logits && (out_stride == stride || rows == 1);
  if ((!in_place && mrn::overlap(in, o)) || mrn::overlap(in, q) || mrn::overlap(o, q))
    return c->fail(MRN_ERR_ARGUMENT, "adjust: an output overlaps the logits or the other output");
  p.out = out, p.out_stride = out_stride, p.priors = priors, p.priors_stride = priors_stride;
  const mrn::DeviceScope device(c->device);
  if (device.error != cudaSuccess) return mrn::launched(c, device.error, "cudaSetDevice");
  return mrn::launched(c, mrn::launch_adjust(p, mrn::stream_of(c, stream)), "adjust logits");
}

MRN_API int mrn_choose_actions(mrn_ctx* c, int rows, int width, const void* logits, int type, int64_t stride,
                               const mrn_rules* rules, const float* temperature, const int32_t* top_k,
                               const float* top_p, const float* uniform, int32_t* column, int32_t* action, float* prob,
                               void* stream) {
  if (!c) return MRN_ERR_ARGUMENT;
  const mrn::OwnStreamLock lock(c, stream);
  mrn::ChooseParams p{};
  const int rc = mrn::logit_params(c, rows, width, logits, type, stride, rules, temperature, &p.in);
  if (rc) return rc;
  if (!column && rows) return c->fail(MRN_ERR_ARGUMENT, "choose: column is NULL");
  for (const void* q : {(const void*)top_k, (const void*)top_p, (const void*)uniform, (const void*)column, (const void*)action,
                        (const void*)prob})
    if (mrn::misaligned(q, 4)) return c->fail(MRN_ERR_ARGUMENT, "choose: a pointer is not aligned to 4 bytes");
  if (rows == 0) return MRN_OK;
  p.top_k = top_k, p.top_p = top_p, p.uniform = uniform, p.column = column, p.action = action, p.prob = prob;
  const mrn::DeviceScope device(c->device);
  if (device.error != cudaSuccess) return mrn::launched(c, device.error, "cudaSetDevice");
  return mrn::launched(c, mrn::launch_choose(p, mrn::stream_of(c, stream)), "choose actions");
}

}  // extern "C"
