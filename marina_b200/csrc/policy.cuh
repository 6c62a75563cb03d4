// The policy operators (policy.cu): slot tables built from move-list lengths, logits under
// penalties, biases and masks, and the choice of one action per row. A row is a position (or any
// request); its columns are either the actions in order or slots that name an action each.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace mrn {

// Widest row: columns of one row that the kernels take.
constexpr int kPolicyMaxWidth = 1 << 18;

enum class LogitType : int { kF32 = 0, kF16 = 1, kBf16 = 2 };

// What changes the logits of a batch of rows, every pointer on the device. Strides are in
// elements between rows; 0 makes every row share the first one's list.
struct RuleParams {
  int actions;              // ids lie in [0, actions)
  const int32_t* columns;   // [rows, width] action of each column, negative: empty; null: column = action
  int64_t columns_stride;
  const uint32_t* mask;     // [rows, ceil(actions / 32)], bit a % 32 of word a / 32: action a is allowed
  int64_t mask_stride;
  const int32_t* bias_actions;  // [rows, bias_len]
  const float* bias_values;
  int bias_len;
  int64_t bias_stride;
  const int32_t* history;   // [rows, history_len], the first history_lens[row] of them
  const int32_t* history_lens;
  int history_len;
  int64_t history_stride;
  const float* repetition;  // [rows] each, or null
  const float* presence;
  const float* frequency;
};

struct LogitParams {
  const void* logits;  // [rows, width]
  LogitType type;
  int64_t stride;
  int rows, width;
  RuleParams rules;
  const float* temperature;  // [rows], or null for 1
  int* status;               // device error word
};

// Rows of one call: every row may take eight blocks of a grid.
constexpr int kPolicyMaxRows = 1 << 27;

struct AdjustParams {
  LogitParams in;
  void* out;  // [rows, width] of the logits' type, or null; may be the logits themselves
  int64_t out_stride;
  float* priors;  // [rows, width], or null
  int64_t priors_stride;
};

struct ChooseParams {
  LogitParams in;
  const int32_t* top_k;   // [rows], or null
  const float* top_p;     // [rows], or null
  const float* uniform;   // [rows] in [0, 1), or null: the largest logit
  int32_t* column;        // [rows]
  int32_t* action;        // [rows], or null
  float* prob;            // [rows], or null
};

struct SlotTableParams {
  int rows, width;
  const int32_t* lengths;  // [rows]
  int count;               // entries, and map slots, in the buffers
  const int32_t* entries;  // [count]
  int32_t* starts;         // [rows + 1]
  int32_t* table;          // [rows, width]
  int32_t* map;            // [count], or null
  int* status;
};

cudaError_t launch_slot_table(const SlotTableParams& p, cudaStream_t s);
cudaError_t launch_adjust(const AdjustParams& p, cudaStream_t s);
cudaError_t launch_choose(const ChooseParams& p, cudaStream_t s);
// Loads every kernel above on the current device and opts it into its shared memory.
cudaError_t prepare_policy();

// Device error code: a list length outside [0, width], or lists longer than the entries given.
constexpr int kErrBadLength = 17;

}  // namespace mrn
