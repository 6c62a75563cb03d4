// The policy operators' argument checks, for the entry points that run them inside a pass.
#pragma once

#include "../../include/marina_b200.h"
#include "policy.cuh"
#include "runtime.h"

namespace mrn {
// Checks `rules` (null: none) for rows of `width` columns and converts them; an mrn_status, with the
// message in the context.
int rule_params(mrn_ctx* c, int rows, int width, const mrn_rules* rules, RuleParams* out);
}  // namespace mrn
