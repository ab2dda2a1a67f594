// iam_rope.h -- frequencies of rotary positions (iam_rope.cu), for the operator and for the model's table.
#pragma once

#include "../../include/iam_b200.h"

namespace iam {

// IAM_ERR_ARG (and a message) for a configuration that iam_rope_config's comment does not allow.
int rope_check(const iam_rope_config* c);
// Radians per position of the rot_dim / 2 pairs, and the factor on the rotated values (of a checked configuration).
void rope_frequencies(const iam_rope_config& c, double* w, double* factor);

}  // namespace iam
