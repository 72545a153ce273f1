// q1env_head_bf16.hip - the wide categorical head's kernels for bfloat16 operands (q1head_calls.hpp).
#include "q1head_calls.hpp"

Q1_HEAD_DEFINE(bf16, q1head::BF16)
