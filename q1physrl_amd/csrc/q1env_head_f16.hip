// q1env_head_f16.hip - the wide categorical head's kernels for float16 operands (q1head_calls.hpp).
#include "q1head_calls.hpp"

Q1_HEAD_DEFINE(f16, q1head::F16)
