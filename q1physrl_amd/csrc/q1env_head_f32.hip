// q1env_head_f32.hip - the wide categorical head's kernels for float32 operands (q1head_calls.hpp).
#include "q1head_calls.hpp"

Q1_HEAD_DEFINE(f32, q1head::F32)
