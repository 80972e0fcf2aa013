// The 8-bit product for short groups (int8_direct.hip): which calls it takes, and its launch.
// grouped_int8.hip's launch asks first.
#pragma once

#include "common.h"

namespace bux {

// Whether a product of `m` rows in `groups` groups goes to rows_split_kernel rather than
// grouped_int8.hip's rows_kernel.
bool int8_rows_direct(int64_t m, int32_t groups);

// As grouped_int8.hip's launch_rows: `list` a tile list of `slots` records, bias NULL or (groups,
// n) of out_dtype, y (height, n) of it.
int launch_int8_direct(const uint8_t* a_values, const float* a_scales, const uint8_t* b_values,
                       const float* b_scales, const void* list, int64_t slots, int32_t groups,
                       int64_t m, int64_t n, int64_t k, int64_t height, int out_dtype,
                       const void* bias, void* y, hipStream_t s);

}  // namespace bux
