// Sums of the columns of fp32 partial rows, for the gradients of weights: one
// partial row per CTA of the kernel before, added in a fixed order.
#pragma once

#include "common.cuh"
#include "tc_common.cuh"

namespace la {

// To be called once by every CTA of the kernel that writes the rows: lets the
// sum be set up meanwhile (it waits for all of that kernel before it reads).
__device__ __forceinline__ void column_sum_may_start() { tc::grid_dependents_launch(); }

// out[c] = sum of partial[r][c] over the rows, for a row of `columns`, of which
// the first `columns0` go to out0, the others to out1 (null: not stored).
// dtype: of both outputs.
int launch_column_sum(const float *partial, int64_t rows, int64_t columns, void *out0,
                      int64_t columns0, void *out1, int dtype, cudaStream_t s);

}  // namespace la
