// Group norm of rows: what its launchers take.
#pragma once

#include "common.cuh"

namespace la {

// Rows of (n0, n1, channels), strides in elements, dense last dimension.
struct RowView {
  const void *p = nullptr;
  int64_t s0 = 0, s1 = 0;
};

struct GroupNormCall {
  RowView x, gate, d_out;       // gate.p null: none
  const void *weight = nullptr, *bias = nullptr;  // null: ones, zeros
  int weight_dtype = 0;         // of both
  int64_t rows = 0;
  uint32_t n1 = 1;              // rows of the inner leading dimension
  int groups = 1, size = 1;     // channels = groups * size
  int silu = 0;
  float eps = 0.f;
  float *stats = nullptr;       // (rows, groups, 2): mean (fp32: less the group's first value) and
                                // 1 / sqrt(var + eps); forward: or null
  void *out = nullptr;          // contiguous, as dx and d_gate
  void *dx = nullptr, *d_gate = nullptr;
  float *partial = nullptr;     // null, or rows of (channels for the weight, channels for the bias)
};

constexpr int kGroupMaxSize = 8192;

int launch_group_norm_fwd(const GroupNormCall &c, int dtype, cudaStream_t s);
// *partial_rows: how many rows of `partial` it writes (at most group_norm_partial_rows).
int launch_group_norm_bwd(const GroupNormCall &c, int dtype, int sm_count, int64_t *partial_rows,
                          cudaStream_t s);
int64_t group_norm_partial_rows(int64_t rows, int sm_count);

}  // namespace la
