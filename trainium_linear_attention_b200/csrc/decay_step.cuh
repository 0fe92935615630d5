// Launcher of the decayed linear attention's single-token form.
#pragma once

#include "common.cuh"

namespace la {

struct DecayStep {
  const void *q, *k, *v;  // (batch, heads, width), dense last dimension
  void *out;              // (batch, heads, dv), contiguous
  float *state;           // (batch, heads, dk, dv), dense last two dimensions
  const float *log_decay;
  int64_t q_sb, q_sh, k_sb, k_sh, v_sb, v_sh, state_sb, state_sh;  // strides in elements
  int64_t heads;
  int dk, dv;
  float scale;
};

int launch_decay_step(const DecayStep &p, int64_t batch, int dtype, cudaStream_t s);

}  // namespace la
