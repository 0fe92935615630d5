// Launchers of the single-token forms.
#pragma once

#include "recurrence.cuh"

namespace la {

struct RecurStep {
  const void *x, *gate, *input_gate;  // (batch, channels); input_gate null: none
  int64_t x_sb, gate_sb, input_sb;    // strides in elements
  const float *log_decay;             // null: a = sigmoid(gate)
  float *state;
  int64_t state_sb;
  void *out;                          // contiguous
  int64_t batch;
  int channels;
};

struct ConvStep {
  const void *x;
  int64_t x_sb;
  const void *weight, *bias;          // bias null: none
  int weight_dtype;
  void *state;                        // (batch, taps - 1, channels), dense but for the batch
  int64_t state_sb;
  void *out;                          // contiguous
  int64_t batch;
  int channels, taps, silu;
};

int launch_recur_step(const RecurStep &p, int dtype, cudaStream_t s);
int launch_conv_step(const ConvStep &p, int dtype, cudaStream_t s);

}  // namespace la
