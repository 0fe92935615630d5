// Causal convolution of each channel with a few taps: what its launchers take.
#pragma once

#include "pairs.cuh"
#include "token_tiles.cuh"

namespace la {

struct ConvCall {
  TokenView x, d_out;
  const void *weight = nullptr;  // (channels, taps), contiguous
  const void *bias = nullptr;    // null, or (channels)
  const void *init = nullptr;    // null, or (batch, taps - 1, channels): the tokens before
  const void *lengths = nullptr;
  int lengths64 = 0;
  TokenSizes sizes;
  int taps = 0, silu = 0;
  int weight_dtype = 0;          // of weight and bias
  bool wide_in = false, wide_out = false;  // pairs of channels that are read alone, and those
                                           // that are written, start at their own size (set by
                                           // the launchers)
  // forward
  void *out = nullptr, *final_state = nullptr;
  // gradient
  const void *d_final = nullptr;  // null, or as init
  void *dx = nullptr, *d_init = nullptr;
  float *partial = nullptr;       // null, or rows of (channels * taps + channels)
};

constexpr int kConvMinTaps = 2, kConvMaxTaps = 4;

int launch_conv_fwd(const ConvCall &c, int dtype, cudaStream_t s);
int launch_conv_bwd(const ConvCall &c, int dtype, cudaStream_t s);
// Rows of `partial`.
int64_t conv_partial_rows(const TokenSizes &z);

}  // namespace la
