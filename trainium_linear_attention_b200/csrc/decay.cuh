// Linear attention with a decay for each head: what its launchers share.
//
//   S_t = e^g S_{t-1} + b_t v_t^T,   out_t = a_t S_t     (g = log_decay[head])
//
// over a chunk of C tokens that starts with the state S:
//   out = (tril(A B^T) * lambda^(i-j)) V + lambda^(i+1) A S,
//   S'  = lambda^C S + (B * lambda^(C-1-j))^T V,         lambda = e^g.
//
// One walk of this recurrence serves the forward pass and every gradient
// ("role"), with a, b, v bound to different tensors:
//   out  a = q,     b = k,     v = v,     seed S_0
//   dq   a = d_out, b = v,     v = k,     seed S_0^T
//   dv   a = k,     b = q,     v = d_out, seed dS_T,   last token first
//   dk   a = v,     b = d_out, v = q,     seed dS_T^T, last token first
// The reversed walks read their state before its decay (dv_j = k_j R with R
// the gradient of S_j), so their exponents are one lower where the state is
// read and one higher where a token enters it; the state that the dv walk
// ends with is the gradient of S_0.
#pragma once

#include "common.cuh"

namespace la {

// A (batch, heads, tokens, width) tensor with a dense last dimension; strides
// in elements.
struct DecayView {
  const void *p = nullptr;
  int64_t sb = 0, sh = 0, st = 0;
};

struct DecayRole {
  DecayView a, b, v;
  DecayView out;                 // written; unused by a state pass
  const float *init = nullptr;   // null, or the state the walk starts with, per head
  // What each segment of a split head adds to the state, in the walk's order,
  // the last one's left out: states[(bh - whole) * segments + o].  Written by a state pass, read by the
  // output pass, whose segment o starts with
  //   lambda^(tokens before o) init + sum_{i<o} lambda^(tokens between i and o) states_i.
  float *states = nullptr;
  float *final_state = nullptr;  // null, or (bh, da, dvo)
  int da = 0, dvo = 0;           // widths of a and b, and of v and out
  int transposed = 0;            // init and states are (dvo, da), else (da, dvo)
  int reverse = 0;
  // factors of the tile's own part of out, of the state's part, and of what
  // enters the state
  float intra = 1.f, inter = 1.f, inc = 1.f;
};

constexpr int kDecayMaxRoles = 3;
constexpr int kDecayMaxWidth = 128;
constexpr int kDecayTile = 128;   // segment boundaries are multiples of this
constexpr int kDecaySlice = 64;   // columns of v and out that one CTA takes

struct DecayCall {
  DecayRole role[kDecayMaxRoles];
  int roles = 0;
  const float *log_decay = nullptr;
  int64_t batch = 0, heads = 0, n = 0;
  // heads [0, whole) of batch x heads are walked by one CTA each, the others in
  // `segments` segments of seg_len tokens
  int64_t whole = 0;
  int64_t seg_len = 0;
  int segments = 1;
  // Tensor-core kernel: with `lead` > 0 every head is walked in two parts (segments
  // = 2) without a state pass or a workspace: the outputs of the walk's first `lead`
  // tiles by one CTA, those of the others by a second one that walks the first
  // tiles for the state alone.
  int lead = 0;
  int dtype = 0;
};

// lambda^n for lambda = e^g, n >= 0: 1 at n = 0 whatever g is; the rounding of
// n * g is put back to first order, so the relative error stays a few ulp
// while n * g grows.
__device__ __forceinline__ float decay_pow(float g, int n) {
  if (n <= 0) return 1.f;
  const float x = (float)n * g;
  if (x < -104.f) return 0.f;  // below the smallest fp32 value
  const float lost = fmaf((float)n, g, -x);
  return expf(x) * (1.f + lost);
}

// Tokens of the walk's segment o (the ragged one comes last, or first in a
// reversed walk).
__host__ __device__ __forceinline__ int segment_tokens(int o, bool reverse, int segments,
                                                       int64_t seg_len, int64_t n) {
  const int64_t at = (int64_t)(reverse ? segments - 1 - o : o) * seg_len;
  return (int)min64(seg_len, n - at);
}

// States of every (split head, segment but the walk's last) of each role into
// role.states.  The CUDA-core kernels take no whole heads beside split ones.
int launch_decay_state_simt(const DecayCall &c, cudaStream_t s);
// Outputs (and final states) of every role.
int launch_decay_output_simt(const DecayCall &c, cudaStream_t s);

// The same on tensor cores: bf16, every tensor of the call as decay_tc_view
// wants it (16-byte rows), n > 0.
bool decay_tc_view(const DecayView &x, int width, const DecayCall &c);
int launch_decay_state_tc(const DecayCall &c, cudaStream_t s);
int launch_decay_output_tc(const DecayCall &c, cudaStream_t s);

}  // namespace la
