// C entry points of the gated linear recurrence, the short convolution and the
// group norm: the checks of their arguments.
#include <initializer_list>

#include "column_sum.cuh"
#include "group_norm.cuh"
#include "recurrent_step.cuh"
#include "short_conv.cuh"

namespace la {
namespace {

bool valid_type(int t) { return t == LA_DTYPE_FLOAT32 || t == LA_DTYPE_BFLOAT16; }

// Whether all of them start at an element's size.
bool placed(int size, std::initializer_list<const void *> pointers) {
  uintptr_t bits = 0;
  for (const void *p : pointers) bits |= (uintptr_t)p;
  return bits % size == 0;
}
int size_of(int dtype) { return dtype == LA_DTYPE_FLOAT32 ? 4 : 2; }

// Sizes whose elements, and the bytes of a few tensors of them, fit 63 bits.
bool fits(int64_t batch, int64_t tokens, int64_t channels) {
  constexpr int64_t kMost = INT64_MAX / 64;
  if (batch && tokens > kMost / batch) return false;
  return !(batch * tokens) || channels <= kMost / (batch * tokens);
}

int check_device(DeviceInfo *info) {
  const int st = current_device_info(info);
  if (st != LA_OK) return st;
  return info->cc_major == 10 ? LA_OK : LA_ERR_NO_DEVICE;
}

TokenView tokens_of(const void *p, const int64_t *s) {
  TokenView v;
  v.p = p;
  if (p) v.sb = s[0], v.st = s[1];
  return v;
}

bool valid_strides(const int64_t *s) { return s && s[0] >= 0 && s[1] >= 0; }

// Whether pairs of channels can be written together.
bool in_pairs(int64_t channels, std::initializer_list<const void *> written) {
  uintptr_t bits = 0;
  for (const void *p : written) bits |= (uintptr_t)p;
  return channels % 2 == 0 && bits % 8 == 0;
}

int64_t check_rows(int64_t tokens) { return (tokens + kRecurCheck - 1) / kRecurCheck; }

int check_sizes(int64_t batch, int64_t tokens, int64_t channels, int dtype) {
  if (batch < 0 || tokens < 0 || channels < 1 || !valid_type(dtype)) return LA_ERR_INVALID_ARGUMENT;
  if (channels > INT32_MAX / 8 || tokens > INT32_MAX / 2 || !fits(batch, tokens, channels)) return LA_ERR_UNSUPPORTED;
  return LA_OK;
}

int check_lengths(const void *lengths, int bits) {
  if (!lengths) return LA_OK;
  return (bits == 32 || bits == 64) && placed(bits / 8, {lengths}) ? LA_OK : LA_ERR_INVALID_ARGUMENT;
}

int zero(void *p, int64_t bytes, cudaStream_t s) {
  return p && bytes ? cuda_status(cudaMemsetAsync(p, 0, (size_t)bytes, s)) : LA_OK;
}
int copy_or_zero(void *dst, const void *src, int64_t bytes, cudaStream_t s) {
  if (!dst || !bytes) return LA_OK;
  return src ? cuda_status(cudaMemcpyAsync(dst, src, (size_t)bytes, cudaMemcpyDeviceToDevice, s))
             : zero(dst, bytes, s);
}

}  // namespace
}  // namespace la

using namespace la;

extern "C" {

int la_recurrence_plan(int64_t batch, int64_t tokens, int64_t channels, size_t *saved_bytes,
                       size_t *workspace_bytes) {
  int st = check_sizes(batch, tokens, channels, LA_DTYPE_FLOAT32);
  if (st != LA_OK) return st;
  if (!saved_bytes || !workspace_bytes) return LA_ERR_INVALID_ARGUMENT;
  *saved_bytes = (size_t)(batch * check_rows(tokens) * channels) * sizeof(float);
  *workspace_bytes = 0;
  if (!batch || !tokens) return LA_OK;
  DeviceInfo info;
  if ((st = check_device(&info)) != LA_OK) return st;
  *workspace_bytes =
      (size_t)(batch * recur_bwd_rows({batch, tokens, (int)channels}, info.sm_count) * channels) *
      sizeof(float);
  return LA_OK;
}

int la_recurrence_fwd(const void *x, const int64_t *x_strides, const void *gate,
                      const int64_t *gate_strides, const void *input_gate,
                      const int64_t *input_strides, const float *log_decay, const float *init_state,
                      const void *lengths, int lengths_bits, void *out, float *final_state,
                      float *saved, int64_t batch, int64_t tokens, int64_t channels, int dtype,
                      void *stream) {
  int st = check_sizes(batch, tokens, channels, dtype);
  if (st != LA_OK || (st = check_lengths(lengths, lengths_bits)) != LA_OK) return st;
  if (!batch) return LA_OK;
  cudaStream_t s = (cudaStream_t)stream;
  if (!tokens) return copy_or_zero(final_state, init_state, batch * channels * 4, s);
  if (!x || !gate || !out || !valid_strides(x_strides) || !valid_strides(gate_strides) ||
      (input_gate && !valid_strides(input_strides)) ||
      !placed(size_of(dtype), {x, gate, input_gate, out}) ||
      !placed(4, {log_decay, init_state, final_state, saved}))
    return LA_ERR_INVALID_ARGUMENT;
  DeviceInfo info;
  if ((st = check_device(&info)) != LA_OK) return st;
  RecurCall c;
  c.x = tokens_of(x, x_strides);
  c.gate = tokens_of(gate, gate_strides);
  c.input_gate = tokens_of(input_gate, input_strides);
  c.log_decay = log_decay, c.init = init_state;
  c.lengths = lengths, c.lengths64 = lengths_bits == 64;
  c.sizes = {batch, tokens, (int)channels};
  c.check = saved, c.out = out, c.final_state = final_state;
  c.pairs = in_pairs(channels, {out, final_state, saved});
  return launch_recur_fwd(c, dtype, s);
}

int la_recurrence_bwd(const void *x, const int64_t *x_strides, const void *gate,
                      const int64_t *gate_strides, const void *input_gate,
                      const int64_t *input_strides, const float *log_decay, const float *saved,
                      const void *lengths, int lengths_bits, const void *d_out,
                      const int64_t *d_out_strides, const float *d_final_state, void *dx,
                      void *d_gate, void *d_input_gate, float *d_log_decay, float *d_init_state,
                      int64_t batch, int64_t tokens, int64_t channels, int dtype, void *workspace,
                      size_t workspace_bytes, void *stream) {
  int st = check_sizes(batch, tokens, channels, dtype);
  if (st != LA_OK || (st = check_lengths(lengths, lengths_bits)) != LA_OK) return st;
  if (d_log_decay && !log_decay) return LA_ERR_INVALID_ARGUMENT;
  cudaStream_t s = (cudaStream_t)stream;
  if (!batch || !tokens) {
    if ((st = zero(d_log_decay, channels * 4, s)) != LA_OK) return st;
    return copy_or_zero(d_init_state, d_final_state, batch * channels * 4, s);
  }
  if (!x || !gate || !saved || !d_out || !dx || !d_gate || !valid_strides(x_strides) ||
      !valid_strides(gate_strides) || !valid_strides(d_out_strides) ||
      (input_gate && (!valid_strides(input_strides) || !d_input_gate)) ||
      !placed(size_of(dtype), {x, gate, input_gate, d_out, dx, d_gate, d_input_gate}) ||
      !placed(4, {log_decay, saved, d_final_state, d_log_decay, d_init_state}))
    return LA_ERR_INVALID_ARGUMENT;
  DeviceInfo info;
  if ((st = check_device(&info)) != LA_OK) return st;
  const int64_t rows = batch * recur_bwd_rows({batch, tokens, (int)channels}, info.sm_count);
  if (d_log_decay && (!workspace || ((uintptr_t)workspace & 15) ||
                      workspace_bytes < (size_t)(rows * channels) * sizeof(float)))
    return LA_ERR_WORKSPACE;
  RecurCall c;
  c.x = tokens_of(x, x_strides);
  c.gate = tokens_of(gate, gate_strides);
  c.input_gate = tokens_of(input_gate, input_strides);
  c.d_out = tokens_of(d_out, d_out_strides);
  c.log_decay = log_decay, c.check = const_cast<float *>(saved);
  c.lengths = lengths, c.lengths64 = lengths_bits == 64;
  c.sizes = {batch, tokens, (int)channels};
  c.d_final = d_final_state, c.dx = dx, c.d_gate = d_gate, c.d_input = d_input_gate;
  c.d_init = d_init_state, c.partial = d_log_decay ? (float *)workspace : nullptr;
  c.pairs = in_pairs(channels, {dx, d_gate, d_input_gate, d_init_state});
  st = launch_recur_bwd(c, dtype, s);
  if (st != LA_OK || !d_log_decay) return st;
  return launch_column_sum(c.partial, rows, channels, d_log_decay, channels, nullptr,
                           LA_DTYPE_FLOAT32, s);
}

int la_recurrence_step(const void *x, int64_t x_stride, const void *gate, int64_t gate_stride,
                       const void *input_gate, int64_t input_stride, const float *log_decay,
                       float *state, int64_t state_stride, void *out, int64_t batch,
                       int64_t channels, int dtype, void *stream) {
  int st = check_sizes(batch, 1, channels, dtype);
  if (st != LA_OK) return st;
  if (!batch) return LA_OK;
  if (!x || !gate || !state || !out || x_stride < 0 || gate_stride < 0 || input_stride < 0 ||
      (batch > 1 && state_stride < channels) ||
      !placed(size_of(dtype), {x, gate, input_gate, out}) || !placed(4, {log_decay, state}))
    return LA_ERR_INVALID_ARGUMENT;
  DeviceInfo info;
  if ((st = check_device(&info)) != LA_OK) return st;
  const RecurStep p{x, gate, input_gate, x_stride, gate_stride, input_stride, log_decay, state,
                    state_stride, out, batch, (int)channels};
  return launch_recur_step(p, dtype, (cudaStream_t)stream);
}

int la_short_conv_workspace_size(int64_t batch, int64_t tokens, int64_t channels, int64_t taps,
                                 size_t *bytes) {
  const int st = check_sizes(batch, tokens, channels, LA_DTYPE_FLOAT32);
  if (st != LA_OK) return st;
  if (!bytes) return LA_ERR_INVALID_ARGUMENT;
  if (taps < kConvMinTaps || taps > kConvMaxTaps) return LA_ERR_UNSUPPORTED;
  *bytes = (size_t)(conv_partial_rows({batch, tokens, (int)channels}) * channels * (taps + 1)) * sizeof(float);
  return LA_OK;
}

static int conv_call(ConvCall *c, const void *x, const int64_t *x_strides, const void *weight,
                     const void *bias, int weight_dtype, const void *init_state,
                     const void *lengths, int lengths_bits, int64_t batch, int64_t tokens,
                     int64_t channels, int64_t taps, int silu, int dtype) {
  int st = check_sizes(batch, tokens, channels, dtype);
  if (st != LA_OK || (st = check_lengths(lengths, lengths_bits)) != LA_OK) return st;
  if (!valid_type(weight_dtype)) return LA_ERR_INVALID_ARGUMENT;
  if (taps < kConvMinTaps || taps > kConvMaxTaps) return LA_ERR_UNSUPPORTED;
  if (!batch) return LA_OK;
  if ((tokens && (!x || !valid_strides(x_strides))) || !weight ||
      !placed(size_of(dtype), {x, init_state}) || !placed(size_of(weight_dtype), {weight, bias}))
    return LA_ERR_INVALID_ARGUMENT;
  c->x = tokens_of(tokens ? x : nullptr, x_strides);
  c->weight = weight, c->bias = bias, c->weight_dtype = weight_dtype, c->init = init_state;
  c->lengths = lengths, c->lengths64 = lengths_bits == 64;
  c->sizes = {batch, tokens, (int)channels}, c->taps = (int)taps;
  c->silu = silu != 0;
  DeviceInfo info;
  return check_device(&info);
}

int la_short_conv_fwd(const void *x, const int64_t *x_strides, const void *weight,
                      const void *bias, int weight_dtype, const void *init_state,
                      const void *lengths, int lengths_bits, void *out, void *final_state,
                      int64_t batch, int64_t tokens, int64_t channels, int64_t taps, int silu,
                      int dtype, void *stream) {
  ConvCall c;
  const int st = conv_call(&c, x, x_strides, weight, bias, weight_dtype, init_state, lengths,
                           lengths_bits, batch, tokens, channels, taps, silu, dtype);
  if (st != LA_OK || !batch || (!tokens && !final_state)) return st;
  if ((tokens && !out) || !placed(size_of(dtype), {out, final_state})) return LA_ERR_INVALID_ARGUMENT;
  c.out = out, c.final_state = final_state;
  return launch_conv_fwd(c, dtype, (cudaStream_t)stream);
}

int la_short_conv_bwd(const void *x, const int64_t *x_strides, const void *weight,
                      const void *bias, int weight_dtype, const void *init_state,
                      const void *lengths, int lengths_bits, const void *d_out,
                      const int64_t *d_out_strides, const void *d_final_state, void *dx,
                      void *d_weight, void *d_bias, void *d_init_state, int64_t batch,
                      int64_t tokens, int64_t channels, int64_t taps, int silu, int dtype,
                      void *workspace, size_t workspace_bytes, void *stream) {
  ConvCall c;
  int st = conv_call(&c, x, x_strides, weight, bias, weight_dtype, init_state, lengths,
                     lengths_bits, batch, tokens, channels, taps, silu, dtype);
  if (st != LA_OK) return st;
  cudaStream_t s = (cudaStream_t)stream;
  if (!batch) {
    const int64_t size = size_of(weight_dtype);
    if ((st = zero(d_weight, channels * taps * size, s)) != LA_OK) return st;
    return zero(d_bias, channels * size, s);
  }
  if ((tokens && (!d_out || !valid_strides(d_out_strides) || !dx)) ||
      !placed(size_of(dtype), {d_out, d_final_state, dx, d_init_state}) ||
      !placed(size_of(weight_dtype), {d_weight, d_bias}))
    return LA_ERR_INVALID_ARGUMENT;
  const int64_t rows = conv_partial_rows({batch, tokens, (int)channels});
  const bool sums = d_weight || d_bias;
  if (sums && (!workspace || ((uintptr_t)workspace & 15) ||
               workspace_bytes < (size_t)(rows * channels * (taps + 1)) * sizeof(float)))
    return LA_ERR_WORKSPACE;
  c.d_out = tokens_of(tokens ? d_out : nullptr, d_out_strides);
  c.d_final = d_final_state, c.dx = dx, c.d_init = d_init_state;
  c.partial = sums ? (float *)workspace : nullptr;
  st = launch_conv_bwd(c, dtype, s);
  if (st != LA_OK || !sums) return st;
  return launch_column_sum(c.partial, rows, channels * (taps + 1), d_weight, channels * taps, d_bias,
                           weight_dtype, s);
}

int la_short_conv_step(const void *x, int64_t x_stride, const void *weight, const void *bias,
                       int weight_dtype, void *state, int64_t state_stride, void *out,
                       int64_t batch, int64_t channels, int64_t taps, int silu, int dtype,
                       void *stream) {
  int st = check_sizes(batch, 1, channels, dtype);
  if (st != LA_OK) return st;
  if (!valid_type(weight_dtype)) return LA_ERR_INVALID_ARGUMENT;
  if (taps < kConvMinTaps || taps > kConvMaxTaps) return LA_ERR_UNSUPPORTED;
  if (!batch) return LA_OK;
  if (!x || !weight || !state || !out || x_stride < 0 ||
      (batch > 1 && state_stride < (taps - 1) * channels) ||
      !placed(size_of(dtype), {x, state, out}) || !placed(size_of(weight_dtype), {weight, bias}))
    return LA_ERR_INVALID_ARGUMENT;
  DeviceInfo info;
  if ((st = check_device(&info)) != LA_OK) return st;
  const ConvStep p{x, x_stride, weight, bias, weight_dtype, state, state_stride, out, batch,
                   (int)channels, (int)taps, silu != 0};
  return launch_conv_step(p, dtype, (cudaStream_t)stream);
}

static int norm_call(GroupNormCall *c, const void *x, const int64_t *x_strides, const void *gate,
                     const int64_t *gate_strides, const void *weight, const void *bias,
                     int weight_dtype, const int64_t *shape, int64_t channels, int64_t groups,
                     int silu, int dtype) {
  if (!shape || shape[0] < 0 || shape[1] < 0 || channels < 1 || groups < 1 || channels % groups ||
      !valid_type(dtype) || !valid_type(weight_dtype))
    return LA_ERR_INVALID_ARGUMENT;
  if (channels / groups > kGroupMaxSize || channels > INT32_MAX / 8 || shape[1] > INT32_MAX ||
      !fits(shape[0], shape[1], channels))
    return LA_ERR_UNSUPPORTED;
  c->rows = shape[0] * shape[1];
  if (!c->rows) return LA_OK;
  if (c->rows > INT32_MAX / 2) return LA_ERR_UNSUPPORTED;
  if (!x || !valid_strides(x_strides) || (gate && !valid_strides(gate_strides)) ||
      !placed(size_of(dtype), {x, gate}) || !placed(size_of(weight_dtype), {weight, bias}))
    return LA_ERR_INVALID_ARGUMENT;
  c->n1 = (uint32_t)shape[1];
  c->x.p = x, c->x.s0 = x_strides[0], c->x.s1 = x_strides[1];
  c->gate.p = gate;
  if (gate) c->gate.s0 = gate_strides[0], c->gate.s1 = gate_strides[1];
  c->weight = weight, c->bias = bias, c->weight_dtype = weight_dtype;
  c->groups = (int)groups, c->size = (int)(channels / groups), c->silu = silu != 0;
  return LA_OK;
}

int la_group_norm_fwd(const void *x, const int64_t *x_strides, const void *gate,
                      const int64_t *gate_strides, const void *weight, const void *bias,
                      int weight_dtype, void *out, float *stats, const int64_t *shape,
                      int64_t channels, int64_t groups, int silu, int dtype, float eps,
                      void *stream) {
  GroupNormCall c;
  int st = norm_call(&c, x, x_strides, gate, gate_strides, weight, bias, weight_dtype, shape,
                     channels, groups, silu, dtype);
  if (st != LA_OK || !c.rows) return st;
  if (!out || !placed(size_of(dtype), {out}) || !placed(8, {stats})) return LA_ERR_INVALID_ARGUMENT;
  DeviceInfo info;
  if ((st = check_device(&info)) != LA_OK) return st;
  c.out = out, c.stats = stats, c.eps = eps;
  return launch_group_norm_fwd(c, dtype, (cudaStream_t)stream);
}

int la_group_norm_bwd_workspace_size(int64_t rows, int64_t channels, size_t *bytes) {
  if (!bytes || rows < 0 || channels < 1) return LA_ERR_INVALID_ARGUMENT;
  if (channels > INT32_MAX / 8) return LA_ERR_UNSUPPORTED;
  *bytes = 0;
  if (!rows) return LA_OK;
  DeviceInfo info;
  const int st = check_device(&info);
  if (st != LA_OK) return st;
  *bytes = (size_t)(group_norm_partial_rows(rows, info.sm_count) * 2 * channels) * sizeof(float);
  return LA_OK;
}

int la_group_norm_bwd(const void *x, const int64_t *x_strides, const void *gate,
                      const int64_t *gate_strides, const void *weight, const void *bias,
                      int weight_dtype, const float *stats, const void *d_out,
                      const int64_t *d_out_strides, void *dx, void *d_gate, void *d_weight,
                      void *d_bias, const int64_t *shape, int64_t channels, int64_t groups,
                      int silu, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
  GroupNormCall c;
  int st = norm_call(&c, x, x_strides, gate, gate_strides, weight, bias, weight_dtype, shape,
                     channels, groups, silu, dtype);
  if (st != LA_OK) return st;
  cudaStream_t s = (cudaStream_t)stream;
  if (!c.rows) {
    const int64_t bytes = channels * size_of(weight_dtype);
    if ((st = zero(d_weight, bytes, s)) != LA_OK) return st;
    return zero(d_bias, bytes, s);
  }
  if (!stats || !d_out || !valid_strides(d_out_strides) || !dx || (gate && !d_gate) ||
      !placed(8, {stats}) || !placed(size_of(dtype), {d_out, dx, d_gate}) ||
      !placed(size_of(weight_dtype), {d_weight, d_bias}))
    return LA_ERR_INVALID_ARGUMENT;
  DeviceInfo info;
  if ((st = check_device(&info)) != LA_OK) return st;
  const bool sums = d_weight || d_bias;
  if (sums && (!workspace || ((uintptr_t)workspace & 15) ||
               workspace_bytes <
                   (size_t)(group_norm_partial_rows(c.rows, info.sm_count) * 2 * channels) * 4))
    return LA_ERR_WORKSPACE;
  c.d_out.p = d_out, c.d_out.s0 = d_out_strides[0], c.d_out.s1 = d_out_strides[1];
  c.stats = const_cast<float *>(stats), c.dx = dx, c.d_gate = d_gate;
  c.partial = sums ? (float *)workspace : nullptr;
  int64_t rows = 0;
  st = launch_group_norm_bwd(c, dtype, info.sm_count, &rows, s);
  if (st != LA_OK || !sums) return st;
  return launch_column_sum(c.partial, rows, 2 * channels, d_weight, channels, d_bias, weight_dtype,
                           s);
}

}  // extern "C"
