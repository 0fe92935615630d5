// Single tokens of the gated linear recurrence and of the short convolution:
// one token of every sequence, the states updated in place.
//
// Latency for a few sequences, memory for many (recurrence in bf16 with both
// gates: 16 bytes per channel): a thread takes 4 neighbouring channels where
// they are aligned, else one, with all its loads ahead of their use.  1 x 1024 in 1.9
// us, 256 x 4096 in 5.1 (its state stays in L2 between calls).
#include "recurrent_step.cuh"

namespace la {
namespace {

constexpr int kThreads = 128;

template <typename T, int kVec>
__device__ __forceinline__ void load(float (&x)[kVec], const T *p) {
  if constexpr (kVec == 4 && sizeof(T) == 4) {
    const float4 v = *(const float4 *)p;
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else if constexpr (kVec == 4) {
    const uint2 v = *(const uint2 *)p;
    x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xFFFF0000u);
    x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xFFFF0000u);
  } else {
    x[0] = to_f32(*p);
  }
}
template <typename T, int kVec>
__device__ __forceinline__ void store(T *p, const float (&x)[kVec]) {
  if constexpr (kVec == 4 && sizeof(T) == 4) {
    *(float4 *)p = make_float4(x[0], x[1], x[2], x[3]);
  } else if constexpr (kVec == 4) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
    *(uint2 *)p = make_uint2(*(const uint32_t *)&a, *(const uint32_t *)&b);
  } else {
    *p = from_f32<T>(x[0]);
  }
}

template <typename T, int kVec, bool kDecay, bool kInput>
__global__ void __launch_bounds__(kThreads) recur_step_kernel(const RecurStep p) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int packs = p.channels / kVec;
  const int64_t ib = i / packs;
  if (ib >= p.batch) return;
  const int c = (int)(i % packs) * kVec;
  float x[kVec], g[kVec], u[kVec] = {}, h[kVec], lambda[kVec] = {};
  load<T, kVec>(x, (const T *)p.x + ib * p.x_sb + c);
  load<T, kVec>(g, (const T *)p.gate + ib * p.gate_sb + c);
  if (kInput) load<T, kVec>(u, (const T *)p.input_gate + ib * p.input_sb + c);
  float *state = p.state + ib * p.state_sb + c;
  load<float, kVec>(h, state);
  if (kDecay) load<float, kVec>(lambda, p.log_decay + c);
#pragma unroll
  for (int e = 0; e < kVec; e += 2) {
    const int f = e + 1 < kVec ? e + 1 : e;
    const Token y = token_of<T, kDecay, kInput, false, false>(
        make_float2(g[e], g[f]), make_float2(u[e], u[f]), make_float2(lambda[e], lambda[f]));
    const float2 old = make_float2(h[e], h[f]);
    const float2 now = __ffma2_rn(y.bu, make_float2(x[e], x[f]), __ffma2_rn(y.am1, old, old));
    h[e] = now.x;
    if (f != e) h[f] = now.y;
  }
  store<float, kVec>(state, h);
  store<T, kVec>((T *)p.out + ib * p.channels + c, h);
}

template <typename T, int kVec, int kTaps>
__global__ void __launch_bounds__(kThreads) conv_step_kernel(const ConvStep p) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int packs = p.channels / kVec;
  const int64_t ib = i / packs;
  if (ib >= p.batch) return;
  const int c = (int)(i % packs) * kVec;
  float x[kTaps][kVec], z[kVec];
  T *state = (T *)p.state + ib * p.state_sb + c;
#pragma unroll
  for (int j = 0; j < kTaps - 1; ++j) load<T, kVec>(x[j], state + (int64_t)j * p.channels);
  load<T, kVec>(x[kTaps - 1], (const T *)p.x + ib * p.x_sb + c);
  auto affine = [&](auto *weight, auto *bias) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      z[e] = bias ? to_f32(bias[c + e]) : 0.f;
#pragma unroll
      for (int j = 0; j < kTaps; ++j)
        z[e] = fmaf(to_f32(weight[(int64_t)(c + e) * kTaps + j]), x[j][e], z[e]);
    }
  };
  if (p.weight_dtype == LA_DTYPE_FLOAT32)
    affine((const float *)p.weight, (const float *)p.bias);
  else
    affine((const __nv_bfloat16 *)p.weight, (const __nv_bfloat16 *)p.bias);
  if (p.silu) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) z[e] *= sigmoid_two<T>(two(z[e])).x;  // (as the prompts' kernel)
  }
  store<T, kVec>((T *)p.out + ib * p.channels + c, z);
#pragma unroll
  for (int j = 0; j < kTaps - 1; ++j) store<T, kVec>(state + (int64_t)j * p.channels, x[j + 1]);
}

template <class F>
int by_grid(int64_t batch, int channels, int vec, F &&launch) {
  const int64_t grid = (batch * (channels / vec) + kThreads - 1) / kThreads;
  if (grid > INT32_MAX) return LA_ERR_UNSUPPORTED;
  launch((unsigned)grid);
  return check_launch();
}

template <typename T, int kVec>
int launch_recur(const RecurStep &p, cudaStream_t s) {
  return by_grid(p.batch, p.channels, kVec, [&](unsigned grid) {
    if (p.log_decay && p.input_gate)
      recur_step_kernel<T, kVec, true, true><<<grid, kThreads, 0, s>>>(p);
    else if (p.log_decay)
      recur_step_kernel<T, kVec, true, false><<<grid, kThreads, 0, s>>>(p);
    else if (p.input_gate)
      recur_step_kernel<T, kVec, false, true><<<grid, kThreads, 0, s>>>(p);
    else
      recur_step_kernel<T, kVec, false, false><<<grid, kThreads, 0, s>>>(p);
  });
}

template <typename T, int kVec>
int launch_conv(const ConvStep &p, cudaStream_t s) {
  return by_grid(p.batch, p.channels, kVec, [&](unsigned grid) {
    if (p.taps == 2) conv_step_kernel<T, kVec, 2><<<grid, kThreads, 0, s>>>(p);
    else if (p.taps == 3) conv_step_kernel<T, kVec, 3><<<grid, kThreads, 0, s>>>(p);
    else conv_step_kernel<T, kVec, 4><<<grid, kThreads, 0, s>>>(p);
  });
}

// Whether packs of 4 elements of `size` bytes start at their own size.
bool aligned(const void *p, int64_t stride, int size) {
  return ((uintptr_t)p % (4 * size)) == 0 && stride % 4 == 0;
}

}  // namespace

int launch_recur_step(const RecurStep &p, int dtype, cudaStream_t s) {
  const int size = dtype == LA_DTYPE_FLOAT32 ? 4 : 2;
  const bool vec = p.channels % 4 == 0 && aligned(p.x, p.x_sb, size) &&
                   aligned(p.gate, p.gate_sb, size) && aligned(p.input_gate, p.input_sb, size) &&
                   aligned(p.state, p.state_sb, 4) && aligned(p.log_decay, 0, 4) &&
                   aligned(p.out, 0, size);
  if (dtype == LA_DTYPE_FLOAT32) return vec ? launch_recur<float, 4>(p, s) : launch_recur<float, 1>(p, s);
  return vec ? launch_recur<__nv_bfloat16, 4>(p, s) : launch_recur<__nv_bfloat16, 1>(p, s);
}

int launch_conv_step(const ConvStep &p, int dtype, cudaStream_t s) {
  const int size = dtype == LA_DTYPE_FLOAT32 ? 4 : 2;
  const bool vec = p.channels % 4 == 0 && aligned(p.x, p.x_sb, size) &&
                   aligned(p.state, p.state_sb, size) && aligned(p.out, 0, size);
  if (dtype == LA_DTYPE_FLOAT32) return vec ? launch_conv<float, 4>(p, s) : launch_conv<float, 1>(p, s);
  return vec ? launch_conv<__nv_bfloat16, 4>(p, s) : launch_conv<__nv_bfloat16, 1>(p, s);
}

}  // namespace la
