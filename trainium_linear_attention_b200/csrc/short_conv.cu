// Causal convolution of each channel with 2 to 4 taps, an activation, and its
// gradient.
//
//   z_t = bias + sum_j w_j x_{t - taps + 1 + j},   y = z, or z sigmoid(z)
//   dz = dy, or dy sigmoid(z) (1 + z (1 - sigmoid(z)))
//   dx_t = sum_j w_j dz_{t + taps - 1 - j},  dw_j = sum_t dz_t x_{t - taps + 1 + j}
//
// Bound by memory: x read and y written once (4 bytes per element in bf16),
// the gradient also reads dy (6).  A lane has one or two pairs of neighbouring
// channels and walks a run of tokens with the taps' window in registers, a batch of
// tokens ahead on its way; the tokens before a run are read twice, the second
// time from the caches.  The gradient computes z again instead of keeping it.
// Its walk meets dz_t once and adds it to the taps' sums that are still open, so
// that dx, dw and the bias' gradient come from one pass; the sums over tokens are
// joined over the CTA's warps in shared memory, written as one row per CTA, and
// the rows added by a second kernel in a fixed order.
#include "column_sum.cuh"
#include "short_conv.cuh"

namespace la {
namespace {

#ifndef CONV_F
#define CONV_F 4
#endif
#ifndef CONV_B
#define CONV_B 3
#endif
#ifndef CONV_FR
#define CONV_FR 32
#endif
#ifndef CONV_BR
#define CONV_BR 32
#endif
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kBatch = 8;    // tokens whose loads are on their way together
constexpr int kRest = 4;     // the same where a sequence or a run ends
constexpr int kFwdRun = CONV_FR;  // tokens of a lane, at most
constexpr int kBwdRun = CONV_BR;

// NP pairs of neighbouring channels as they lie in memory.
template <typename T, int NP>
struct Pack {
  static constexpr int kWords = NP * (int)sizeof(T) / 2;
  uint32_t w[kWords];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  // `wide`: the pack starts at its own size (NP = 1: else by elements, of which the
  // last may be beyond the row).
  __device__ __forceinline__ void load(const T *p, bool wide, bool second) {
    if (NP > 1 || wide) {
      if constexpr (kWords == 4) {
        const uint4 v = *(const uint4 *)p;
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
      } else if constexpr (kWords == 2) {
        const uint2 v = *(const uint2 *)p;
        w[0] = v.x, w[1] = v.y;
      } else {
        w[0] = *(const uint32_t *)p;
      }
    } else if constexpr (sizeof(T) == 2) {
      const uint16_t *q = (const uint16_t *)p;
      w[0] = q[0] | (second ? (uint32_t)q[1] << 16 : 0);
    } else {
      w[0] = ((const uint32_t *)p)[0];
      w[1] = second ? ((const uint32_t *)p)[1] : 0;
    }
  }
  __device__ __forceinline__ void store(T *p, bool wide, bool second) const {
    if (NP > 1 || wide) {
      if constexpr (kWords == 4) *(uint4 *)p = make_uint4(w[0], w[1], w[2], w[3]);
      else if constexpr (kWords == 2) *(uint2 *)p = make_uint2(w[0], w[1]);
      else *(uint32_t *)p = w[0];
    } else if constexpr (sizeof(T) == 2) {
      uint16_t *q = (uint16_t *)p;
      q[0] = (uint16_t)w[0];
      if (second) q[1] = (uint16_t)(w[0] >> 16);
    } else {
      ((uint32_t *)p)[0] = w[0];
      if (second) ((uint32_t *)p)[1] = w[1];
    }
  }
  __device__ __forceinline__ float2 get(int i) const {
    if constexpr (sizeof(T) == 4)
      return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    else
      return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
  }
  __device__ __forceinline__ void set(int i, float2 v) {
    if constexpr (sizeof(T) == 4) {
      w[2 * i] = __float_as_uint(v.x), w[2 * i + 1] = __float_as_uint(v.y);
    } else {
      const __nv_bfloat162 b = __floats2bfloat162_rn(v.x, v.y);
      w[i] = *(const uint32_t *)&b;
    }
  }
};

// A sequence's rows at a lane's channels, with the tokens before it.
template <typename T, int NP, int kTaps>
struct Row {
  const T *x;
  const T *init;   // null, or the kTaps - 1 rows before
  int64_t st;
  int channels, len;
  bool wide, second;
  __device__ __forceinline__ void load(Pack<T, NP> &v, int t) const {
    v.zero();
    if (t >= 0) {
      if (t < len) v.load(x + t * st, wide, second);
    } else if (init && t >= -(kTaps - 1)) {
      v.load(init + (int64_t)(t + kTaps - 1) * channels, wide, second);
    }
  }
  __device__ __forceinline__ void load_inside(Pack<T, NP> &v, int t) const {
    v.load(x + t * st, wide, second);
  }
};

template <int NP, int kTaps>
struct Weights {
  float2 w[kTaps][NP], b[NP];
  template <typename TW>
  __device__ __forceinline__ void load_as(const ConvCall &p, int c) {
    const TW *src = (const TW *)p.weight + (int64_t)c * kTaps;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const bool second = c + 2 * i + 1 < p.channels;
      if (sizeof(TW) == 2 && second && ((uintptr_t)src & 3) == 0) {  // a pair's in words
        const uint32_t *words = (const uint32_t *)src + i * kTaps;
        float v[2 * kTaps];
#pragma unroll
        for (int j = 0; j < kTaps; ++j) {
          const uint32_t u = words[j];
          v[2 * j] = __uint_as_float(u << 16), v[2 * j + 1] = __uint_as_float(u & 0xFFFF0000u);
        }
#pragma unroll
        for (int j = 0; j < kTaps; ++j) w[j][i] = make_float2(v[j], v[kTaps + j]);
      } else {
#pragma unroll
        for (int j = 0; j < kTaps; ++j)
          w[j][i] = make_float2(to_f32(src[2 * i * kTaps + j]),
                                second ? to_f32(src[(2 * i + 1) * kTaps + j]) : 0.f);
      }
      b[i] = two(0.f);
      if (p.bias) {
        const TW *bias = (const TW *)p.bias + c + 2 * i;
        b[i] = make_float2(to_f32(bias[0]), second ? to_f32(bias[1]) : 0.f);
      }
    }
  }
  __device__ __forceinline__ void load(const ConvCall &p, int c) {
    if (p.weight_dtype == LA_DTYPE_FLOAT32) load_as<float>(p, c);
    else load_as<__nv_bfloat16>(p, c);
  }
};

// A CTA: 32 packs of channels, kWarps runs of tokens.
template <typename T, int NP, int kTaps, bool kSilu>
__global__ void __launch_bounds__(kThreads, CONV_F) conv_fwd_kernel(const ConvCall p, const int run,
                                                          const int columns, const int blocks) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = (blockIdx.x % columns * 32 + lane) * 2 * NP;
  const int64_t ib = blockIdx.x / columns / blocks;
  const int t0 = (blockIdx.x / columns % blocks * kWarps + warp) * run;
  if (c >= p.channels || (t0 >= p.tokens && t0 > 0)) return;
  const int len = (int)sequence_length(p.lengths, p.lengths64, ib, p.tokens);
  const int end = min(t0 + run, (int)p.tokens);
  Row<T, NP, kTaps> row;
  row.x = (const T *)p.x.p + ib * p.x.sb + c;
  row.init = p.init ? (const T *)p.init + ib * (kTaps - 1) * p.channels + c : nullptr;
  row.st = p.x.st, row.channels = p.channels, row.len = len;
  row.wide = p.wide, row.second = c + 1 < p.channels;
  if (p.final_state && t0 == 0) {
    T *dst = (T *)p.final_state + ib * (kTaps - 1) * p.channels + c;
#pragma unroll
    for (int j = 0; j < kTaps - 1; ++j) {
      Pack<T, NP> v;
      row.load(v, len - (kTaps - 1) + j);
      v.store(dst + (int64_t)j * p.channels, p.wide, row.second);
    }
  }
  Weights<NP, kTaps> w;
  w.load(p, c);
  float2 x[kTaps][NP];  // the window; the last one is the token's own
#pragma unroll
  for (int j = 0; j < kTaps - 1; ++j) {
    Pack<T, NP> v;
    row.load(v, t0 - (kTaps - 1) + j);
#pragma unroll
    for (int i = 0; i < NP; ++i) x[j + 1][i] = v.get(i);
  }
  T *out = (T *)p.out + ib * p.tokens * p.channels + c;
  auto token = [&](const Pack<T, NP> &in, int t, bool inside) {
    Pack<T, NP> y;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
#pragma unroll
      for (int j = 0; j < kTaps - 1; ++j) x[j][i] = x[j + 1][i];
      x[kTaps - 1][i] = in.get(i);
      float2 z = w.b[i];
#pragma unroll
      for (int j = 0; j < kTaps; ++j) z = __ffma2_rn(w.w[j][i], x[j][i], z);
      if constexpr (kSilu) z = __fmul2_rn(z, sigmoid_two<T>(z));
      y.set(i, z);
    }
    if (!inside) y.zero();
    y.store(out + (int64_t)t * p.channels, p.wide, row.second);
  };
  int t = t0;
  const int whole = min(end, len);
  for (; t + kBatch <= whole; t += kBatch) {
    Pack<T, NP> in[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) row.load_inside(in[i], t + i);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) token(in[i], t + i, true);
  }
  for (; t < end; t += kRest) {
    Pack<T, NP> in[kRest];
#pragma unroll
    for (int i = 0; i < kRest; ++i) row.load(in[i], t + i);
#pragma unroll
    for (int i = 0; i < kRest; ++i)
      if (t + i < end) token(in[i], t + i, t + i < len);
  }
}

// A CTA: 32 pairs of channels, kWarps runs of kBwdRun tokens.
template <typename T, int kTaps, bool kSilu>
__global__ void __launch_bounds__(kThreads, CONV_B) conv_bwd_kernel(const ConvCall p, const int columns,
                                                          const int blocks) {
  constexpr int kSums = kTaps + 1;
  __shared__ float2 part[kWarps][kSums][32];
  column_sum_may_start();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c0 = blockIdx.x % columns * 64, c = c0 + 2 * lane;
  const int sums_row = blockIdx.x / columns;
  const int64_t ib = sums_row / blocks;
  const int t0 = (sums_row % blocks * kWarps + warp) * kBwdRun;
  const bool first = t0 == 0;  // also ends the initial state's rows
  float2 sums[kSums] = {};
  if (c < p.channels && (t0 < p.tokens || first)) {
    const int len = (int)sequence_length(p.lengths, p.lengths64, ib, p.tokens);
    const int end = min(t0 + kBwdRun, (int)p.tokens);
    Row<T, 1, kTaps> row, dy;
    row.x = (const T *)p.x.p + ib * p.x.sb + c;
    row.init = p.init ? (const T *)p.init + ib * (kTaps - 1) * p.channels + c : nullptr;
    row.st = p.x.st, row.channels = p.channels, row.len = len;
    row.wide = p.wide, row.second = c + 1 < p.channels;
    dy = row;
    dy.x = (const T *)p.d_out.p + ib * p.d_out.sb + c;
    dy.st = p.d_out.st, dy.init = nullptr;
    Weights<1, kTaps> w;
    w.load(p, c);
    float2 x[kTaps], open[kTaps] = {};  // the window; dx of its tokens so far
#pragma unroll
    for (int j = 0; j < kTaps - 1; ++j) {
      Pack<T, 1> v;
      row.load(v, t0 - (kTaps - 1) + j);
      x[j + 1] = v.get(0);
    }
    T *dx = (T *)p.dx + ib * p.tokens * p.channels + c;
    // Takes a token's x and dy; open[0] is then the gradient of the window's oldest.
    auto token = [&](const Pack<T, 1> &in, const Pack<T, 1> &up, bool inside, bool own) {
#pragma unroll
      for (int j = 0; j < kTaps - 1; ++j) x[j] = x[j + 1], open[j] = open[j + 1];
      x[kTaps - 1] = in.get(0);
      float2 g = up.get(0);
      if constexpr (kSilu) {
        float2 z = w.b[0];
#pragma unroll
        for (int j = 0; j < kTaps; ++j) z = __ffma2_rn(w.w[j][0], x[j], z);
        const float2 s = sigmoid_two<T>(z);
        // s (1 + z (1 - s)) = s + z s - z s s
        const float2 zs = __fmul2_rn(z, s);
        const float2 slope = __fadd2_rn(s, __ffma2_rn(__fmul2_rn(zs, two(-1.f)), s, zs));
        g = __fmul2_rn(g, slope);
      }
      if (!inside) g = two(0.f);
#pragma unroll
      for (int j = 0; j < kTaps; ++j) {
        open[j] = j == kTaps - 1 ? __fmul2_rn(w.w[j][0], g) : __ffma2_rn(w.w[j][0], g, open[j]);
        if (own) sums[j] = __ffma2_rn(g, x[j], sums[j]);
      }
      if (own) sums[kTaps] = __fadd2_rn(sums[kTaps], g);
    };
    auto finish = [&](int at) {  // stores open[0], of token `at` (< 0: the initial state's)
      const int back = at - (len - (kTaps - 1));  // its row of the final state
      if (p.d_final && back >= 0 && back < kTaps - 1) {
        Pack<T, 1> v;
        v.load((const T *)p.d_final + (ib * (kTaps - 1) + back) * p.channels + c, p.wide, row.second);
        open[0] = __fadd2_rn(open[0], v.get(0));
      }
      Pack<T, 1> v;
      v.set(0, open[0]);
      if (at >= 0)
        v.store(dx + (int64_t)at * p.channels, p.wide, row.second);
      else if (p.d_init)
        v.store((T *)p.d_init + (ib * (kTaps - 1) + at + kTaps - 1) * p.channels + c, p.wide,
                row.second);
    };
    int t = t0;
    // Whole batches whose tokens all are the run's own and whose dx all are plain:
    // not the sequence's first ones, nor those that the final state reaches.
    const int plain = min(end, p.d_final ? len - (kTaps - 1) : len);
    for (; !first && t + kBatch <= plain; t += kBatch) {
      Pack<T, 1> in[kBatch], up[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) row.load_inside(in[i], t + i), dy.load_inside(up[i], t + i);
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        token(in[i], up[i], true, true);
        if (i >= kTaps - 1 || t > t0) {  // (else the run before stores it)
          Pack<T, 1> v;
          v.set(0, open[0]);
          v.store(dx + (int64_t)(t + i - (kTaps - 1)) * p.channels, p.wide, row.second);
        }
      }
    }
    for (; t < end + kTaps - 1; t += kRest) {
      Pack<T, 1> in[kRest], up[kRest];
#pragma unroll
      for (int i = 0; i < kRest; ++i) row.load(in[i], t + i), dy.load(up[i], t + i);
#pragma unroll
      for (int i = 0; i < kRest; ++i) {
        if (t + i >= end + kTaps - 1) break;
        token(in[i], up[i], t + i < len, t + i < min(len, end));
        const int at = t + i - (kTaps - 1);
        if (at >= t0 || first) finish(at);
      }
    }
  }
  if (!p.partial) return;
#pragma unroll
  for (int j = 0; j < kSums; ++j) part[warp][j][lane] = sums[j];
  __syncthreads();
  float *dst = p.partial + (int64_t)sums_row * p.channels * kSums;
  for (int i = threadIdx.x; i < kSums * 64; i += kThreads) {
    const int j = i / 64, channel = c0 + i % 64;
    if (channel >= p.channels) continue;
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) {
      const float2 v = part[k][j][i % 64 / 2];
      sum += i & 1 ? v.y : v.x;
    }
    if (j < kTaps) dst[(int64_t)channel * kTaps + j] = sum;
    else dst[(int64_t)p.channels * kTaps + channel] = sum;
  }
}

template <typename T, int NP, int kTaps>
int launch_fwd(const ConvCall &p, cudaStream_t s) {
  const int columns = (p.channels + 64 * NP - 1) / (64 * NP);
  int run = kFwdRun;  // shorter runs where long ones leave SMs without a CTA
  DeviceInfo info;
  const int st = current_device_info(&info);
  if (st != LA_OK) return st;
  while (run > kBatch && p.batch * columns * ((p.tokens + run * kWarps - 1) / (run * kWarps)) <
                             4 * info.sm_count)
    run /= 2;
  const int64_t blocks = max64(1, (p.tokens + run * kWarps - 1) / (run * kWarps));
  if (blocks > INT32_MAX / p.batch / columns) return LA_ERR_UNSUPPORTED;
  const unsigned grid = (unsigned)(blocks * p.batch * columns);
  if (p.silu)
    conv_fwd_kernel<T, NP, kTaps, true><<<grid, kThreads, 0, s>>>(p, run, columns, (int)blocks);
  else
    conv_fwd_kernel<T, NP, kTaps, false><<<grid, kThreads, 0, s>>>(p, run, columns, (int)blocks);
  return check_launch();
}

template <typename T, int kTaps>
int launch_bwd(const ConvCall &p, cudaStream_t s) {
  const int64_t blocks = conv_partial_rows(1, p.tokens);
  const int columns = (p.channels + 63) / 64;
  if (blocks > INT32_MAX / p.batch / columns) return LA_ERR_UNSUPPORTED;
  const unsigned grid = (unsigned)(blocks * p.batch * columns);
  if (p.silu) conv_bwd_kernel<T, kTaps, true><<<grid, kThreads, 0, s>>>(p, columns, (int)blocks);
  else conv_bwd_kernel<T, kTaps, false><<<grid, kThreads, 0, s>>>(p, columns, (int)blocks);
  return check_launch();
}

// The widest pack (in bytes, 16 at most) that the channels and every row's start allow.
int pack_of(const ConvCall &p, bool grad, int size) {
  uint64_t bits = (uint64_t)p.channels * size;
  auto at = [&](const void *q) { bits |= (uint64_t)(uintptr_t)q; };
  auto view = [&](const TokenView &v) {
    at(v.p);
    bits |= (uint64_t)(v.sb * (int64_t)size) | (uint64_t)(v.st * (int64_t)size);
  };
  view(p.x);
  at(p.init);
  if (grad) {
    view(p.d_out);
    at(p.dx), at(p.d_init), at(p.d_final);
  } else {
    at(p.out), at(p.final_state);
  }
  return bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : 2;
}

template <typename T, int NP>
int fwd_by_taps(const ConvCall &p, cudaStream_t s) {
  if (p.taps == 2) return launch_fwd<T, NP, 2>(p, s);
  if (p.taps == 3) return launch_fwd<T, NP, 3>(p, s);
  return launch_fwd<T, NP, 4>(p, s);
}

template <typename T>
int run_fwd(ConvCall p, cudaStream_t s) {
  const int bytes = pack_of(p, false, sizeof(T));
  p.wide = bytes >= 2 * (int)sizeof(T);
  return bytes >= 4 * (int)sizeof(T) ? fwd_by_taps<T, 2>(p, s) : fwd_by_taps<T, 1>(p, s);
}

template <typename T>
int run_bwd(ConvCall p, cudaStream_t s) {
  p.wide = pack_of(p, true, sizeof(T)) >= 2 * (int)sizeof(T);
  if (p.taps == 2) return launch_bwd<T, 2>(p, s);
  if (p.taps == 3) return launch_bwd<T, 3>(p, s);
  return launch_bwd<T, 4>(p, s);
}

}  // namespace

int64_t conv_partial_rows(int64_t batch, int64_t tokens) {
  constexpr int64_t kSpan = (int64_t)kWarps * kBwdRun;
  return batch * max64(1, (tokens + kSpan - 1) / kSpan);
}

int launch_conv_fwd(const ConvCall &p, int dtype, cudaStream_t s) {
  return dtype == LA_DTYPE_FLOAT32 ? run_fwd<float>(p, s) : run_fwd<__nv_bfloat16>(p, s);
}

int launch_conv_bwd(const ConvCall &p, int dtype, cudaStream_t s) {
  return dtype == LA_DTYPE_FLOAT32 ? run_bwd<float>(p, s) : run_bwd<__nv_bfloat16>(p, s);
}

}  // namespace la
