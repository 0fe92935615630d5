// Causal convolution of each channel with 2 to 4 taps, an activation, and its
// gradient.
//
//   z_t = bias + sum_j w_j x_{t - taps + 1 + j},   y = z, or z sigmoid(z)
//   dz = dy, or dy sigmoid(z) (1 + z (1 - sigmoid(z)))
//   dx_t = sum_j w_j dz_{t + taps - 1 - j},  dw_j = sum_t dz_t x_{t - taps + 1 + j}
//
// Bound by memory: x read and y written once (4 bytes per element in bf16),
// the gradient also reads dy (6).  A thread has a pack of neighbouring channels,
// as wide as their alignment allows (16 bytes at most), and walks tokens with the
// taps' window in registers; the tokens ahead of its own are read twice, the
// second time from the caches.  The gradient computes z again instead of
// keeping it.  A walk there meets dz_t once and adds it to the taps' sums
// that are still open, so that dx, dw and the bias' gradient come from one pass;
// the sums over tokens are joined over the CTA's warps in shared memory, written
// as one row per CTA, and the rows added by a second kernel in a fixed order.
#include "column_sum.cuh"
#include "short_conv.cuh"

namespace la {
namespace {

constexpr int kThreads = 256;
constexpr int kRun = 8;        // tokens of a thread, forward
constexpr int kBwdRun = 32;    // tokens of a thread, gradient
constexpr int kBwdWarps = 8;
constexpr int kBatch = 4;      // tokens whose loads are on their way together, gradient

// kVec neighbouring elements as they lie in memory.
template <typename T, int kVec> struct Pack {
  static constexpr int kBytes = kVec * (int)sizeof(T);
  static constexpr int kWords = kBytes >= 4 ? kBytes / 4 : 1;
  uint32_t w[kWords];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  __device__ __forceinline__ void load(const T *p) {
    if constexpr (kBytes == 16) {
      const uint4 v = *(const uint4 *)p;
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else if constexpr (kBytes == 8) {
      const uint2 v = *(const uint2 *)p;
      w[0] = v.x, w[1] = v.y;
    } else if constexpr (kBytes == 4) {
      w[0] = *(const uint32_t *)p;
    } else {
      w[0] = *(const uint16_t *)p;
    }
  }
  __device__ __forceinline__ void store(T *p) const {
    if constexpr (kBytes == 16) *(uint4 *)p = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (kBytes == 8) *(uint2 *)p = make_uint2(w[0], w[1]);
    else if constexpr (kBytes == 4) *(uint32_t *)p = w[0];
    else *(uint16_t *)p = (uint16_t)w[0];
  }
  __device__ __forceinline__ void get(float (&x)[kVec]) const {
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      if constexpr (sizeof(T) == 4) x[e] = __uint_as_float(w[e]);
      else x[e] = __uint_as_float(e & 1 ? w[e / 2] & 0xFFFF0000u : w[e / 2] << 16);
    }
  }
  __device__ __forceinline__ void set(const float (&x)[kVec]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) w[e] = __float_as_uint(x[e]);
    } else if constexpr (kVec == 1) {
      w[0] = __bfloat16_as_ushort(__float2bfloat16_rn(x[0]));
    } else {
#pragma unroll
      for (int e = 0; e < kVec / 2; ++e) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]);
        w[e] = *(const uint32_t *)&b;
      }
    }
  }
};

// A sequence's rows with the tokens before it.
template <typename T, int kVec, int kTaps>
struct Row {
  const T *x;      // this sequence, this thread's channels
  const T *init;   // null, or the kTaps - 1 rows before
  int64_t st;
  int channels;
  int64_t len;
  __device__ __forceinline__ void load(Pack<T, kVec> &v, int64_t t) const {
    v.zero();
    if (t >= 0) {
      if (t < len) v.load(x + t * st);
    } else if (init && t >= -(kTaps - 1)) {
      v.load(init + (t + kTaps - 1) * channels);
    }
  }
};

template <int kVec, int kTaps>
struct Weights {
  float w[kTaps][kVec], b[kVec];
  template <typename TW>
  __device__ __forceinline__ void load_as(const ConvCall &p, int c) {
    const TW *src = (const TW *)p.weight + (int64_t)c * kTaps;
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
#pragma unroll
      for (int j = 0; j < kTaps; ++j) w[j][e] = to_f32(src[e * kTaps + j]);
      b[e] = p.bias ? to_f32(((const TW *)p.bias)[c + e]) : 0.f;
    }
  }
  __device__ __forceinline__ void load(const ConvCall &p, int c) {
    if (p.weight_dtype == LA_DTYPE_FLOAT32) load_as<float>(p, c);
    else load_as<__nv_bfloat16>(p, c);
  }
};

template <typename T>
__device__ __forceinline__ float sigmoid_of(float z) {
  const float e = Fn<T>::exp(-fabsf(z));
  const float r = Fn<T>::rcp(1.f + e);
  return z < 0.f ? e * r : r;
}

// A CTA: `lanes` packs of channels, 256 / lanes runs of kRun tokens.
template <typename T, int kVec, int kTaps>
__global__ void __launch_bounds__(kThreads) conv_fwd_kernel(const ConvCall p, const int lanes,
                                                          const int columns,
                                                          const unsigned blocks) {
  const int packs = p.channels / kVec;
  const int column = blockIdx.x % columns * lanes + threadIdx.x % lanes;
  const unsigned block = blockIdx.x / columns;
  const int64_t ib = block / blocks;
  const int64_t run = (int64_t)(block % blocks) * (kThreads / lanes) + threadIdx.x / lanes;
  const int64_t t0 = run * kRun;
  if (column >= packs || (t0 >= p.tokens && run > 0)) return;
  const int c = column * kVec;
  Row<T, kVec, kTaps> row;
  row.x = (const T *)p.x.p + ib * p.x.sb + c;
  row.init = p.init ? (const T *)p.init + ib * (kTaps - 1) * p.channels + c : nullptr;
  row.st = p.x.st, row.channels = p.channels;
  row.len = recur_length(p.lengths, p.lengths64, ib, p.tokens);
  Pack<T, kVec> in[kRun + kTaps - 1];
#pragma unroll
  for (int i = 0; i < kRun + kTaps - 1; ++i) row.load(in[i], t0 + i - (kTaps - 1));
  Weights<kVec, kTaps> w;
  w.load(p, c);
  T *out = (T *)p.out + (ib * p.tokens + t0) * p.channels + c;
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    float z[kVec];
#pragma unroll
    for (int e = 0; e < kVec; ++e) z[e] = w.b[e];
#pragma unroll
    for (int j = 0; j < kTaps; ++j) {
      float x[kVec];
      in[i + j].get(x);
#pragma unroll
      for (int e = 0; e < kVec; ++e) z[e] = fmaf(w.w[j][e], x[e], z[e]);
    }
    if (p.silu) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) z[e] *= sigmoid_of<T>(z[e]);
    }
    if (t0 + i < p.tokens) {
      Pack<T, kVec> y;
      y.set(z);
      if (t0 + i >= row.len) y.zero();
      y.store(out + (int64_t)i * p.channels);
    }
  }
  if (p.final_state && run == 0) {
    T *dst = (T *)p.final_state + ib * (kTaps - 1) * p.channels + c;
#pragma unroll
    for (int j = 0; j < kTaps - 1; ++j) {
      Pack<T, kVec> v;
      row.load(v, row.len - (kTaps - 1) + j);
      v.store(dst + (int64_t)j * p.channels);
    }
  }
}

// A CTA: 32 packs of channels, kBwdWarps runs of kBwdRun tokens.
template <typename T, int kVec, int kTaps>
__global__ void __launch_bounds__(kBwdWarps * 32) conv_bwd_kernel(const ConvCall p,
                                                                 const int columns,
                                                                 const unsigned blocks) {
  constexpr int kSums = kTaps + 1;
  __shared__ float part[kBwdWarps][kSums][32 * kVec];
  column_sum_may_start();
  const int packs = p.channels / kVec;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int column0 = blockIdx.x % columns * 32, column = column0 + lane;
  const unsigned sums_row = blockIdx.x / columns;
  const bool live = column < packs;
  const int c = live ? column * kVec : 0;
  const int64_t ib = sums_row / blocks, block = sums_row % blocks;
  const int64_t t0 = (block * kBwdWarps + warp) * kBwdRun;
  Row<T, kVec, kTaps> row, dy;
  row.x = (const T *)p.x.p + ib * p.x.sb + c;
  row.init = p.init ? (const T *)p.init + ib * (kTaps - 1) * p.channels + c : nullptr;
  row.st = p.x.st, row.channels = p.channels;
  row.len = live ? recur_length(p.lengths, p.lengths64, ib, p.tokens) : 0;
  if (!live) row.init = nullptr;
  dy = row;
  dy.x = (const T *)p.d_out.p + ib * p.d_out.sb + c;
  dy.st = p.d_out.st;
  dy.init = nullptr;
  float sums[kSums][kVec] = {};
  // (the first run also ends the initial state's rows)
  const bool first = t0 == 0;
  if (t0 < p.tokens || first) {
    Weights<kVec, kTaps> w;
    w.load(p, c);
    float x[kTaps][kVec], open[kTaps][kVec] = {};  // the window; dx of its tokens so far
#pragma unroll
    for (int j = 0; j < kTaps - 1; ++j) {
      Pack<T, kVec> v;
      row.load(v, t0 - (kTaps - 1) + j);
      v.get(x[j + 1]);
    }
    T *dx = (T *)p.dx + ib * p.tokens * p.channels + c;
    T *d_init = p.d_init ? (T *)p.d_init + ib * (kTaps - 1) * p.channels + c : nullptr;
    const T *d_final = p.d_final ? (const T *)p.d_final + ib * (kTaps - 1) * p.channels + c : nullptr;
    const int64_t len = recur_length(p.lengths, p.lengths64, ib, p.tokens);
    const int64_t end = min64(t0 + kBwdRun, p.tokens);
    for (int64_t t = t0; t < end + kTaps - 1; t += kBatch) {
      Pack<T, kVec> px[kBatch], pd[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) row.load(px[i], t + i), dy.load(pd[i], t + i);
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (t + i >= end + kTaps - 1) break;
#pragma unroll
        for (int j = 0; j < kTaps - 1; ++j)
#pragma unroll
          for (int e = 0; e < kVec; ++e) x[j][e] = x[j + 1][e], open[j][e] = open[j + 1][e];
        px[i].get(x[kTaps - 1]);
        float g[kVec];
        pd[i].get(g);
#pragma unroll
        for (int e = 0; e < kVec; ++e) open[kTaps - 1][e] = 0.f;
        if (p.silu) {
          float z[kVec];
#pragma unroll
          for (int e = 0; e < kVec; ++e) {
            z[e] = w.b[e];
#pragma unroll
            for (int j = 0; j < kTaps; ++j) z[e] = fmaf(w.w[j][e], x[j][e], z[e]);
            const float s = sigmoid_of<T>(z[e]);
            g[e] *= s * fmaf(z[e], 1.f - s, 1.f);
          }
        }
        const bool inside = t + i < len;
        const bool own = inside && t + i < end;
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          if (!inside) g[e] = 0.f;
          const float own_g = own ? g[e] : 0.f;
#pragma unroll
          for (int j = 0; j < kTaps; ++j) {
            open[j][e] = fmaf(w.w[j][e], g[e], open[j][e]);
            if (own) sums[j][e] = fmaf(own_g, x[j][e], sums[j][e]);
          }
          sums[kTaps][e] += own_g;
        }
        // the window's oldest token is done
        const int64_t at = t + i - (kTaps - 1);
        if (live && (at >= t0 || first)) {
          const int64_t back = at - (len - (kTaps - 1));  // row of the final state
          if (d_final && back >= 0 && back < kTaps - 1) {
            Pack<T, kVec> v;
            v.load(d_final + back * p.channels);
            float f[kVec];
            v.get(f);
#pragma unroll
            for (int e = 0; e < kVec; ++e) open[0][e] += f[e];
          }
          Pack<T, kVec> v;
          v.set(open[0]);
          if (at >= 0) v.store(dx + at * p.channels);
          else if (d_init) v.store(d_init + (at + kTaps - 1) * p.channels);
        }
      }
    }
  }
  if (!p.partial) return;
#pragma unroll
  for (int j = 0; j < kSums; ++j)
#pragma unroll
    for (int e = 0; e < kVec; ++e) part[warp][j][e * 32 + lane] = sums[j][e];
  __syncthreads();
  float *dst = p.partial + (int64_t)sums_row * p.channels * kSums;
  for (int i = threadIdx.x; i < kSums * 32 * kVec; i += kBwdWarps * 32) {
    const int j = i / (32 * kVec), at = i % (32 * kVec);
    const int channel = (column0 + at % 32) * kVec + at / 32;
    if (channel >= p.channels) continue;
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < kBwdWarps; ++k) sum += part[k][j][at];
    if (j < kTaps) dst[(int64_t)channel * kTaps + j] = sum;
    else dst[(int64_t)p.channels * kTaps + channel] = sum;
  }
}

template <typename T, int kVec, int kTaps>
int launch_fwd(const ConvCall &p, cudaStream_t s) {
  const int packs = p.channels / kVec;
  int lanes = 32;  // packs of a CTA's row: a warp's, fewer where there are few
  while (lanes > 1 && lanes / 2 >= packs) lanes /= 2;
  const int64_t runs = max64(1, (p.tokens + kRun - 1) / kRun);
  const int per = kThreads / lanes;
  const int64_t blocks = (runs + per - 1) / per;
  const int columns = (packs + lanes - 1) / lanes;
  if (blocks > INT32_MAX / p.batch / columns) return LA_ERR_UNSUPPORTED;
  conv_fwd_kernel<T, kVec, kTaps><<<(unsigned)(blocks * p.batch * columns), kThreads, 0, s>>>(
      p, lanes, columns, (unsigned)blocks);
  return check_launch();
}

template <typename T, int kVec, int kTaps>
int launch_bwd(const ConvCall &p, cudaStream_t s) {
  const int packs = p.channels / kVec;
  const int64_t blocks = conv_partial_rows(1, p.tokens);
  const int columns = (packs + 31) / 32;
  if (blocks > INT32_MAX / p.batch / columns) return LA_ERR_UNSUPPORTED;
  conv_bwd_kernel<T, kVec, kTaps><<<(unsigned)(blocks * p.batch * columns), kBwdWarps * 32, 0, s>>>(
      p, columns, (unsigned)blocks);
  return check_launch();
}

// The widest pack that the channels and every row's start allow.
template <typename T>
int pack_of(const ConvCall &p, bool grad) {
  const uint64_t size = sizeof(T);
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
  return (int)((bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : 2) / size);
}

template <typename T, int kVec>
int by_taps(const ConvCall &p, bool grad, cudaStream_t s) {
  // the gradient keeps the taps' sums in registers: packs of 4 at most
  constexpr int kBwdVec = kVec > 4 ? 4 : kVec;
  if (p.taps == 2) return grad ? launch_bwd<T, kBwdVec, 2>(p, s) : launch_fwd<T, kVec, 2>(p, s);
  if (p.taps == 3) return grad ? launch_bwd<T, kBwdVec, 3>(p, s) : launch_fwd<T, kVec, 3>(p, s);
  return grad ? launch_bwd<T, kBwdVec, 4>(p, s) : launch_fwd<T, kVec, 4>(p, s);
}

template <typename T>
int by_pack(const ConvCall &p, bool grad, cudaStream_t s) {
  const int vec = pack_of<T>(p, grad);
  if constexpr (sizeof(T) == 2) {
    if (vec == 8) return by_taps<T, 8>(p, grad, s);
  }
  if (vec == 4) return by_taps<T, 4>(p, grad, s);
  if (vec == 2) return by_taps<T, 2>(p, grad, s);
  return by_taps<T, 1>(p, grad, s);
}

}  // namespace

int64_t conv_partial_rows(int64_t batch, int64_t tokens) {
  constexpr int64_t kSpan = (int64_t)kBwdWarps * kBwdRun;
  return batch * max64(1, (tokens + kSpan - 1) / kSpan);
}

int launch_conv_fwd(const ConvCall &p, int dtype, cudaStream_t s) {
  return dtype == LA_DTYPE_FLOAT32 ? by_pack<float>(p, false, s)
                                   : by_pack<__nv_bfloat16>(p, false, s);
}

int launch_conv_bwd(const ConvCall &p, int dtype, cudaStream_t s) {
  return dtype == LA_DTYPE_FLOAT32 ? by_pack<float>(p, true, s) : by_pack<__nv_bfloat16>(p, true, s);
}

}  // namespace la
