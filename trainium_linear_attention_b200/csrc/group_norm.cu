// Group norm of each row's channels, with an activation or an activated gate,
// and its gradient.
//
//   n = (x - mean) rstd over a group of `size` neighbouring channels of a row,
//   z = n w + b,   y = act(z), or with a gate y = z act(gate)
//   gradient, with g = dy act'(z), or dy act(gate):
//     dx = rstd (g w - mean(g w) - n mean(g w n)),  d_gate = dy z act'(gate)
//     dw = sum_rows g n,  db = sum_rows g
//
// Bound by memory (6 bytes per element in bf16 with a gate, the gradient 10).
// TPR threads (2 to 512) hold a group in registers, NV packs of 8 elements
// each, so x is read once and the variance is the mean of squared differences,
// without the cancellation of E[x^2] - mean^2.  The threads walk over rows and ask
// for the next row before they compute this one.  In the gradient a thread keeps
// its columns for all its rows: the sums for dw and db stay in registers, are
// joined over the CTA's row lanes in shared memory, written as one row per CTA,
// and added by a second kernel in a fixed order.
//
// 16384 x 1024 in 16 groups with a gate's SiLU in 27 us (57% of the copy rate), its gradient
// in 41 (62%); the wait for loads, one row ahead, comes first (62 and 51% of the issue
// slots).  In fp32 38 us (80%) and 60 (85%).  Groups whose starts are not on 16 bytes
// take pairs or single values, whose accesses bound them: 16384 x 1023 in 11 groups 66.
#include <initializer_list>

#include "column_sum.cuh"
#include "group_norm.cuh"
#include "pairs.cuh"

namespace la {
namespace {

// Threads of a CTA: at least 256, or one group's.
constexpr int threads_for(int tpr) { return tpr > 256 ? tpr : 256; }

__device__ __forceinline__ int64_t row_offset(const RowView &v, uint32_t n1, int row, int rows) {
  if (n1 == (uint32_t)rows) return row * v.s1;
  const uint32_t i0 = (uint32_t)row / n1;
  return (int64_t)i0 * v.s0 + (int64_t)((uint32_t)row - i0 * n1) * v.s1;
}

// How a group's values are accessed: packs of 8 neighbours by 16 bytes (all groups
// start at 16 bytes), pairs of neighbours (at a pair's size), or single values.
enum Access { kSingle, kPairs, kPacked };

// 8 NV values of a group as they lie in memory, neighbours by access, the threads'
// accesses side by side.
template <typename T, int TPR, int NV, Access kA>
struct Held {
  static constexpr int kWords = sizeof(T) == 2 ? 4 : 8;
  uint32_t w[NV][kWords];

  static __device__ __forceinline__ int column(int t, int i, int e) {
    if constexpr (kA == kPacked) return (i * TPR + t) * 8 + e;
    if constexpr (kA == kPairs) return ((i * 4 + e / 2) * TPR + t) * 2 + (e & 1);
    return (i * 8 + e) * TPR + t;
  }
  __device__ __forceinline__ void load(const T *p, int t, int size) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (kA == kPacked) {
        const int c = column(t, i, 0);
        const bool in = c < size;
#pragma unroll
        for (int q = 0; q < kWords / 4; ++q) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (in) v = ((const uint4 *)(p + c))[q];
          w[i][4 * q] = v.x, w[i][4 * q + 1] = v.y, w[i][4 * q + 2] = v.z, w[i][4 * q + 3] = v.w;
        }
      } else if constexpr (kA == kPairs) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = column(t, i, 2 * e);
          if constexpr (sizeof(T) == 4) {
            const uint2 v = c < size ? *(const uint2 *)(p + c) : make_uint2(0, 0);
            w[i][2 * e] = v.x, w[i][2 * e + 1] = v.y;
          } else {
            w[i][e] = c < size ? *(const uint32_t *)(p + c) : 0;
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int c = column(t, i, e);
          if constexpr (sizeof(T) == 4) {
            w[i][e] = c < size ? ((const uint32_t *)p)[c] : 0;
          } else {
            const uint32_t v = c < size ? ((const uint16_t *)p)[c] : 0;
            if (e & 1) w[i][e / 2] |= v << 16;
            else w[i][e / 2] = v;
          }
        }
      }
    }
  }
  __device__ __forceinline__ void get(float2 (&x)[NV][4]) const {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (sizeof(T) == 4)
          x[i][e] = make_float2(__uint_as_float(w[i][2 * e]), __uint_as_float(w[i][2 * e + 1]));
        else
          x[i][e] = make_float2(__uint_as_float(w[i][e] << 16), __uint_as_float(w[i][e] & 0xFFFF0000u));
      }
  }
  // f of each pair, (1, 1) for values inside the group and 0 for those beyond it.
  template <class F>
  static __device__ __forceinline__ void each_inside(int t, int size, F &&f) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = column(t, i, kA == kPacked ? 0 : 2 * e) < size ? 1.f : 0.f;
        f(i, e, make_float2(x, kA != kSingle ? x : column(t, i, 2 * e + 1) < size ? 1.f : 0.f));
      }
  }
  // Sum of f(x) over the values inside the group (a pack or pair is whole, or beyond it).
  template <class F>
  static __device__ __forceinline__ float sum(const float2 (&x)[NV][4], int t, int size, F &&f) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (kA == kPacked) {
        float2 s = f(x[i][0], two(0.f));
#pragma unroll
        for (int e = 1; e < 4; ++e) s = f(x[i][e], s);
        sum += column(t, i, 0) < size ? s.x + s.y : 0.f;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 s = f(x[i][e], two(0.f));
          if constexpr (kA == kPairs)
            sum += column(t, i, 2 * e) < size ? s.x + s.y : 0.f;
          else
            sum += (column(t, i, 2 * e) < size ? s.x : 0.f) + (column(t, i, 2 * e + 1) < size ? s.y : 0.f);
        }
      }
    }
    return sum;
  }
  static __device__ __forceinline__ void store(const float2 (&x)[NV][4], T *p, int t, int size) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (kA == kPacked) {
        const int c = column(t, i, 0);
        if (c >= size) continue;
        if constexpr (sizeof(T) == 2) {
          uint32_t u[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(x[i][e].x, x[i][e].y);
            u[e] = *(const uint32_t *)&b;
          }
          *(uint4 *)(p + c) = make_uint4(u[0], u[1], u[2], u[3]);
        } else {
          *(float4 *)(p + c) = make_float4(x[i][0].x, x[i][0].y, x[i][1].x, x[i][1].y);
          *(float4 *)(p + c + 4) = make_float4(x[i][2].x, x[i][2].y, x[i][3].x, x[i][3].y);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = column(t, i, 2 * e);
          if constexpr (kA == kPairs) {
            if (c < size) store_two(p + c, x[i][e], true, true);
          } else {
            if (c < size) p[c] = from_f32<T>(x[i][e].x);
            if (c + TPR < size) p[c + TPR] = from_f32<T>(x[i][e].y);
          }
        }
      }
    }
  }
};

template <int TPR, int NV, Access kA>
__device__ __forceinline__ void load_affine(float2 (&x)[NV][4], const void *p, int dtype, float none,
                                            int64_t at, int t, int size) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[i][e] = two(none);
  } else if (dtype == LA_DTYPE_FLOAT32) {
    Held<float, TPR, NV, kA> h;
    h.load((const float *)p + at, t, size);
    h.get(x);
  } else {
    Held<__nv_bfloat16, TPR, NV, kA> h;
    h.load((const __nv_bfloat16 *)p + at, t, size);
    h.get(x);
  }
}

// Sums of two values over the TPR threads of a group; every thread gets them.
// `slot`: shared memory, two floats per warp.  With TPR > 32 every thread of the
// CTA takes part.
template <int TPR>
__device__ __forceinline__ float2 group_sum(float2 v, float2 *slot) {
#pragma unroll
  for (int m = 1; m < (TPR < 32 ? TPR : 32); m <<= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, m);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, m);
  }
  if constexpr (TPR > 32) {
    constexpr int kWarps = TPR / 32;
    const int warp = threadIdx.x >> 5;
    __syncthreads();  // the slots of the use before are read
    if ((threadIdx.x & 31) == 0) slot[warp] = v;
    __syncthreads();
    const int first = warp / kWarps * kWarps;
    v = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      const float2 x = slot[first + i];
      v.x += x.x, v.y += x.y;
    }
  }
  return v;
}
template <int TPR>
__device__ __forceinline__ float group_sum(float v, float2 *slot) {
  if constexpr (TPR <= 32) {
#pragma unroll
    for (int m = 1; m < TPR; m <<= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
  } else {
    return group_sum<TPR>(make_float2(v, 0.f), slot).x;
  }
}

template <int NV, class F>
__device__ __forceinline__ void each(F &&f) {
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) f(i, e);
}

// How a CTA's sets of TPR threads ("lanes") lie over a row's groups and the rows:
// `across` groups, threads / TPR / across rows at a time.
struct Lanes {
  int across, rows, columns;  // columns: CTAs along a row's groups
};

// Whether a group's mean is kept for the gradient as it is found, from the group's first
// value on.  Rounded together with that value it would be off by 2^-24 of it: beside fp32
// values that differ by little that is much of their differences, and the gradient's n
// would not be the forward pass'.  bf16 values that differ do so by 2^-8 of themselves at
// least: a single one among 8192 leaves a deviation of 2^-14.5 of them, and the mean is off by
// 2^-9.5 of that, under half a rounding of the outputs.  There the sum is kept (16384 x 1024,
// gradient: 41 us, with the first value read again 52).
template <typename T> constexpr bool kFromPivot = sizeof(T) == 4;

// CTAs walk the rows, the next row's loads on their way ahead of a row's sums.
template <typename T, int TPR, int NV, Access kA>
__global__ void __launch_bounds__(threads_for(TPR), TPR <= 256 && NV == 1 ? 4 : 1)
group_norm_fwd_kernel(const GroupNormCall p, const Lanes lanes) {
  using H = Held<T, TPR, NV, kA>;
  __shared__ float2 slot[32];
  const int t = threadIdx.x % TPR, lane = threadIdx.x / TPR;
  const int lane_row = lane / lanes.across;
  const int group = blockIdx.x % lanes.columns * lanes.across + lane - lane_row * lanes.across;
  const bool member = group < p.groups && lane_row < lanes.rows;
  const int64_t c0 = member ? (int64_t)group * p.size : 0;
  const int ctas = gridDim.x / lanes.columns, cta = blockIdx.x / lanes.columns;
  const int stride = ctas * lanes.rows, rows = (int)p.rows;  // (stride is far below 2^30)
  H hx, hg;
  float next_pivot;
  auto fetch = [&](int first) {
    // (idle lanes redo a row, unstored)
    const int row = member && first + lane_row < rows ? first + lane_row : first;
    const T *src = (const T *)p.x.p + row_offset(p.x, p.n1, row, rows) + c0;
    hx.load(src, t, p.size);
    if (p.gate.p) hg.load((const T *)p.gate.p + row_offset(p.gate, p.n1, row, rows) + c0, t, p.size);
    next_pivot = to_f32(*src);
  };
  fetch(cta * lanes.rows);
  float2 w[NV][4], b[NV][4];
  load_affine<TPR, NV, kA>(w, p.weight, p.weight_dtype, 1.f, c0, t, p.size);
  load_affine<TPR, NV, kA>(b, p.bias, p.weight_dtype, 0.f, c0, t, p.size);
  const float inv = 1.f / (float)p.size;
  for (int first = cta * lanes.rows; first < rows; first += stride) {
    const int row = first + lane_row;
    const bool live = member && row < rows;
    // Everything is taken from the group's first value on: a large common part
    // then costs the mean and the differences no digits, and equal values give 0.
    float2 x[NV][4], g[NV][4];
    hx.get(x);
    if (p.gate.p) hg.get(g);
    const float pivot = next_pivot;
    if (first + stride < rows) fetch(first + stride);
    each<NV>([&](int i, int e) { x[i][e] = __fadd2_rn(x[i][e], two(-pivot)); });
    const float sum = H::sum(x, t, p.size, [](float2 v, float2 s) { return __fadd2_rn(v, s); });
    const float mean = group_sum<TPR>(sum, slot) * inv;
    each<NV>([&](int i, int e) { x[i][e] = __fadd2_rn(x[i][e], two(-mean)); });
    const float sq = H::sum(x, t, p.size, [](float2 v, float2 s) { return __ffma2_rn(v, v, s); });
    const float rstd = 1.f / sqrtf(fmaf(group_sum<TPR>(sq, slot), inv, p.eps));
    if (p.stats && live && t == 0)
      *(float2 *)(p.stats + 2 * ((int64_t)row * p.groups + group)) =
          make_float2(kFromPivot<T> ? mean : pivot + mean, rstd);
    each<NV>([&](int i, int e) {
      x[i][e] = __ffma2_rn(__fmul2_rn(x[i][e], two(rstd)), w[i][e], b[i][e]);
    });
    if (p.gate.p) {
      if (p.silu)
        each<NV>([&](int i, int e) { g[i][e] = __fmul2_rn(g[i][e], sigmoid_two<T>(g[i][e])); });
      each<NV>([&](int i, int e) { x[i][e] = __fmul2_rn(x[i][e], g[i][e]); });
    } else if (p.silu) {
      each<NV>([&](int i, int e) { x[i][e] = __fmul2_rn(x[i][e], sigmoid_two<T>(x[i][e])); });
    }
    if (live) H::store(x, (T *)p.out + (int64_t)row * p.groups * p.size + c0, t, p.size);
  }
}

template <typename T, int TPR, int NV, Access kA>
__global__ void __launch_bounds__(threads_for(TPR), TPR <= 256 && NV == 1 ? 2 : 1) group_norm_bwd_kernel(const GroupNormCall p,
                                                                        const Lanes lanes) {
  using H = Held<T, TPR, NV, kA>;
  __shared__ float2 slot[32];
  extern __shared__ float joined[];  // (rows - 1, across, 2, size) with several rows
  column_sum_may_start();
  const int t = threadIdx.x % TPR, lane = threadIdx.x / TPR;
  const int lane_row = lane / lanes.across;
  const int group = blockIdx.x % lanes.columns * lanes.across + lane - lane_row * lanes.across;
  const bool member = group < p.groups && lane_row < lanes.rows;
  const int64_t c0 = member ? (int64_t)group * p.size : 0;
  float2 w[NV][4], b[NV][4], dw[NV][4] = {}, db[NV][4] = {};
  load_affine<TPR, NV, kA>(w, p.weight, p.weight_dtype, 1.f, c0, t, p.size);
  load_affine<TPR, NV, kA>(b, p.bias, p.weight_dtype, 0.f, c0, t, p.size);
  const float inv = 1.f / (float)p.size;
  const int ctas = gridDim.x / lanes.columns, cta = blockIdx.x / lanes.columns;
  const int stride = ctas * lanes.rows, rows = (int)p.rows;  // (stride is far below 2^30)
  // The next row is loaded ahead of this one's sums.
  H hx, hd, hg;
  float2 next_st;
  float next_pivot = 0.f;
  auto fetch = [&](int first) {
    const int row = member && first + lane_row < rows ? first + lane_row : first;
    const T *src = (const T *)p.x.p + row_offset(p.x, p.n1, row, rows) + c0;
    hx.load(src, t, p.size);
    if (kFromPivot<T>) next_pivot = to_f32(*src);
    hd.load((const T *)p.d_out.p + row_offset(p.d_out, p.n1, row, rows) + c0, t, p.size);
    if (p.gate.p)
      hg.load((const T *)p.gate.p + row_offset(p.gate, p.n1, row, rows) + c0, t, p.size);
    next_st = *(const float2 *)(p.stats + 2 * ((int64_t)row * p.groups + (member ? group : 0)));
  };
  fetch(cta * lanes.rows);
  for (int first = cta * lanes.rows; first < rows; first += stride) {
    const int row = first + lane_row;
    const bool live = member && row < rows;  // others redo a row, unstored
    float2 n[NV][4], g[NV][4], u[NV][4];
    hx.get(n);
    hd.get(g);
    if (p.gate.p) hg.get(u);
    const float2 st = next_st;
    const float pivot = next_pivot;
    if (first + stride < rows) fetch(first + stride);
    // (0 beyond the group, where the sums below would meet an infinite -mean rstd)
    H::each_inside(t, p.size, [&](int i, int e, float2 in) {
      if constexpr (kFromPivot<T>) n[i][e] = __fadd2_rn(n[i][e], two(-pivot));
      n[i][e] = __fmul2_rn(__fadd2_rn(n[i][e], two(-st.x)), make_float2(in.x * st.y, in.y * st.y));
    });
    // act'(v) = s + v s (1 - s) with s = sigmoid(v); the activation v s
    auto slope = [](float2 vs, float2 s) {
      return __ffma2_rn(vs, __ffma2_rn(s, two(-1.f), two(1.f)), s);
    };
    if (p.gate.p) {
      if (p.silu) {
        each<NV>([&](int i, int e) {
          const float2 z = __ffma2_rn(n[i][e], w[i][e], b[i][e]);
          const float2 s = sigmoid_two<T>(u[i][e]), us = __fmul2_rn(u[i][e], s);
          u[i][e] = __fmul2_rn(__fmul2_rn(g[i][e], z), slope(us, s));
          g[i][e] = __fmul2_rn(g[i][e], us);
        });
      } else {
        each<NV>([&](int i, int e) {
          const float2 dz = __fmul2_rn(g[i][e], __ffma2_rn(n[i][e], w[i][e], b[i][e]));
          g[i][e] = __fmul2_rn(g[i][e], u[i][e]);
          u[i][e] = dz;
        });
      }
      if (live) H::store(u, (T *)p.d_gate + (int64_t)row * p.groups * p.size + c0, t, p.size);
    } else if (p.silu) {
      each<NV>([&](int i, int e) {
        const float2 z = __ffma2_rn(n[i][e], w[i][e], b[i][e]);
        const float2 s = sigmoid_two<T>(z);
        g[i][e] = __fmul2_rn(g[i][e], slope(__fmul2_rn(z, s), s));
      });
    }
    float2 s0 = two(0.f), s1 = two(0.f);
    if (live) {
      each<NV>([&](int i, int e) {
        dw[i][e] = __ffma2_rn(g[i][e], n[i][e], dw[i][e]);
        db[i][e] = __fadd2_rn(db[i][e], g[i][e]);
      });
    }
    each<NV>([&](int i, int e) {
      g[i][e] = __fmul2_rn(g[i][e], w[i][e]);  // (beyond the group dy is zero)
      s0 = __fadd2_rn(s0, g[i][e]);
      s1 = __ffma2_rn(g[i][e], n[i][e], s1);
    });
    float2 sums = group_sum<TPR>(make_float2(s0.x + s0.y, s1.x + s1.y), slot);
    sums = make_float2(-sums.x * inv, -sums.y * inv);
    each<NV>([&](int i, int e) {
      g[i][e] = __fmul2_rn(__ffma2_rn(n[i][e], two(sums.y), __fadd2_rn(g[i][e], two(sums.x))),
                           two(st.y));
    });
    if (live) H::store(g, (T *)p.dx + (int64_t)row * p.groups * p.size + c0, t, p.size);
  }
  if (!p.partial) return;
  // over the row lanes, in their order
  const int at = lane % lanes.across * 2 * p.size;
  const int wide = lanes.across * 2 * p.size;
  if (lanes.rows > 1) {
    if (member && lane_row > 0) {
      float *dst = joined + (int64_t)(lane_row - 1) * wide + at;
      each<NV>([&](int i, int e) {
        const int c = H::column(t, i, 2 * e), d = H::column(t, i, 2 * e + 1);
        if (c < p.size) dst[c] = dw[i][e].x, dst[p.size + c] = db[i][e].x;
        if (d < p.size) dst[d] = dw[i][e].y, dst[p.size + d] = db[i][e].y;
      });
    }
    __syncthreads();
  }
  if (!member || lane_row > 0) return;
  const int64_t channels = (int64_t)p.groups * p.size;
  float *out = p.partial + (int64_t)cta * 2 * channels + c0;
  auto finish = [&](int c, float vw, float vb) {
    if (c >= p.size) return;
    for (int r = 0; r < lanes.rows - 1; ++r) {
      vw += joined[(int64_t)r * wide + at + c];
      vb += joined[(int64_t)r * wide + at + p.size + c];
    }
    out[c] = vw;
    out[channels + c] = vb;
  };
  each<NV>([&](int i, int e) {
    finish(H::column(t, i, 2 * e), dw[i][e].x, db[i][e].x);
    finish(H::column(t, i, 2 * e + 1), dw[i][e].y, db[i][e].y);
  });
}

// Threads per group and values per thread for a group's size: 8 values a thread
// while 512 threads hold a group, so that few lanes idle; packs of up to 512
// values within one warp.
template <Access kA, class F>
int by_size(int d, F &&f) {
  if (d <= 16) return f.template run<2, 1, kA>();
  if (d <= 32) return f.template run<4, 1, kA>();
  if (d <= 64) return f.template run<8, 1, kA>();
  if (d <= 128) return f.template run<16, 1, kA>();
  if (d <= 256) return f.template run<32, 1, kA>();
  if (d <= 512) {
    if constexpr (kA == kPacked) return f.template run<32, 2, kA>();
    else return f.template run<64, 1, kA>();
  }
  if (d <= 1024) return f.template run<128, 1, kA>();
  if (d <= 2048) return f.template run<256, 1, kA>();
  if (d <= 4096) return f.template run<256, 2, kA>();
  return f.template run<512, 2, kA>();
}
template <class F>
int by_access(const GroupNormCall &p, Access access, F &&f) {
  if (access == kPacked) return by_size<kPacked>(p.size, f);
  if (access == kPairs) return by_size<kPairs>(p.size, f);
  return by_size<kSingle>(p.size, f);
}

constexpr int kMostPerSm = 8;

// The access that every group of the inputs and of the contiguous outputs allows.
Access access_of(const GroupNormCall &p, int dtype, std::initializer_list<const RowView *> views,
                 std::initializer_list<const void *> plain) {
  const uint64_t size = dtype == LA_DTYPE_FLOAT32 ? 4 : 2;
  uint64_t bits = p.size * size, wbits = 0;
  for (const RowView *v : views)
    if (v->p) bits |= (uint64_t)(uintptr_t)v->p | (uint64_t)v->s0 * size | (uint64_t)v->s1 * size;
  for (const void *q : plain) bits |= (uint64_t)(uintptr_t)q;
  for (const void *q : {p.weight, p.bias}) wbits |= (uint64_t)(uintptr_t)q;
  if (p.size % 8 == 0 && bits % 16 == 0 && wbits % 16 == 0) return kPacked;
  return p.size % 2 == 0 && bits % (2 * size) == 0 && wbits % 8 == 0 ? kPairs : kSingle;
}

Lanes lanes_of(int groups, int per) {
  Lanes l;
  l.columns = (groups + per - 1) / per;
  l.across = (groups + l.columns - 1) / l.columns;
  l.rows = per / l.across;
  return l;
}

// One wave of CTAs: this many per SM of a kernel.
template <class Kernel>
int ctas_per_sm(Kernel kernel, int threads, int smem) {
  int n = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem) != cudaSuccess) {
    cudaGetLastError();
    n = 2;
  }
  return n < 1 ? 1 : n > kMostPerSm ? kMostPerSm : n;
}

template <typename T>
struct FwdLaunch {
  const GroupNormCall &p;
  int sm_count;
  cudaStream_t s;
  template <int TPR, int NV, Access kA>
  int run() {
    const Lanes l = lanes_of(p.groups, threads_for(TPR) / TPR);
    auto kernel = group_norm_fwd_kernel<T, TPR, NV, kA>;
    static const int per_sm = ctas_per_sm(kernel, threads_for(TPR), 0);
    const int64_t most = (p.rows + l.rows - 1) / l.rows;
    const int64_t ctas = min64(most, max64(1, (int64_t)sm_count * per_sm / l.columns));
    if (ctas > INT32_MAX / l.columns) return LA_ERR_UNSUPPORTED;
    kernel<<<(unsigned)(ctas * l.columns), threads_for(TPR), 0, s>>>(p, l);
    return check_launch();
  }
};

template <typename T>
struct BwdLaunch {
  const GroupNormCall &p;
  int sm_count;
  int64_t *partial_rows;
  cudaStream_t s;
  template <int TPR, int NV, Access kA>
  int run() {
    constexpr int per = threads_for(TPR) / TPR;
    auto kernel = group_norm_bwd_kernel<T, TPR, NV, kA>;
    const Lanes l = lanes_of(p.groups, per);
    const int smem = p.partial ? (l.rows - 1) * l.across * 2 * p.size * 4 : 0;  // at most 28 KB
    static const int per_sm = ctas_per_sm(kernel, threads_for(TPR), 16 * 1024);
    const int64_t most = (p.rows + l.rows - 1) / l.rows;
    const int64_t ctas = min64(most, max64(1, (int64_t)sm_count * per_sm / l.columns));
    *partial_rows = ctas;
    if (ctas > INT32_MAX / l.columns) return LA_ERR_UNSUPPORTED;
    kernel<<<(unsigned)(ctas * l.columns), threads_for(TPR), smem, s>>>(p, l);
    return check_launch();
  }
};

}  // namespace

int64_t group_norm_partial_rows(int64_t rows, int sm_count) {
  return min64(rows, (int64_t)sm_count * kMostPerSm);
}

int launch_group_norm_fwd(const GroupNormCall &p, int dtype, cudaStream_t s) {
  const Access access = access_of(p, dtype, {&p.x, &p.gate}, {p.out});
  DeviceInfo info;
  const int st = current_device_info(&info);
  if (st != LA_OK) return st;
  if (dtype == LA_DTYPE_FLOAT32) return by_access(p, access, FwdLaunch<float>{p, info.sm_count, s});
  return by_access(p, access, FwdLaunch<__nv_bfloat16>{p, info.sm_count, s});
}

int launch_group_norm_bwd(const GroupNormCall &p, int dtype, int sm_count, int64_t *partial_rows,
                          cudaStream_t s) {
  const Access access = access_of(p, dtype, {&p.x, &p.gate, &p.d_out}, {p.dx, p.d_gate});
  if (dtype == LA_DTYPE_FLOAT32)
    return by_access(p, access, BwdLaunch<float>{p, sm_count, partial_rows, s});
  return by_access(p, access, BwdLaunch<__nv_bfloat16>{p, sm_count, partial_rows, s});
}

}  // namespace la
