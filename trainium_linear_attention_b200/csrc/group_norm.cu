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
// without the cancellation of E[x^2] - mean^2.  In the gradient a thread keeps
// its columns for all its rows: the sums for dw and db stay in registers, are
// joined over the CTA's row lanes in shared memory, written as one row per CTA,
// and added by a second kernel in a fixed order.
#include "column_sum.cuh"
#include "group_norm.cuh"

namespace la {
namespace {

// Threads of a CTA: at least 256, or one group's.
constexpr int threads_for(int tpr) { return tpr > 256 ? tpr : 256; }

struct Unit {  // a row's group
  int64_t row;
  int group;
};

__device__ __forceinline__ int64_t row_offset(const RowView &v, uint32_t n1, int64_t row,
                                              int64_t rows) {
  if (n1 == rows) return row * v.s1;
  if (rows <= UINT32_MAX) {  // 32-bit division
    const uint32_t r = (uint32_t)row, i0 = r / n1;
    return (int64_t)i0 * v.s0 + (int64_t)(r - i0 * n1) * v.s1;
  }
  return row / n1 * v.s0 + row % n1 * v.s1;
}

// Packs of 8 elements of a group as they lie in memory (kPacked: 16-byte
// accesses), or single elements TPR apart.
template <typename T, int TPR, int NV, bool kPacked>
struct Held {
  static constexpr int kWords = sizeof(T) == 2 ? 4 : 8;
  uint32_t w[NV][kWords];

  static __device__ __forceinline__ int column(int t, int i, int e) {
    return kPacked ? (i * TPR + t) * 8 + e : (i * 8 + e) * TPR + t;
  }
  __device__ __forceinline__ void load(const T *p, int t, int size) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (kPacked) {
        const int c = column(t, i, 0);
        const bool in = c < size;
#pragma unroll
        for (int q = 0; q < kWords / 4; ++q) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (in) v = ((const uint4 *)(p + c))[q];
          w[i][4 * q] = v.x, w[i][4 * q + 1] = v.y, w[i][4 * q + 2] = v.z, w[i][4 * q + 3] = v.w;
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
  __device__ __forceinline__ void get(float (&x)[NV][8]) const {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if constexpr (sizeof(T) == 4) x[i][e] = __uint_as_float(w[i][e]);
        else x[i][e] = __uint_as_float(e & 1 ? w[i][e / 2] & 0xFFFF0000u : w[i][e / 2] << 16);
      }
  }
  static __device__ __forceinline__ void store(const float (&x)[NV][8], T *p, int t, int size) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (kPacked) {
        const int c = column(t, i, 0);
        if (c >= size) continue;
        if constexpr (sizeof(T) == 2) {
          uint32_t u[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(x[i][2 * e], x[i][2 * e + 1]);
            u[e] = *(const uint32_t *)&b;
          }
          *(uint4 *)(p + c) = make_uint4(u[0], u[1], u[2], u[3]);
        } else {
          *(float4 *)(p + c) = make_float4(x[i][0], x[i][1], x[i][2], x[i][3]);
          *(float4 *)(p + c + 4) = make_float4(x[i][4], x[i][5], x[i][6], x[i][7]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int c = column(t, i, e);
          if (c < size) p[c] = from_f32<T>(x[i][e]);
        }
      }
    }
  }
};

template <int TPR, int NV, bool kPacked>
__device__ __forceinline__ void load_affine(float (&x)[NV][8], const void *p, int dtype, float none,
                                            int64_t at, int t, int size) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[i][e] = none;
  } else if (dtype == LA_DTYPE_FLOAT32) {
    Held<float, TPR, NV, kPacked> h;
    h.load((const float *)p + at, t, size);
    h.get(x);
  } else {
    Held<__nv_bfloat16, TPR, NV, kPacked> h;
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

// sigmoid(z), as the inputs' type wants it
template <typename T>
__device__ __forceinline__ float sigmoid_of(float z) {
  if constexpr (sizeof(T) == 4) {
    const float e = expf(-fabsf(z));
    return (z < 0.f ? e : 1.f) / (1.f + e);
  } else {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-fabsf(z) * 1.4426950408889634f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
    return z < 0.f ? e * r : r;
  }
}

template <typename T, int TPR, int NV, bool kPacked>
__global__ void __launch_bounds__(threads_for(TPR)) group_norm_fwd_kernel(const GroupNormCall p) {
  using H = Held<T, TPR, NV, kPacked>;
  __shared__ float2 slot[32];
  const int t = threadIdx.x % TPR;
  const int64_t units = p.rows * p.groups;
  const int64_t unit0 = (int64_t)blockIdx.x * (threads_for(TPR) / TPR) + threadIdx.x / TPR;
  const bool live = unit0 < units;
  const int64_t unit = live ? unit0 : units - 1;  // idle lanes redo the last group, unstored
  int64_t row;
  int group;
  if (units <= UINT32_MAX) {
    const uint32_t u = (uint32_t)unit, r = u / (uint32_t)p.groups;
    row = r, group = (int)(u - r * (uint32_t)p.groups);
  } else {
    row = unit / p.groups, group = (int)(unit % p.groups);
  }
  const int64_t c0 = (int64_t)group * p.size;
  H hx, hg;
  const T *src = (const T *)p.x.p + row_offset(p.x, p.n1, row, p.rows) + c0;
  hx.load(src, t, p.size);
  if (p.gate.p) hg.load((const T *)p.gate.p + row_offset(p.gate, p.n1, row, p.rows) + c0, t, p.size);
  // Everything is taken from the group's first value on: a large common part
  // then costs the mean and the differences no digits, and equal values give 0.
  const float pivot = to_f32(*src);
  float x[NV][8];
  hx.get(x);
  const float inv = 1.f / (float)p.size;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[i][e] = H::column(t, i, e) < p.size ? x[i][e] - pivot : 0.f;
      sum += x[i][e];
    }
  const float mean = group_sum<TPR>(sum, slot) * inv;
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[i][e] = H::column(t, i, e) < p.size ? x[i][e] - mean : 0.f;
      sq = fmaf(x[i][e], x[i][e], sq);
    }
  const float rstd = 1.f / sqrtf(fmaf(group_sum<TPR>(sq, slot), inv, p.eps));
  if (p.stats && live && t == 0) *(float2 *)(p.stats + 2 * unit) = make_float2(pivot + mean, rstd);
  float w[NV][8], b[NV][8];
  load_affine<TPR, NV, kPacked>(w, p.weight, p.weight_dtype, 1.f, c0, t, p.size);
  load_affine<TPR, NV, kPacked>(b, p.bias, p.weight_dtype, 0.f, c0, t, p.size);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) x[i][e] = fmaf(x[i][e] * rstd, w[i][e], b[i][e]);
  if (p.gate.p) {
    float g[NV][8];
    hg.get(g);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[i][e] *= p.silu ? g[i][e] * sigmoid_of<T>(g[i][e]) : g[i][e];
  } else if (p.silu) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) x[i][e] *= sigmoid_of<T>(x[i][e]);
  }
  if (live) H::store(x, (T *)p.out + row * p.groups * p.size + c0, t, p.size);
}

// How a gradient CTA's groups of threads ("lanes") lie over a row's groups and
// the rows: `across` groups, threads / TPR / across rows at a time.
struct Lanes {
  int across, rows, columns;  // columns: CTAs along a row's groups
};

template <typename T, int TPR, int NV, bool kPacked>
__global__ void __launch_bounds__(threads_for(TPR)) group_norm_bwd_kernel(const GroupNormCall p,
                                                                        const Lanes lanes) {
  using H = Held<T, TPR, NV, kPacked>;
  __shared__ float2 slot[32];
  extern __shared__ float joined[];  // (rows - 1, across, 2, size) with several rows
  column_sum_may_start();
  const int t = threadIdx.x % TPR, lane = threadIdx.x / TPR;
  const int group = blockIdx.x % lanes.columns * lanes.across + lane % lanes.across;
  const int lane_row = lane / lanes.across;
  const bool member = group < p.groups && lane_row < lanes.rows;
  const int64_t c0 = member ? (int64_t)group * p.size : 0;
  float w[NV][8], b[NV][8], dw[NV][8] = {}, db[NV][8] = {};
  load_affine<TPR, NV, kPacked>(w, p.weight, p.weight_dtype, 1.f, c0, t, p.size);
  load_affine<TPR, NV, kPacked>(b, p.bias, p.weight_dtype, 0.f, c0, t, p.size);
  const float inv = 1.f / (float)p.size;
  const int64_t ctas = gridDim.x / lanes.columns, cta = blockIdx.x / lanes.columns;
  const int64_t stride = ctas * lanes.rows;
  for (int64_t first = cta * lanes.rows; first < p.rows; first += stride) {
    const int64_t mine = first + lane_row;
    const bool live = member && mine < p.rows;
    const int64_t row = live ? mine : first;  // others redo a row, unstored
    H hx, hd, hg;
    hx.load((const T *)p.x.p + row_offset(p.x, p.n1, row, p.rows) + c0, t, p.size);
    hd.load((const T *)p.d_out.p + row_offset(p.d_out, p.n1, row, p.rows) + c0, t, p.size);
    if (p.gate.p)
      hg.load((const T *)p.gate.p + row_offset(p.gate, p.n1, row, p.rows) + c0, t, p.size);
    const float2 st = *(const float2 *)(p.stats + 2 * (row * p.groups + (member ? group : 0)));
    float n[NV][8], g[NV][8];
    hx.get(n);
    hd.get(g);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        n[i][e] = H::column(t, i, e) < p.size ? (n[i][e] - st.x) * st.y : 0.f;
    if (p.gate.p) {
      float u[NV][8];
      hg.get(u);
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float z = fmaf(n[i][e], w[i][e], b[i][e]);
          if (p.silu) {
            const float s = sigmoid_of<T>(u[i][e]);
            const float dz = g[i][e] * z;
            g[i][e] *= u[i][e] * s;
            u[i][e] = dz * s * fmaf(u[i][e], 1.f - s, 1.f);
          } else {
            const float dz = g[i][e] * z;
            g[i][e] *= u[i][e];
            u[i][e] = dz;
          }
        }
      if (live) H::store(u, (T *)p.d_gate + row * p.groups * p.size + c0, t, p.size);
    } else if (p.silu) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float z = fmaf(n[i][e], w[i][e], b[i][e]), s = sigmoid_of<T>(z);
          g[i][e] *= s * fmaf(z, 1.f - s, 1.f);
        }
    }
    float2 sums = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (live) {
          dw[i][e] = fmaf(g[i][e], n[i][e], dw[i][e]);
          db[i][e] += g[i][e];
        }
        g[i][e] *= w[i][e];
        sums.x += g[i][e];
        sums.y = fmaf(g[i][e], n[i][e], sums.y);
      }
    sums = group_sum<TPR>(sums, slot);
    sums.x *= inv, sums.y *= inv;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) g[i][e] = st.y * (g[i][e] - sums.x - n[i][e] * sums.y);
    if (live) H::store(g, (T *)p.dx + row * p.groups * p.size + c0, t, p.size);
  }
  if (!p.partial) return;
  // over the row lanes, in their order
  const int at = lane % lanes.across * 2 * p.size;
  const int wide = lanes.across * 2 * p.size;
  if (lanes.rows > 1) {
    if (member && lane_row > 0) {
      float *dst = joined + (int64_t)(lane_row - 1) * wide + at;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int c = H::column(t, i, e);
          if (c < p.size) dst[c] = dw[i][e], dst[p.size + c] = db[i][e];
        }
    }
    __syncthreads();
  }
  if (!member || lane_row > 0) return;
  const int64_t channels = (int64_t)p.groups * p.size;
  float *out = p.partial + cta * 2 * channels + c0;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = H::column(t, i, e);
      if (c >= p.size) continue;
      for (int r = 0; r < lanes.rows - 1; ++r) {
        dw[i][e] += joined[(int64_t)r * wide + at + c];
        db[i][e] += joined[(int64_t)r * wide + at + p.size + c];
      }
      out[c] = dw[i][e];
      out[channels + c] = db[i][e];
    }
}

// Threads per group and packs per thread for a group's size: enough that a
// group's loads are few per thread, within one warp while that leaves at most 4.
template <class F>
int by_size(const GroupNormCall &p, bool packed, F &&f) {
  const int d = p.size;
  if (!packed) {
    if (d <= 32) return f.template run<4, 1, false>();
    if (d <= 64) return f.template run<8, 1, false>();
    if (d <= 256) return f.template run<32, 1, false>();
    if (d <= 1024) return f.template run<128, 1, false>();
    if (d <= 4096) return f.template run<256, 2, false>();
    return f.template run<512, 2, false>();
  }
  if (d <= 16) return f.template run<2, 1, true>();
  if (d <= 32) return f.template run<4, 1, true>();
  if (d <= 64) return f.template run<8, 1, true>();
  if (d <= 128) return f.template run<16, 1, true>();
  if (d <= 256) return f.template run<32, 1, true>();
  if (d <= 512) return f.template run<32, 2, true>();
  if (d <= 1024) return f.template run<128, 1, true>();
  if (d <= 2048) return f.template run<256, 1, true>();
  if (d <= 4096) return f.template run<256, 2, true>();
  return f.template run<512, 2, true>();
}

constexpr int kBwdPerSm = 8;

// Whether every group of a tensor starts at 16 bytes.
bool packed_rows(const RowView &v, int size) {
  const int64_t pack = 16 / size;
  return !v.p || (((uintptr_t)v.p & 15) == 0 && v.s0 % pack == 0 && v.s1 % pack == 0);
}
bool at16(const void *p) { return ((uintptr_t)p & 15) == 0; }

template <typename T>
struct FwdLaunch {
  const GroupNormCall &p;
  cudaStream_t s;
  template <int TPR, int NV, bool kPacked>
  int run() {
    constexpr int per = threads_for(TPR) / TPR;
    const int64_t units = p.rows * p.groups, grid = (units + per - 1) / per;
    if (grid > INT32_MAX) return LA_ERR_UNSUPPORTED;
    group_norm_fwd_kernel<T, TPR, NV, kPacked><<<(unsigned)grid, threads_for(TPR), 0, s>>>(p);
    return check_launch();
  }
};

template <typename T>
struct BwdLaunch {
  const GroupNormCall &p;
  int sm_count;
  int64_t *partial_rows;
  cudaStream_t s;
  template <int TPR, int NV, bool kPacked>
  int run() {
    constexpr int per = threads_for(TPR) / TPR;
    auto kernel = group_norm_bwd_kernel<T, TPR, NV, kPacked>;
    Lanes l;
    l.columns = (p.groups + per - 1) / per;
    l.across = (p.groups + l.columns - 1) / l.columns;
    l.rows = per / l.across;
    const int smem = p.partial ? (l.rows - 1) * l.across * 2 * p.size * 4 : 0;  // at most 28 KB
    // one wave of CTAs, each walking many rows
    static const int per_sm = [&] {
      int n = 0;
      if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads_for(TPR), 16 * 1024) !=
          cudaSuccess) {
        cudaGetLastError();
        n = 2;
      }
      return n < 1 ? 1 : n > kBwdPerSm ? kBwdPerSm : n;
    }();
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
  return min64(rows, (int64_t)sm_count * kBwdPerSm);
}

int launch_group_norm_fwd(const GroupNormCall &p, int dtype, cudaStream_t s) {
  const int size = dtype == LA_DTYPE_FLOAT32 ? 4 : 2;
  const bool packed = p.size % 8 == 0 && packed_rows(p.x, size) && packed_rows(p.gate, size) &&
                      at16(p.weight) && at16(p.bias) && at16(p.out);
  if (dtype == LA_DTYPE_FLOAT32) return by_size(p, packed, FwdLaunch<float>{p, s});
  return by_size(p, packed, FwdLaunch<__nv_bfloat16>{p, s});
}

int launch_group_norm_bwd(const GroupNormCall &p, int dtype, int sm_count, int64_t *partial_rows,
                          cudaStream_t s) {
  const int size = dtype == LA_DTYPE_FLOAT32 ? 4 : 2;
  const bool packed = p.size % 8 == 0 && packed_rows(p.x, size) && packed_rows(p.gate, size) &&
                      packed_rows(p.d_out, size) && at16(p.weight) && at16(p.bias) && at16(p.dx) &&
                      at16(p.d_gate);
  if (dtype == LA_DTYPE_FLOAT32)
    return by_size(p, packed, BwdLaunch<float>{p, sm_count, partial_rows, s});
  return by_size(p, packed, BwdLaunch<__nv_bfloat16>{p, sm_count, partial_rows, s});
}

}  // namespace la
