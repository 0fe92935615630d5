// Root-mean-square norm with the residual's addition, its gradient, and the
// form whose output is held in e4m3 with fp32 scales.
//
//   s = x + r,   y = s * rstd * w,   rstd = 1 / sqrt(mean(s^2) + eps)
//   ds = rstd * (w dy - s rstd^2 mean(w dy s)) + d_sum,   dw = sum_rows dy s rstd
//   fp8: scale = max(amax |y|, 2^-96) / 448 over a row or a group, e4m3(y / scale)
//
// All of it is bound by memory.  A row is held in registers by `TPR` threads
// (8 per row of 64 up to a whole CTA), `NV` packs of 8 elements each, loaded
// once with 16-byte loads; the statistics are fp32 sums over shuffles (and
// shared memory where a row spans warps).  The gradient's CTAs walk the rows
// with a fixed set of columns per thread, so dw is summed in registers, then
// over the CTA's row lanes, and a second kernel adds the CTAs' partial rows in
// a fixed order: no atomics, the same bits every time.  It works on the saved
// sum, which is rounded to the inputs' type (half a step: 2^-8 in bf16).
//
// Measured in a CUDA graph over inputs larger than L2, bf16 with a residual and two
// upstream gradients, of the copy rate (6.5 TB/s; the last of the output is still in
// L2): 16384 x 1024 in 24 us (86%), its gradient 28 (75%); 32768 x 4096 in 159
// (104%), to e4m3 158 (91%), gradient 176 (94%); 131072 rows of 64 in 14.7 us (70%),
// gradient 18.8 (55%); 4096 x 16384 in 90 us (92%), gradient 150 (55%: 64 registers
// a thread spill 268 bytes); 16384 x 1023 (shifted) in 63 us, gradient 92.  fp32:
// 16384 x 4096 in 160 us, to e4m3 128, gradient 175 (94%); 4096 x 16384 in 170,
// gradient 350 (47%).
#include <cuda_fp8.h>
#include <math.h>

#include "common.cuh"
#include "tc_common.cuh"

namespace la {
namespace {

constexpr float kE4m3Max = 448.f;
constexpr float kAmaxMin = 1.f / 79228162514264337593543950336.f;  // 2^-96
constexpr int64_t kMaxWidth = 16384;

// Rows of a tensor with up to three leading dimensions (strides in elements)
// and a dense last one.
struct Rows {
  const void *p;
  int64_t s0, s1, s2;
};
struct Shape {
  int64_t rows;
  uint32_t n1, n2;  // the two inner leading dimensions
};

__device__ __forceinline__ int64_t row_offset(const Rows &t, const Shape &sh, int64_t row) {
  if (sh.n2 == sh.rows) return row * t.s2;
  if (sh.rows <= UINT32_MAX) {  // 32-bit divisions
    const uint32_t r = (uint32_t)row, outer = r / sh.n2;
    return (int64_t)(outer / sh.n1) * t.s0 + (int64_t)(outer % sh.n1) * t.s1 +
           (int64_t)(r % sh.n2) * t.s2;
  }
  const int64_t outer = row / sh.n2;
  return (outer / sh.n1) * t.s0 + (outer % sh.n1) * t.s1 + (row % sh.n2) * t.s2;
}

// How a row is accessed: single elements (any strides); packs of 8 neighbours by
// 16 bytes (rows that start at 16 bytes, d a multiple of 8); or, for contiguous
// rows of any other width, packs of the memory the row lies in: the first pack
// starts up to 7 elements before the row, and the row's two edge packs are
// accessed element by element.
enum Access { kSingle, kPacked, kShifted };

// Elements from the 16-byte boundary before a contiguous row to the row.
template <typename T, Access kA>
__device__ __forceinline__ int row_shift(int64_t row, int d) {
  return kA == kShifted ? (int)((row * d) & (16 / (int)sizeof(T) - 1)) : 0;
}

// Column of element e of pack i of thread t.
template <int TPR, Access kA>
__device__ __forceinline__ int column(int t, int i, int e, int shift) {
  return kA == kSingle ? (i * 8 + e) * TPR + t : (i * TPR + t) * 8 + e - shift;
}
__device__ __forceinline__ bool inside(int c, int d) { return (unsigned)c < (unsigned)d; }
// Whether the whole pack at column c is the row's.
template <Access kA>
__device__ __forceinline__ bool whole_pack(int c, int d) {
  return kA == kPacked ? c < d : kA == kShifted && c >= 0 && c + 8 <= d;
}

__device__ __forceinline__ void unpack(const uint4 &w, float (&x)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[2 * e] = __uint_as_float(u[e] << 16);
    x[2 * e + 1] = __uint_as_float(u[e] & 0xFFFF0000u);
  }
}

template <typename T, int TPR, int NV, Access kA>
__device__ __forceinline__ void load_row(float (&x)[NV][8], const T *p, int t, int d, int shift) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = column<TPR, kA>(t, i, 0, shift);
    if (whole_pack<kA>(c, d)) {
      if constexpr (sizeof(T) == 2) {
        unpack(*(const uint4 *)(p + c), x[i]);
      } else {
        const float4 a = *(const float4 *)(p + c), b = *(const float4 *)(p + c + 4);
        x[i][0] = a.x; x[i][1] = a.y; x[i][2] = a.z; x[i][3] = a.w;
        x[i][4] = b.x; x[i][5] = b.y; x[i][6] = b.z; x[i][7] = b.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int ce = column<TPR, kA>(t, i, e, shift);
        x[i][e] = kA != kPacked && inside(ce, d) ? to_f32(p[ce]) : 0.f;
      }
    }
  }
}

template <typename T, int TPR, int NV, Access kA>
__device__ __forceinline__ void store_row(const float (&x)[NV][8], T *p, int t, int d, int shift) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = column<TPR, kA>(t, i, 0, shift);
    if (whole_pack<kA>(c, d)) {
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
    } else if constexpr (kA != kPacked) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int ce = column<TPR, kA>(t, i, e, shift);
        if (inside(ce, d)) p[ce] = from_f32<T>(x[i][e]);
      }
    }
  }
}

// The weight row (fp32 or bf16; null: ones), which starts at 16 bytes whatever
// the other rows do: by elements where their packs are shifted.
template <typename TW, int TPR, int NV, Access kA>
__device__ __forceinline__ void load_weight_as(float (&w)[NV][8], const TW *p, int t, int d,
                                               int shift) {
  if constexpr (kA == kShifted) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = column<TPR, kA>(t, i, e, shift);
        w[i][e] = inside(c, d) ? to_f32(p[c]) : 0.f;
      }
  } else {
    load_row<TW, TPR, NV, kA>(w, p, t, d, 0);
  }
}
template <int TPR, int NV, Access kA>
__device__ __forceinline__ void load_weight(float (&w)[NV][8], const void *p, int dtype, int t,
                                            int d, int shift) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) w[i][e] = 1.f;
  } else if (dtype == LA_DTYPE_FLOAT32) {
    load_weight_as<float, TPR, NV, kA>(w, (const float *)p, t, d, shift);
  } else {
    load_weight_as<__nv_bfloat16, TPR, NV, kA>(w, (const __nv_bfloat16 *)p, t, d, shift);
  }
}

// A row as it is loaded, ahead of its use: bf16 packs stay packed.
template <typename T, int NV, Access kA>
struct Held {
  float x[NV][8];
  template <int TPR>
  __device__ __forceinline__ void load(const T *p, int t, int d, int shift) {
    load_row<T, TPR, NV, kA>(x, p, t, d, shift);
  }
  __device__ __forceinline__ void get(float (&y)[NV][8]) const {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) y[i][e] = x[i][e];
  }
};
template <int NV, Access kA>
struct HeldPacks {
  uint4 x[NV];
  template <int TPR>
  __device__ __forceinline__ void load(const __nv_bfloat16 *p, int t, int d, int shift) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = column<TPR, kA>(t, i, 0, shift);
      x[i] = make_uint4(0, 0, 0, 0);
      if (whole_pack<kA>(c, d)) {
        x[i] = *(const uint4 *)(p + c);
      } else if (kA == kShifted && c > -8 && c < d) {
        const uint16_t *q = (const uint16_t *)p;
        auto two = [&](int e) {
          const uint32_t lo = inside(c + e, d) ? q[c + e] : 0;
          return lo | (inside(c + e + 1, d) ? (uint32_t)q[c + e + 1] << 16 : 0);
        };
        x[i] = make_uint4(two(0), two(2), two(4), two(6));
      }
    }
  }
  __device__ __forceinline__ void get(float (&y)[NV][8]) const {
#pragma unroll
    for (int i = 0; i < NV; ++i) unpack(x[i], y[i]);
  }
};
template <int NV>
struct Held<__nv_bfloat16, NV, kPacked> : HeldPacks<NV, kPacked> {};
template <int NV>
struct Held<__nv_bfloat16, NV, kShifted> : HeldPacks<NV, kShifted> {};

struct Add {
  static __device__ __forceinline__ float zero() { return 0.f; }
  static __device__ __forceinline__ float of(float a, float b) { return a + b; }
};
// The larger of two values; a NaN stays.
struct Max {
  static __device__ __forceinline__ float zero() { return 0.f; }
  static __device__ __forceinline__ float of(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
  }
};

// Over the TPR threads of a row; every thread gets the result.  `slot`: shared
// memory for the warps of a row, one per warp of the CTA.  With TPR > 32 the
// CTA holds whole rows and every thread takes part.
template <int TPR, class Op>
__device__ __forceinline__ float reduce_row(float x, float *slot) {
#pragma unroll
  for (int m = 1; m < (TPR < 32 ? TPR : 32); m <<= 1)
    x = Op::of(x, __shfl_xor_sync(0xffffffffu, x, m));
  if constexpr (TPR > 32) {
    constexpr int kWarps = TPR / 32;
    const int warp = threadIdx.x >> 5;
    __syncthreads();  // the slots of the use before are read
    if ((threadIdx.x & 31) == 0) slot[warp] = x;
    __syncthreads();
    const int first = warp / kWarps * kWarps;
    x = Op::zero();
#pragma unroll
    for (int i = 0; i < kWarps; ++i) x = Op::of(x, slot[first + i]);
  }
  return x;
}

// Threads of a CTA.  Forward: one row per CTA from 128 threads a row on, so that
// no row waits at another's barrier; gradient: at least 256, fewer partial rows.
constexpr int fwd_threads(int tpr) { return tpr >= 128 ? tpr : 256; }
constexpr int bwd_threads(int tpr) { return tpr > 256 ? tpr : 256; }
// Forward rows of several packs a thread fetch the weight (from the caches) behind
// the sum of squares instead of holding it over it, and packed ones are kept to 64
// registers (80 in fp32, which spills more), so that more rows are on their way (0: no
// limit, better for 32 threads a row in the plain form).  32768 x 4096 in 164 -> 158 us,
// to e4m3 189 -> 155 us, 167 with 80 registers; 16384 x 4096 in fp32 164 -> 160 and 138
// -> 130, 143 with 64.  With one pack a thread the later fetch costs more (131072 x 128
// in 25.5 -> 27.3).
constexpr bool fwd_late_weight(int tpr, int nv) { return nv > 1 && tpr < 1024; }
constexpr int fwd_per_sm(int tpr, int nv, Access a, bool fp8, int size) {
  return a == kPacked && fwd_late_weight(tpr, nv) && (fp8 || tpr > 32)
             ? (size == 2 ? 1024 : 768) / fwd_threads(tpr) : 0;
}

struct NormFwd {
  Rows x, r;              // r.p null: no residual
  const void *weight;     // null: ones
  int weight_dtype;
  void *y;                // output (T, or e4m3), contiguous rows
  void *sum;              // null, or x + r, contiguous rows
  float *rstd;            // null, or one per row
  float *scales;          // fp8: (rows, d / group)
  Shape sh;
  int d;
  int group_log2;         // fp8: -1 for one scale per row, else log2 of the group
  float eps, inv_d;
};

template <typename T, int TPR, int NV, Access kA, bool kFp8>
__global__ void __launch_bounds__(fwd_threads(TPR), fwd_per_sm(TPR, NV, kA, kFp8, sizeof(T)))
rms_norm_fwd_kernel(const NormFwd p) {
  constexpr int kRowsPer = fwd_threads(TPR) / TPR;
  __shared__ float slot[32];
  __shared__ float slot_max[32];
  const int t = threadIdx.x % TPR;
  const int64_t row0 = (int64_t)blockIdx.x * kRowsPer + threadIdx.x / TPR;
  const bool live = row0 < p.sh.rows;
  const int64_t row = live ? row0 : p.sh.rows - 1;  // idle lanes redo the last row, unstored
  const int shift = row_shift<T, kA>(row, p.d);
  float s[NV][8];
  load_row<T, TPR, NV, kA>(s, (const T *)p.x.p + row_offset(p.x, p.sh, row), t, p.d, shift);
  if (p.r.p) {
    float r[NV][8];
    load_row<T, TPR, NV, kA>(r, (const T *)p.r.p + row_offset(p.r, p.sh, row), t, p.d, shift);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) s[i][e] += r[i][e];
  }
  float w[NV][8];
  if (!fwd_late_weight(TPR, NV)) load_weight<TPR, NV, kA>(w, p.weight, p.weight_dtype, t, p.d, shift);
  if (p.sum && live) store_row<T, TPR, NV, kA>(s, (T *)p.sum + row * p.d, t, p.d, shift);
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) sq = fmaf(s[i][e], s[i][e], sq);
  sq = reduce_row<TPR, Add>(sq, slot);
  const float rstd = 1.f / sqrtf(fmaf(sq, p.inv_d, p.eps));
  if (p.rstd && live && t == 0) p.rstd[row] = rstd;
  if (fwd_late_weight(TPR, NV)) load_weight<TPR, NV, kA>(w, p.weight, p.weight_dtype, t, p.d, shift);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) s[i][e] = s[i][e] * rstd * w[i][e];
  if constexpr (!kFp8) {
    if (live) store_row<T, TPR, NV, kA>(s, (T *)p.y + row * p.d, t, p.d, shift);
  } else {
    float m[NV], all = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {  // (columns beyond d are zero)
      m[i] = fabsf(s[i][0]);
#pragma unroll
      for (int e = 1; e < 8; ++e) m[i] = Max::of(m[i], fabsf(s[i][e]));
      all = Max::of(all, m[i]);
    }
    const bool whole = p.group_log2 < 0;
    if (whole) {
      all = reduce_row<TPR, Max>(all, slot_max);
#pragma unroll
      for (int i = 0; i < NV; ++i) m[i] = all;
    } else {  // a group is group / 8 neighbouring lanes of one pack (packed rows only)
      const int lanes = 1 << (p.group_log2 - 3);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        for (int x = 1; x < lanes; x <<= 1)
          m[i] = Max::of(m[i], __shfl_xor_sync(0xffffffffu, m[i], x));
    }
    uint8_t *y = (uint8_t *)p.y + row * p.d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = column<TPR, kA>(t, i, 0, shift);
      const float scale = Max::of(m[i], kAmaxMin) * (1.f / kE4m3Max);
      // one division per group: y * (1 / scale) is within an ulp of y / scale
      // ahead of the rounding to 4 bits
      const float inv = 1.f / scale;
      if (whole) {
        if (live && t == 0 && i == 0) p.scales[row] = scale;
      } else if (live && c < p.d && (c & ((1 << p.group_log2) - 1)) == 0) {
        p.scales[row * (p.d >> p.group_log2) + (c >> p.group_log2)] = scale;
      }
      uint16_t q[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        q[e] = __nv_cvt_float2_to_fp8x2(make_float2(s[i][2 * e] * inv, s[i][2 * e + 1] * inv),
                                        __NV_SATFINITE, __NV_E4M3);
      if (!live) continue;
      if (whole_pack<kA>(c, p.d)) {
        const uint2 u = make_uint2(q[0] | ((uint32_t)q[1] << 16), q[2] | ((uint32_t)q[3] << 16));
        if constexpr (kA == kPacked || sizeof(T) == 2) {
          *(uint2 *)(y + c) = u;
        } else {  // packs of 8 at a multiple of 4 values
          *(uint32_t *)(y + c) = u.x;
          *(uint32_t *)(y + c + 4) = u.y;
        }
      } else if constexpr (kA != kPacked) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int ce = column<TPR, kA>(t, i, e, shift);
          if (inside(ce, p.d)) y[ce] = (uint8_t)(q[e / 2] >> (8 * (e & 1)));
        }
      }
    }
  }
}

struct NormBwd {
  Rows s, dy, dsum;     // s: the normed rows (x + r); dsum.p null: none
  const void *weight;     // null: ones
  int weight_dtype;
  const float *rstd;
  void *ds;             // contiguous rows
  float *partial;       // null (no dw), or (gridDim.x, d)
  Shape sh;
  int d;
  float inv_d;
};

template <typename T, int TPR, int NV, Access kA>
__global__ void __launch_bounds__(bwd_threads(TPR))
rms_norm_bwd_kernel(const NormBwd p) {
  constexpr int kThreads = bwd_threads(TPR);
  constexpr int kRowsPer = kThreads / TPR;
  __shared__ float slot[32];
  extern __shared__ float lanes_dw[];  // (kRowsPer - 1, d) with kRowsPer > 1
  tc::grid_dependents_launch();        // the sum of dw waits for all of this grid
  const int t = threadIdx.x % TPR, lane_row = threadIdx.x / TPR;
  float w[NV][8], dw[NV][8] = {};
  // the rows of a row lane are a multiple of 8 apart where their packs are
  // shifted, so that its columns stay the same
  const int shift = row_shift<T, kA>((int64_t)blockIdx.x * kRowsPer + lane_row, p.d);
  load_weight<TPR, NV, kA>(w, p.weight, p.weight_dtype, t, p.d, shift);
  // The next row is loaded before this one's sum over the row's threads (not
  // where 1024 threads leave 64 registers each).
  constexpr bool kAhead = TPR < 1024;
  Held<T, NV, kA> hs, hg, ha;
  float rstd_next = 0.f;
  const int64_t stride = (int64_t)gridDim.x * kRowsPer;
  auto fetch = [&](int64_t first) {
    // idle lanes redo the last row, unstored; shifted, a row of their own shift
    int64_t row = first + lane_row;
    const int d = kA == kShifted && row >= p.sh.rows ? 0 : p.d;
    row = min64(row, p.sh.rows - 1);
    hs.template load<TPR>((const T *)p.s.p + row_offset(p.s, p.sh, row), t, d, shift);
    hg.template load<TPR>((const T *)p.dy.p + row_offset(p.dy, p.sh, row), t, d, shift);
    if (p.dsum.p)
      ha.template load<TPR>((const T *)p.dsum.p + row_offset(p.dsum, p.sh, row), t, d, shift);
    rstd_next = p.rstd[row];
  };
  if (kAhead) fetch((int64_t)blockIdx.x * kRowsPer);
  for (int64_t first = (int64_t)blockIdx.x * kRowsPer; first < p.sh.rows; first += stride) {
    const int64_t row = first + lane_row;
    const bool live = row < p.sh.rows;
    if (!kAhead) fetch(first);
    float s[NV][8], g[NV][8], a[NV][8];
    hs.get(s);
    hg.get(g);
    if (p.dsum.p) ha.get(a);
    const float rstd = rstd_next;
    if (kAhead && first + stride < p.sh.rows) fetch(first + stride);
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (live) dw[i][e] = fmaf(g[i][e] * s[i][e], rstd, dw[i][e]);
        g[i][e] *= w[i][e];
        dot = fmaf(g[i][e], s[i][e], dot);
      }
    dot = reduce_row<TPR, Add>(dot, slot) * p.inv_d;
    const float c = rstd * rstd * dot;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) g[i][e] = rstd * (g[i][e] - s[i][e] * c);
    if (p.dsum.p) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) g[i][e] += a[i][e];
    }
    if (live) store_row<T, TPR, NV, kA>(g, (T *)p.ds + row * p.d, t, p.d, shift);
  }
  if (!p.partial) return;
  if constexpr (kRowsPer > 1) {
    if (lane_row > 0) {
      float *dst = lanes_dw + (int64_t)(lane_row - 1) * p.d;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int c = column<TPR, kA>(t, i, e, shift);
          if (inside(c, p.d)) dst[c] = dw[i][e];
        }
    }
    __syncthreads();
  }
  float *dst = p.partial + (int64_t)blockIdx.x * p.d;
  for (int c = threadIdx.x; kRowsPer > 1 && c < p.d; c += kThreads) {
    float sum = 0.f;
    for (int r = 0; r < kRowsPer - 1; ++r) sum += lanes_dw[(int64_t)r * p.d + c];
    lanes_dw[c] = sum;  // read by the first row lane below
  }
  if constexpr (kRowsPer > 1) __syncthreads();
  if (lane_row == 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = column<TPR, kA>(t, i, e, shift);
        if (inside(c, p.d)) dst[c] = dw[i][e] + (kRowsPer > 1 ? lanes_dw[c] : 0.f);
      }
  }
}

// dw = sum of the partial rows: 32 columns x 32 row lanes per CTA.
template <typename TW>
__global__ void __launch_bounds__(1024)
rms_norm_dw_kernel(const float *partial, int rows, int d, TW *dw) {
  __shared__ float part[32][33];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), lane = threadIdx.x >> 5;
  tc::grid_dependency_wait();  // launched behind the kernel that writes the rows
  float sum = 0.f;
  if (c < d) {
#pragma unroll 8
    for (int r = lane; r < rows; r += 32) sum += partial[(int64_t)r * d + c];
  }
  part[lane][threadIdx.x & 31] = sum;
  __syncthreads();
  // warp w adds column w over the row lanes
  sum = part[threadIdx.x & 31][lane];
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
  if ((threadIdx.x & 31) == 0 && blockIdx.x * 32 + lane < d)
    dw[blockIdx.x * 32 + lane] = from_f32<TW>(sum);
}

template <typename TW>
int launch_dw(const float *partial, int rows, int d, void *dw, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((d + 31) / 32));
  cfg.blockDim = dim3(1024);
  cfg.stream = s;
  cudaLaunchAttribute pdl;
  pdl.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &pdl;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, rms_norm_dw_kernel<TW>, partial, rows, d, (TW *)dw);
  return check_launch();
}

// The threads per row and packs per thread for a width.  Few packs keep the
// registers low enough for many CTAs per SM, whose loads then cover one
// another's reductions.  Shifted and single-element rows take fewer variants.
template <class F>
int by_width_single(int64_t d, F &&f) {
  if (d <= 256) return f.template run<32, 1, kSingle>();
  if (d <= 1024) return f.template run<128, 1, kSingle>();
  if (d <= 4096) return f.template run<256, 2, kSingle>();
  return f.template run<1024, 2, kSingle>();
}
template <class F>
int by_width_shifted(int64_t d, F &&f) {  // one pack more than the row's own
  if (d + 8 <= 256) return f.template run<32, 1, kShifted>();
  if (d + 8 <= 1024) return f.template run<128, 1, kShifted>();
  if (d + 8 <= 2048) return f.template run<256, 1, kShifted>();
  if (d + 8 <= 4096) return f.template run<256, 2, kShifted>();
  if (d + 8 <= 8192) return f.template run<512, 2, kShifted>();
  return f.template run<1024, 2, kShifted>();
}
// Forward: rows of up to 1024 within one warp (32768 x 4096 with a residual, one
// row of 128 threads x 4 packs per CTA against 256 x 2: 164 and 171 us, to e4m3
// 188 and 196).
template <class F>
int by_width_fwd(int64_t d, Access access, F &&f) {
  if (access == kSingle) return by_width_single(d, f);
  if (access == kShifted) return by_width_shifted(d, f);
  if (d <= 64) return f.template run<8, 1, kPacked>();
  if (d <= 128) return f.template run<16, 1, kPacked>();
  if (d <= 256) return f.template run<32, 1, kPacked>();
  if (d <= 512) return f.template run<32, 2, kPacked>();
  // Rows that all fit the SMs at once with one pack a thread take that form, the
  // shortest way through a row: 8 / 1200 rows of 1024 to e4m3 2.9 / 3.9 us against
  // 4.2 / 5.2; 2400 rows 5.6 either way, 16384 rows 30 against 24.  (The sums of the
  // two forms are in other orders: a row's last bit may go by the number of rows.)
  const bool few = d <= 4096 && f.p.sh.rows * ((d + 1023) / 1024) <= f.sm_count * 8;
  if (d <= 1024) return few ? f.template run<128, 1, kPacked>() : f.template run<32, 4, kPacked>();
  if (d <= 2048) return few ? f.template run<256, 1, kPacked>() : f.template run<128, 2, kPacked>();
  if (d <= 4096) return few ? f.template run<512, 1, kPacked>() : f.template run<128, 4, kPacked>();
  if (d <= 8192) return f.template run<256, 4, kPacked>();
  return f.template run<512, 4, kPacked>();
}
// Gradient: it also holds w and the running dw.
template <class F>
int by_width_bwd(int64_t d, Access access, F &&f) {
  if (access == kSingle) return by_width_single(d, f);
  if (access == kShifted) return by_width_shifted(d, f);
  if (d <= 64) return f.template run<8, 1, kPacked>();
  if (d <= 128) return f.template run<16, 1, kPacked>();
  if (d <= 256) return f.template run<32, 1, kPacked>();
  if (d <= 512) return f.template run<32, 2, kPacked>();
  if (d <= 1024) return f.template run<64, 2, kPacked>();
  if (d <= 2048) return f.template run<128, 2, kPacked>();
  if (d <= 4096) return f.template run<128, 4, kPacked>();
  if (d <= 8192) return f.template run<512, 2, kPacked>();
  return f.template run<1024, 2, kPacked>();
}

// The gradient's CTAs walk the rows: this many per SM at most.
constexpr int kBwdPerSm = 8;

// One partial row of dw for each CTA, at most.
size_t partial_bytes(int64_t rows, int64_t d, int sm_count) {
  return (size_t)min64(rows, (int64_t)sm_count * kBwdPerSm) * (size_t)d * sizeof(float);
}

// Whether rows start at 16 bytes; whether they are contiguous from there on.
bool packed_rows(const Rows &t, int size) {
  const int64_t pack = 16 / size;
  return !t.p || (((uintptr_t)t.p & 15) == 0 && t.s0 % pack == 0 && t.s1 % pack == 0 &&
                  t.s2 % pack == 0);
}
bool plain_rows(const Rows &t, const Shape &sh, int64_t d) {
  return !t.p || (((uintptr_t)t.p & 15) == 0 && sh.n2 == sh.rows && t.s2 == d);
}
bool at16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// The access for inputs a, b, c and contiguous outputs u, v.
Access access_of(const Shape &sh, int64_t d, int dtype, const Rows &a, const Rows &b, const Rows &c,
                 const void *weight, const void *u, const void *v) {
  const int size = dtype == LA_DTYPE_FLOAT32 ? 4 : 2;
  if (!at16(u) || !at16(v)) return kSingle;
  if (d % 8 == 0 && at16(weight) && packed_rows(a, size) && packed_rows(b, size) &&
      packed_rows(c, size))
    return kPacked;
  if (d + 8 <= kMaxWidth && plain_rows(a, sh, d) && plain_rows(b, sh, d) && plain_rows(c, sh, d))
    return kShifted;
  return kSingle;
}

template <typename T, bool kFp8>
struct FwdLaunch {
  const NormFwd &p;
  int sm_count;
  cudaStream_t s;
  template <int TPR, int NV, Access kA>
  int run() {
    constexpr int per = fwd_threads(TPR) / TPR;
    const int64_t grid = (p.sh.rows + per - 1) / per;
    if (grid > INT32_MAX) return LA_ERR_UNSUPPORTED;
    rms_norm_fwd_kernel<T, TPR, NV, kA, kFp8><<<(unsigned)grid, fwd_threads(TPR), 0, s>>>(p);
    return check_launch();
  }
};

template <typename T>
struct BwdLaunch {
  const NormBwd &p;
  int sm_count;
  int *grid;
  cudaStream_t s;
  template <int TPR, int NV, Access kA>
  int run() {
    constexpr int per = bwd_threads(TPR) / TPR;
    // one wave of CTAs, each walking many rows
    static const int per_sm = [] {
      int n = 0;
      if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(
              &n, rms_norm_bwd_kernel<T, TPR, NV, kA>, bwd_threads(TPR), 28 * 1024) != cudaSuccess) {
        cudaGetLastError();
        n = 2;
      }
      return n < 1 ? 1 : n > kBwdPerSm ? kBwdPerSm : n;
    }();
    const int64_t groups = (p.sh.rows + per - 1) / per;
    *grid = (int)min64(groups, (int64_t)sm_count * per_sm);
    if (kA == kShifted && *grid < groups) *grid = *grid / 8 * 8;  // whole periods of the shift
    const int smem = p.partial ? (per - 1) * p.d * 4 : 0;  // at most 28 KB
    rms_norm_bwd_kernel<T, TPR, NV, kA><<<*grid, bwd_threads(TPR), smem, s>>>(p);
    return check_launch();
  }
};

bool valid_type(int t) { return t == LA_DTYPE_FLOAT32 || t == LA_DTYPE_BFLOAT16; }

// Checks what the entry points share; LA_OK with *empty set where there is
// nothing to do.
int check_norm(const int64_t *shape, int64_t d, int dtype, int weight_dtype, Shape *sh,
               bool *empty) {
  *empty = false;
  if (!shape || shape[0] < 0 || shape[1] < 0 || shape[2] < 0 || d < 1)
    return LA_ERR_INVALID_ARGUMENT;
  if (!valid_type(dtype) || !valid_type(weight_dtype)) return LA_ERR_INVALID_ARGUMENT;
  if (d > kMaxWidth) return LA_ERR_UNSUPPORTED;
  if (shape[0] == 0 || shape[1] == 0 || shape[2] == 0) {
    *empty = true;
    return LA_OK;
  }
  if (shape[1] > INT32_MAX || shape[2] > INT32_MAX) return LA_ERR_UNSUPPORTED;
  const int64_t inner = shape[1] * shape[2];
  if (inner > INT64_MAX / d / 8 / shape[0]) return LA_ERR_UNSUPPORTED;
  sh->rows = shape[0] * inner;
  sh->n1 = (uint32_t)shape[1];
  sh->n2 = (uint32_t)shape[2];
  DeviceInfo info;
  const int st = current_device_info(&info);
  if (st != LA_OK) return st;
  return info.cc_major == 10 ? LA_OK : LA_ERR_NO_DEVICE;
}

Rows rows_of(const void *p, const int64_t *s) {
  Rows r{p, 0, 0, 0};
  if (p && s) r.s0 = s[0], r.s1 = s[1], r.s2 = s[2];
  return r;
}

template <bool kFp8>
int launch_fwd(const NormFwd &p, int dtype, cudaStream_t s) {
  const Access access = access_of(p.sh, p.d, dtype, p.x, p.r, Rows{}, p.weight, p.y, p.sum);
  if (kFp8 && p.group_log2 >= 0 && access != kPacked) return LA_ERR_UNSUPPORTED;
  DeviceInfo info;
  const int st = current_device_info(&info);
  if (st != LA_OK) return st;
  if (dtype == LA_DTYPE_FLOAT32)
    return by_width_fwd(p.d, access, FwdLaunch<float, kFp8>{p, info.sm_count, s});
  return by_width_fwd(p.d, access, FwdLaunch<__nv_bfloat16, kFp8>{p, info.sm_count, s});
}

int launch_bwd(const NormBwd &p, int dtype, int sm_count, int *grid, cudaStream_t s) {
  const Access access =
      access_of(p.sh, p.d, dtype, p.s, p.dy, p.dsum, p.weight, p.ds, nullptr);
  if (dtype == LA_DTYPE_FLOAT32)
    return by_width_bwd(p.d, access, BwdLaunch<float>{p, sm_count, grid, s});
  return by_width_bwd(p.d, access, BwdLaunch<__nv_bfloat16>{p, sm_count, grid, s});
}

}  // namespace
}  // namespace la

using namespace la;

extern "C" {

int la_rms_norm_fwd(const void *x, const int64_t *x_strides, const void *residual,
                    const int64_t *residual_strides, const void *weight, void *y, void *sum,
                    float *rstd, const int64_t *shape, int64_t d, int dtype, int weight_dtype,
                    float eps, void *stream) {
  NormFwd p{};
  bool empty;
  const int st = check_norm(shape, d, dtype, weight_dtype, &p.sh, &empty);
  if (st != LA_OK || empty) return st;
  if (!x || !x_strides || !y || (residual && !residual_strides)) return LA_ERR_INVALID_ARGUMENT;
  p.x = rows_of(x, x_strides);
  p.r = rows_of(residual, residual_strides);
  p.weight = weight, p.weight_dtype = weight_dtype, p.y = y, p.sum = sum, p.rstd = rstd;
  p.d = (int)d;
  p.eps = eps;
  p.inv_d = 1.f / (float)d;
  return launch_fwd<false>(p, dtype, (cudaStream_t)stream);
}

int la_rms_norm_fp8(const void *x, const int64_t *x_strides, const void *residual,
                    const int64_t *residual_strides, const void *weight, void *y, float *scales,
                    void *sum, const int64_t *shape, int64_t d, int64_t group, int dtype,
                    int weight_dtype, float eps, void *stream) {
  NormFwd p{};
  bool empty;
  const int st = check_norm(shape, d, dtype, weight_dtype, &p.sh, &empty);
  if (st != LA_OK) return st;
  if (group != d && (group < 16 || group > 256 || (group & (group - 1)) || d % group))
    return LA_ERR_INVALID_ARGUMENT;
  if (empty) return LA_OK;
  if (!x || !x_strides || !y || !scales || (residual && !residual_strides))
    return LA_ERR_INVALID_ARGUMENT;
  p.x = rows_of(x, x_strides);
  p.r = rows_of(residual, residual_strides);
  p.weight = weight, p.weight_dtype = weight_dtype, p.y = y, p.sum = sum, p.scales = scales;
  p.d = (int)d;
  p.group_log2 = -1;
  for (int i = 4; group != d && i <= 8; ++i)
    if (group == (int64_t)1 << i) p.group_log2 = i;
  p.eps = eps;
  p.inv_d = 1.f / (float)d;
  return launch_fwd<true>(p, dtype, (cudaStream_t)stream);
}

int la_rms_norm_bwd_workspace_size(int64_t rows, int64_t d, size_t *bytes) {
  if (!bytes || rows < 0 || d < 1) return LA_ERR_INVALID_ARGUMENT;
  if (d > kMaxWidth) return LA_ERR_UNSUPPORTED;
  DeviceInfo info;
  const int st = current_device_info(&info);
  if (st != LA_OK) return st;
  *bytes = partial_bytes(rows, d, info.sm_count);
  return LA_OK;
}

int la_rms_norm_bwd(const void *s, const int64_t *s_strides, const void *weight, const void *d_y,
                    const int64_t *d_y_strides, const void *d_sum, const int64_t *d_sum_strides,
                    const float *rstd, void *d_s, void *d_weight, const int64_t *shape, int64_t d,
                    int dtype, int weight_dtype, void *workspace, size_t workspace_bytes,
                    void *stream) {
  NormBwd p{};
  bool empty;
  int st = check_norm(shape, d, dtype, weight_dtype, &p.sh, &empty);
  if (st != LA_OK) return st;
  cudaStream_t cs = (cudaStream_t)stream;
  if (empty) {
    if (!d_weight) return LA_OK;
    const size_t size = weight_dtype == LA_DTYPE_FLOAT32 ? 4 : 2;
    return cuda_status(cudaMemsetAsync(d_weight, 0, (size_t)d * size, cs));
  }
  if (!s || !s_strides || !d_y || !d_y_strides || !rstd || !d_s || (d_sum && !d_sum_strides))
    return LA_ERR_INVALID_ARGUMENT;
  DeviceInfo info;
  if ((st = current_device_info(&info)) != LA_OK) return st;
  if (d_weight && (!workspace || workspace_bytes < partial_bytes(p.sh.rows, d, info.sm_count) ||
                   ((uintptr_t)workspace & 15)))
    return LA_ERR_WORKSPACE;
  p.s = rows_of(s, s_strides);
  p.dy = rows_of(d_y, d_y_strides);
  p.dsum = rows_of(d_sum, d_sum_strides);
  p.weight = weight, p.weight_dtype = weight_dtype, p.rstd = rstd, p.ds = d_s;
  p.partial = d_weight ? (float *)workspace : nullptr;
  p.d = (int)d;
  p.inv_d = 1.f / (float)d;
  int grid = 0;
  st = launch_bwd(p, dtype, info.sm_count, &grid, cs);
  if (st != LA_OK || !d_weight) return st;
  if (weight_dtype == LA_DTYPE_FLOAT32) return launch_dw<float>(p.partial, grid, p.d, d_weight, cs);
  return launch_dw<__nv_bfloat16>(p.partial, grid, p.d, d_weight, cs);
}

}  // extern "C"
