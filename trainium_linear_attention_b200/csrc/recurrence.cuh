// Gated linear recurrence of each channel: what its kernels share.
//
//   h_t = a_t h_{t-1} + beta_t u_t x_t,   u = sigmoid(input gate), 1 without one
//   with a decay:   a = exp(lambda s), beta = sqrt(1 - a^2),   s = sigmoid(gate)
//   without:        a = s,             beta = 1 - s
//
// The kernels hold a - 1 instead of a: it keeps its relative accuracy where a
// rounds to 1, and beta = sqrt((a - 1)(-1 - a)) needs no difference of near
// numbers.
#pragma once

#include "common.cuh"
#include "tc_common.cuh"
#include "tma_host.cuh"

namespace la {

// A (batch, tokens, channels) tensor with a dense last dimension; strides in
// elements.
struct TokenView {
  const void *p = nullptr;
  int64_t sb = 0, st = 0;
};

struct RecurCall {
  TokenView x, gate, input_gate;     // input_gate.p null: none
  const float *log_decay = nullptr;  // null: a = sigmoid(gate)
  const float *init = nullptr;       // null, or (batch, channels)
  const void *lengths = nullptr;     // null, or one per sequence
  int lengths64 = 0;                 // int64 (else int32)
  int64_t batch = 0, tokens = 0;
  int channels = 0;
  bool pairs = false;                // channels are even and what is written starts at 8 bytes
  float *check = nullptr;            // null, or (batch, blocks of kRecurCheck tokens, channels):
                                     // the state before each block
  // forward
  void *out = nullptr;               // contiguous
  float *final_state = nullptr;      // null, or (batch, channels)
  // gradient
  TokenView d_out;
  const float *d_final = nullptr;    // null, or (batch, channels)
  void *dx = nullptr, *d_gate = nullptr, *d_input = nullptr;  // contiguous
  float *d_init = nullptr;           // null, or (batch, channels)
  float *partial = nullptr;          // rows of d_log_decay's sums, one per CTA of a channel group
};

// Tokens from one saved state to the next: those of a forward thread's step.
constexpr int kRecurCheck = 16;
constexpr int kRecurThreads = 256;
constexpr int kRecurMaxCluster = 8;

__device__ __forceinline__ int64_t recur_length(const void *lengths, int is64, int64_t b,
                                                int64_t tokens) {
  if (!lengths) return tokens;
  const int64_t n = is64 ? ((const int64_t *)lengths)[b] : ((const int32_t *)lengths)[b];
  return n < 0 ? 0 : n < tokens ? n : tokens;
}

// ---- two channels at a time ---------------------------------------------------
__device__ __forceinline__ float2 two(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 load_two(const __nv_bfloat16 *p) {
  const uint32_t w = *(const uint32_t *)p;
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ float2 load_two(const float *p) { return *(const float2 *)p; }

// Channels c and c + 1 of a row of n (the second may be beyond it); `pair`: the
// row's pairs are aligned.
__device__ __forceinline__ void store_two(__nv_bfloat16 *p, float2 v, bool pair, bool second) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(v.x, v.y);
  if (pair) {
    *(__nv_bfloat162 *)p = b;
  } else {
    p[0] = b.x;
    if (second) p[1] = b.y;
  }
}
__device__ __forceinline__ void store_two(float *p, float2 v, bool pair, bool second) {
  if (pair) {
    *(float2 *)p = v;
  } else {
    p[0] = v.x;
    if (second) p[1] = v.y;
  }
}

// Functions by the inputs' type: bf16 inputs are 2^-9 apart, and the special-
// function unit's 2^-22 is far below what they carry; fp32 ones take the library's.
template <typename T> struct Fn;
template <> struct Fn<__nv_bfloat16> {
  static __device__ __forceinline__ float exp(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
    return y;
  }
  static __device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
  }
  static __device__ __forceinline__ float rsqrt(float x) {
    float y;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
  }
};
template <> struct Fn<float> {
  static __device__ __forceinline__ float exp(float x) { return expf(x); }
  static __device__ __forceinline__ float rcp(float x) { return 1.f / x; }
  static __device__ __forceinline__ float rsqrt(float x) { return 1.f / sqrtf(x); }
};

// exp(z) - 1 for z <= 0, to a relative 2^-23: z = n ln 2 + f with |f| <= ln 2 / 2,
// exp(z) - 1 = 2^n (exp(f) - 1) + (2^n - 1), exp(f) - 1 = f + f^2 q(f).  q is the
// Chebyshev fit of degree 4 on that interval (1.2e-8 of exp(f) - 1).  On the
// FMA pipe: the special-function unit is as busy as memory without it.
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float2 expm1_neg(float2 z) {
  z.x = max_nan(z.x, -80.f);  // exp(-80) is far below half an ulp of 1
  z.y = max_nan(z.y, -80.f);
  const float2 magic = two(12582912.f);  // 1.5 * 2^23: the sum's low bits hold n
  const float2 t = __ffma2_rn(z, two(1.4426950408889634f), magic);
  const float2 n = __fadd2_rn(t, two(-12582912.f));
  // (ln 2 in one constant: n times its error is 2^-26 n, which 2^n makes small)
  const float2 f = __ffma2_rn(n, two(-0.69314718055994531f), z);
  float2 q = __ffma2_rn(two(0.0013933685841038823f), f, two(0.008369184099137783f));
  q = __ffma2_rn(q, f, two(0.041666463017463684f));
  q = __ffma2_rn(q, f, two(0.16666504740715027f));
  q = __ffma2_rn(q, f, two(0.5f));
  const float2 p = __ffma2_rn(__fmul2_rn(f, f), q, f);
  const float2 s = make_float2(__int_as_float(__float_as_int(t.x) * (1 << 23) + 0x3F800000),
                               __int_as_float(__float_as_int(t.y) * (1 << 23) + 0x3F800000));
  return __ffma2_rn(s, p, __fadd2_rn(s, two(-1.f)));
}

// The floor of 1 - a^2 under a root or a division, where it meets a zero.
constexpr float kBetaFloor = 1e-36f;
constexpr float kExpMost = 8.5070592e37f;  // 2^126, whose reciprocal is still normal

__device__ __forceinline__ float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float2 min_nan(float2 a, float b) {
  return make_float2(min_nan(a.x, b), min_nan(a.y, b));
}
__device__ __forceinline__ float2 max_nan(float2 a, float b) {
  return make_float2(max_nan(a.x, b), max_nan(a.y, b));
}
template <typename T> __device__ __forceinline__ float2 rcp_two(float2 x) {
  return make_float2(Fn<T>::rcp(x.x), Fn<T>::rcp(x.y));
}
template <typename T> __device__ __forceinline__ float2 rsqrt_two(float2 x) {
  return make_float2(Fn<T>::rsqrt(x.x), Fn<T>::rsqrt(x.y));
}
// exp(-x)
template <typename T> __device__ __forceinline__ float2 exp_minus(float2 x) {
  if constexpr (sizeof(T) == 2) {
    const float2 t = __fmul2_rn(x, two(-1.4426950408889634f));
    float2 y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y.x) : "f"(t.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y.y) : "f"(t.y));
    return y;
  } else {
    return make_float2(expf(-x.x), expf(-x.y));
  }
}

// What a token's gates come to, for two channels.
struct Token {
  float2 am1;  // a - 1
  float2 bu;   // beta u
  float2 s;    // sigmoid(gate)
  float2 sc;   // 1 - s and 1 - u, for the gradient (uc with an input gate)
  float2 uc;
};
// beta^2 = 1 - a^2 = (a - 1) (-1 - a), without a difference of near numbers, and
// the same with a floor.
__device__ __forceinline__ float2 beta_squared(float2 am1, float2 &floored) {
  const float2 n = __ffma2_rn(am1, two(-1.f), two(-2.f));
  floored = __ffma2_rn(am1, n, two(kBetaFloor));
  return __fmul2_rn(am1, n);
}
// A closed gate (s = 0; s = 1 without a decay) and a closed input gate (u = 0)
// give beta u = 0 to the bit, whatever the other is: a masked token changes
// nothing even where its x is the type's lowest value.
template <typename T, bool kDecay, bool kInput, bool kGrad>
__device__ __forceinline__ Token token_of(float2 g, float2 i, float2 lambda) {
  Token y;
  float2 eg = exp_minus<T>(g);
  if constexpr (!kDecay) eg = min_nan(eg, kExpMost);  // 1 - s = e s, and not inf * 0
  y.s = rcp_two<T>(__fadd2_rn(eg, two(1.f)));
  if constexpr (!kDecay) y.sc = __fmul2_rn(eg, y.s);
  else if constexpr (kGrad) y.sc = __fmul2_rn(min_nan(eg, kExpMost), y.s);
  float2 eu = two(0.f), pu = two(1.f), u = two(1.f);
  if constexpr (kInput) {
    eu = exp_minus<T>(i);
    pu = __fadd2_rn(eu, two(1.f));
    if constexpr (!kDecay || kGrad) u = rcp_two<T>(pu);
    if constexpr (kGrad) y.uc = __fmul2_rn(min_nan(eu, kExpMost), u);
  }
  if constexpr (kDecay) {
    y.am1 = expm1_neg(__fmul2_rn(lambda, y.s));
    float2 w;
    const float2 v = beta_squared(y.am1, w);
    if constexpr (kInput && !kGrad) {
      // one root for both: beta / p = beta^2 / sqrt(beta^2 p^2), p = 1 + exp(-i)
      y.bu = __fmul2_rn(v, rsqrt_two<T>(__fmul2_rn(w, __fmul2_rn(pu, pu))));
    } else {
      y.bu = __fmul2_rn(v, rsqrt_two<T>(w));
      if constexpr (kInput) y.bu = __fmul2_rn(y.bu, u);
    }
  } else {
    y.am1 = make_float2(-y.sc.x, -y.sc.y);
    y.bu = kInput ? __fmul2_rn(y.sc, u) : y.sc;
  }
  return y;
}

// ---- tiles ------------------------------------------------------------------------
// A warp's tile: a lane has two channels and kL neighbouring tokens.  A CTA takes
// `ch` = 64, 32 or 16 channels; the ch / 2 lanes of a "part" share its tokens, the
// 64 / ch parts of a warp and the CTA's warps have neighbouring groups of kL.  In
// shared memory token k of part p lies at (k * parts + p) * ch: lane l finds
// its two channels at 64 k + 2 l whatever ch is, in other banks than its warp's
// other lanes.  A warp fetches its own tile and reads no other.
constexpr int kRecurWarps = kRecurThreads / 32;
template <typename T, int kL_>
struct RecurTile {
  static constexpr int kL = kL_;
  static constexpr int kElems = 64 * kL;
  static constexpr int kBytes = kElems * (int)sizeof(T);
};

// Bytes that one copy into shared memory moves: the widest that every row's
// start allows (2: by plain loads).
inline int copy_bytes(const TokenView &v, int size) {
  const uint64_t bits = (uint64_t)(uintptr_t)v.p | (uint64_t)(v.sb * size) | (uint64_t)(v.st * size);
  return bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : 2;
}

template <int kN>
__device__ __forceinline__ void copy_async(uint32_t dst, const void *src, int bytes) {
  if constexpr (kN == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
                 : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(kN),
                 "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kN>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kN) : "memory");
}

// A warp's tile from the rows of tokens [t0, t0 + 64 / ch * kL) of `row0` (the
// tensor at this sequence's first token and this CTA's first channel), all of
// which the sequence has; channels beyond `width` are set to zero and not read.
template <typename T, int kL, int kN>
__device__ __forceinline__ void copy_tile_by(T *tile, const T *row0, int64_t st, int t0, int ch,
                                             int width) {
  constexpr int kPer = kN / (int)sizeof(T);  // elements of a copy
  const int lane = threadIdx.x & 31;
#pragma unroll 4
  for (int n = lane; n < 64 * kL / kPer; n += 32) {
    const int at = n * kPer, k = at / 64, part = at % 64 / ch, q = at % ch;
    const T *src = row0 + (int64_t)(t0 + part * kL + k) * st + q;
    const int bytes = max(0, min(kN, (width - q) * (int)sizeof(T)));
    if constexpr (kN < 4) tile[at] = bytes ? *src : from_f32<T>(0.f);
    else copy_async<kN>((uint32_t)__cvta_generic_to_shared(tile + at), bytes ? src : row0, bytes);
  }
}
template <typename T, int kL>
__device__ __forceinline__ void copy_tile(T *tile, const T *row0, int64_t st, int t0, int ch,
                                          int width, int copy) {
  if (copy == 16) copy_tile_by<T, kL, 16>(tile, row0, st, t0, ch, width);
  else if (copy == 8) copy_tile_by<T, kL, 8>(tile, row0, st, t0, ch, width);
  else if (copy == 4) copy_tile_by<T, kL, 4>(tile, row0, st, t0, ch, width);
  else if constexpr (sizeof(T) == 2) copy_tile_by<T, kL, 2>(tile, row0, st, t0, ch, width);
}
// The same for a tile that the sequence ends in, or that lies beside it: tokens
// outside [0, len) become `outside` and are not read.
template <typename T, int kL>
__device__ __forceinline__ void ragged_tile(T *tile, const T *row0, int64_t st, int t0, int len,
                                            int ch, int width, float outside) {
  const T none = from_f32<T>(outside);
#pragma unroll 8
  for (int at = threadIdx.x & 31; at < 64 * kL; at += 32) {
    const int t = t0 + at % 64 / ch * kL + at / 64, q = at % ch;
    T v = none;
    if (t >= 0 && t < len && q < width) v = row0[(int64_t)t * st + q];
    tile[at] = v;
  }
}

// Over a warp's parts (the lanes `half` = ch / 2 apart): (a, e) becomes the
// summary of all of them, in token order; returned is that of the parts before
// the lane's own, (1, 0) for the first.
struct Summary {
  float2 a, e;
};
__device__ __forceinline__ float2 shuffle_up(float2 v, int by) {
  return make_float2(__shfl_up_sync(0xffffffffu, v.x, by), __shfl_up_sync(0xffffffffu, v.y, by));
}
__device__ __forceinline__ float2 shuffle_down(float2 v, int by) {
  return make_float2(__shfl_down_sync(0xffffffffu, v.x, by), __shfl_down_sync(0xffffffffu, v.y, by));
}
__device__ __forceinline__ float2 shuffle(float2 v, int from) {
  return make_float2(__shfl_sync(0xffffffffu, v.x, from), __shfl_sync(0xffffffffu, v.y, from));
}
template <bool kBackward>  // the other order: the last part first
__device__ __forceinline__ Summary join_parts(float2 &a, float2 &e, int half, int lane) {
  Summary own{two(1.f), two(0.f)};
  if (half == 32) return own;
  const int at = kBackward ? 31 - lane : lane;
  for (int d = half; d < 32; d *= 2) {
    const float2 ao = kBackward ? shuffle_down(a, d) : shuffle_up(a, d);
    const float2 eo = kBackward ? shuffle_down(e, d) : shuffle_up(e, d);
    if (at >= d) e = __ffma2_rn(a, eo, e), a = __fmul2_rn(a, ao);
  }
  const float2 ao = kBackward ? shuffle_down(a, half) : shuffle_up(a, half);
  const float2 eo = kBackward ? shuffle_down(e, half) : shuffle_up(e, half);
  if (at >= half) own = Summary{ao, eo};
  const int last = kBackward ? lane % half : 32 - half + lane % half;
  a = shuffle(a, last);
  e = shuffle(e, last);
  return own;
}

// ---- clusters ---------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Into the shared memory of the cluster's CTA `rank`, at this CTA's address `p`,
// counted there on the mbarrier at this CTA's address `bar`.
__device__ __forceinline__ void store_remote(float4 *p, uint64_t *bar, uint32_t rank, float4 v) {
  uint32_t at, on;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(at)
               : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(on)
               : "r"((uint32_t)__cvta_generic_to_shared(bar)), "r"(rank));
  asm volatile(
      "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];"
      ::"r"(at), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w), "r"(on)
      : "memory");
}

__device__ __forceinline__ void tma_load_4d(void *dst, const CUtensorMap *map, uint64_t *bar, int x,
                                            int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(tc::smem_u32(dst)),
      "l"(map), "r"(tc::smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// What a launch hands its kernel besides the call.
struct RecurLaunch {
  int ch;           // channels of a CTA
  int cluster;      // CTAs along the tokens
  int copy;         // bytes of a cp.async copy; unused with TMA
  int *err;         // the library's device error word
};
constexpr int kRecurMaps = 4;
struct RecurMaps {  // (batch, tokens, channels), with boxes of a tile
  CUtensorMap m[kRecurMaps];
};
// Whether TMA can address the tensor: rows at 16 bytes, no broadcast dimension.
inline bool recur_tma_view(const TokenView &v, const RecurCall &c, int size) {
  return !v.p || (((uintptr_t)v.p & 15) == 0 && v.st * size % 16 == 0 && v.sb * size % 16 == 0 &&
                  v.st >= c.channels && (v.sb > 0 || c.batch == 1) &&
                  v.st < ((int64_t)1 << 32) && v.sb < ((int64_t)1 << 37) && c.batch <= INT32_MAX);
}
// (channels, groups of l tokens, tokens of a group, batch), with boxes that fill a
// warp's tile; for the sequences' whole groups only.
inline bool recur_map(CUtensorMap *map, const TokenView &v, const RecurCall &c, int dtype, int ch,
                      int l) {
  const EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const uint64_t size = dtype == LA_DTYPE_FLOAT32 ? 4 : 2;
  const cuuint64_t st = (cuuint64_t)v.st * size;
  const cuuint64_t dim[4] = {(cuuint64_t)c.channels, (cuuint64_t)(c.tokens / l), (cuuint64_t)l,
                             (cuuint64_t)c.batch};
  const cuuint64_t stride[3] = {st * l, st, c.batch == 1 ? st * l : (cuuint64_t)v.sb * size};
  const cuuint32_t box[4] = {(cuuint32_t)ch, (cuuint32_t)(64 / ch), (cuuint32_t)l, 1};
  const cuuint32_t one[4] = {1, 1, 1, 1};
  return fn(map, dtype == LA_DTYPE_FLOAT32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                           : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
            4, const_cast<void *>(v.p), dim, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Channels of a CTA and CTAs along the tokens for a size: a CTA for every SM from
// narrower channel groups, and only then from clusters along the tokens, each of
// whose CTAs has tokens of its own (l for each of its parts).  A cluster's
// exchange at every step costs more than an idle SM: 16384 x 2048 in 65 us by 128
// CTAs of 16 channels, in 86 by 256 in clusters of two; 2048 x 1024 in 12.0 us by 64
// CTAs, 10.7 by 128 in clusters of two.
struct RecurShape {
  int ch, cluster;
};
inline RecurShape recur_shape(int64_t batch, int64_t tokens, int channels, int sm_count, int l,
                              int widest) {
  RecurShape s{widest, 1};
  auto ctas = [&] { return batch * ((channels + s.ch - 1) / s.ch) * s.cluster; };
  while (s.ch > 16 && ctas() < sm_count) s.ch /= 2;
  while (s.cluster < kRecurMaxCluster && ctas() * 2 <= sm_count &&
         tokens > (int64_t)s.cluster * (64 / s.ch) * l * kRecurWarps)
    s.cluster *= 2;
  return s;
}

template <class Kernel>
int launch_clusters(Kernel kernel, const RecurCall &p, const RecurLaunch &l, const RecurMaps &maps,
                    int smem, cudaStream_t s) {
  const int64_t grid = p.batch * ((p.channels + l.ch - 1) / l.ch) * l.cluster;
  if (grid > INT32_MAX) return LA_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kRecurThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = l.cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = l.cluster > 1 ? 1 : 0;
  cudaLaunchKernelEx(&cfg, kernel, p, l, maps);
  return check_launch();
}

int launch_recur_fwd(const RecurCall &c, int dtype, cudaStream_t s);
int launch_recur_bwd(const RecurCall &c, int dtype, cudaStream_t s);
// CTAs along the tokens that the gradient of this size runs with (rows of
// `partial` per sequence).
int recur_bwd_rows(int64_t batch, int64_t tokens, int channels, int sm_count);

}  // namespace la
