// Gated linear recurrence of each channel: what its kernels share.
//
//   h_t = a_t h_{t-1} + beta_t u_t x_t,   u = sigmoid(input gate), 1 without one
//   with a decay:   a = exp(lambda s), beta = sqrt(1 - a^2),   s = sigmoid(gate)
//   without:        a = s,             beta = 1 - s
//
// The kernels hold 1 - a instead of a: it keeps its relative accuracy where a
// rounds to 1, so that channels with a memory of many thousand tokens forget at
// their own rate, and beta = sqrt((1 - a)(2 - (1 - a))) needs no difference of
// near numbers.
#pragma once

#include "common.cuh"

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

constexpr int kRecurCheck = 64;
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

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// exp(z) - 1 for z <= 0, to a relative 2^-23: z = n ln 2 + f with |f| <= ln 2 / 2,
// exp(z) - 1 = 2^n (exp(f) - 1) + (2^n - 1), exp(f) - 1 = f + f^2 q(f).  q is the
// Chebyshev fit of degree 4 on that interval (1.2e-8 of exp(f) - 1).  On the
// FMA pipe: the special-function unit is as busy as memory without it.
__device__ __forceinline__ float2 expm1_neg(float2 z) {
  z.x = max_nan(z.x, -80.f);  // exp(-80) is far below half an ulp of 1
  z.y = max_nan(z.y, -80.f);
  const float2 magic = two(12582912.f);  // 1.5 * 2^23: the sum's low bits hold n
  const float2 t = __ffma2_rn(z, two(1.4426950408889634f), magic);
  const float2 n = __fadd2_rn(t, two(-12582912.f));
  float2 f = __ffma2_rn(n, two(-0.693145751953125f), z);
  f = __ffma2_rn(n, two(-1.42860682e-6f), f);
  float2 q = __ffma2_rn(two(0.0013933685841038823f), f, two(0.008369184099137783f));
  q = __ffma2_rn(q, f, two(0.041666463017463684f));
  q = __ffma2_rn(q, f, two(0.16666504740715027f));
  q = __ffma2_rn(q, f, two(0.5f));
  const float2 p = __ffma2_rn(__fmul2_rn(f, f), q, f);
  const float2 s = make_float2(__int_as_float((__float_as_int(t.x) << 23) + 0x3F800000),
                               __int_as_float((__float_as_int(t.y) << 23) + 0x3F800000));
  return __ffma2_rn(s, p, __fadd2_rn(s, two(-1.f)));
}

// sigmoid(g) and 1 - sigmoid(g) from e = exp(-|g|) and 1 / (1 + e): both keep
// their relative accuracy, and an infinite gate gives 0 and 1 themselves.
__device__ __forceinline__ void sigmoid_parts(float g, float e, float r, float &s, float &c) {
  const float small = e * r;
  s = g < 0.f ? small : r;
  c = g < 0.f ? r : small;
}

constexpr float kBetaFloor = 1e-36f;  // of 1 - a^2 under a root or a division

// What a token's gates come to, for two channels.
struct Gates {
  float2 s, sc;  // sigmoid(gate) and 1 minus it
  float2 u, uc;  // of the input gate
};
template <typename T, bool kInput>
__device__ __forceinline__ Gates gates_of(float2 g, float2 i) {
  Gates y;
  const float egx = Fn<T>::exp(-fabsf(g.x)), egy = Fn<T>::exp(-fabsf(g.y));
  if constexpr (kInput) {
    const float eux = Fn<T>::exp(-fabsf(i.x)), euy = Fn<T>::exp(-fabsf(i.y));
    const float2 pg = __fadd2_rn(make_float2(egx, egy), two(1.f));
    const float2 pu = __fadd2_rn(make_float2(eux, euy), two(1.f));
    float2 rg, ru;
    if constexpr (sizeof(T) == 2) {  // one reciprocal for both: the product is at most 4
      const float2 pp = __fmul2_rn(pg, pu);
      const float2 r = make_float2(Fn<T>::rcp(pp.x), Fn<T>::rcp(pp.y));
      rg = __fmul2_rn(r, pu);
      ru = __fmul2_rn(r, pg);
    } else {
      rg = make_float2(Fn<T>::rcp(pg.x), Fn<T>::rcp(pg.y));
      ru = make_float2(Fn<T>::rcp(pu.x), Fn<T>::rcp(pu.y));
    }
    sigmoid_parts(g.x, egx, rg.x, y.s.x, y.sc.x);
    sigmoid_parts(g.y, egy, rg.y, y.s.y, y.sc.y);
    sigmoid_parts(i.x, eux, ru.x, y.u.x, y.uc.x);
    sigmoid_parts(i.y, euy, ru.y, y.u.y, y.uc.y);
  } else {
    sigmoid_parts(g.x, egx, Fn<T>::rcp(1.f + egx), y.s.x, y.sc.x);
    sigmoid_parts(g.y, egy, Fn<T>::rcp(1.f + egy), y.s.y, y.sc.y);
  }
  return y;
}

// a - 1, and beta (and, with a decay, beta^2 where the gradient wants it).
template <typename T, bool kDecay>
__device__ __forceinline__ void decay_of(const Gates &y, float2 lambda, float2 &am1, float2 &beta,
                                         float2 &beta2) {
  if constexpr (kDecay) {
    am1 = expm1_neg(__fmul2_rn(lambda, y.s));
    // 1 - a^2 = -(a - 1)(2 + (a - 1)); a gate that forgets nothing adds nothing (0, not 0 * inf)
    beta2 = __fmul2_rn(make_float2(-am1.x, -am1.y), __fadd2_rn(am1, two(2.f)));
    beta = __fmul2_rn(beta2, make_float2(Fn<T>::rsqrt(max_nan(beta2.x, kBetaFloor)),
                                         Fn<T>::rsqrt(max_nan(beta2.y, kBetaFloor))));
  } else {
    am1 = make_float2(-y.sc.x, -y.sc.y);
    beta = y.sc;
  }
}

// ---- tiles ------------------------------------------------------------------------
// Channels that a CTA takes, and how its lanes share a tile: a lane has two
// channels, a group of CH / 2 lanes ("slot") kL neighbouring tokens, the slots
// of the CTA neighbouring groups of tokens.
template <typename T, int CH, int kL>
struct RecurTile {
  static constexpr int kPairs = CH / 2;
  static constexpr int kSlots = kRecurThreads / kPairs;
  static constexpr int kTokens = kSlots * kL;
  // Rows of 64 bytes: every slot starts 64 bytes on, so that the two slots of a
  // warp read other banks.
  static constexpr int kPad = CH * sizeof(T) < 128 ? 64 / sizeof(T) : 0;
  static constexpr int kElems = kTokens * CH + kSlots * kPad;
  static constexpr int kBytes = kElems * sizeof(T);
  static __device__ __forceinline__ int at(int token) { return token * CH + token / kL * kPad; }
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

// Rows [t0, t0 + kTokens) of `row0` (the tensor at this sequence's first token
// and this CTA's first channel), `width` channels of them, into `tile`; what is
// outside [0, len) or beyond the width is set to zero and not read.
template <typename T, int CH, int kL, int kN>
__device__ __forceinline__ void load_tile_by(T *tile, const T *row0, int64_t st, int64_t t0,
                                             int64_t len, int width) {
  using Tile = RecurTile<T, CH, kL>;
  constexpr int kPer = kN / (int)sizeof(T);  // elements of a copy
  constexpr int kRow = CH / kPer;            // copies of a row
  static_assert(kRecurThreads % kRow == 0 || kRow % kRecurThreads == 0, "whole rows per turn");
  const int q = threadIdx.x % kRow * kPer;
  const int left = max(0, min(kN, (width - q) * (int)sizeof(T)));
  constexpr int kStep = kRecurThreads / kRow;
  int row = threadIdx.x / kRow;
  const T *src = row0 + (t0 + row) * st + q;
#pragma unroll 4
  for (; row < Tile::kTokens; row += kStep, src += kStep * st) {
    const int64_t t = t0 + row;
    const int bytes = t >= 0 && t < len ? left : 0;
    T *dst = tile + Tile::at(row) + q;
    if constexpr (kN < 4) {
      T v = from_f32<T>(0.f);
      if (bytes) v = *src;
      *dst = v;
    } else {
      copy_async<kN>((uint32_t)__cvta_generic_to_shared(dst), bytes ? src : row0, bytes);
    }
  }
}
template <typename T, int CH, int kL>
__device__ __forceinline__ void load_tile(T *tile, const T *row0, int64_t st, int64_t t0,
                                          int64_t len, int width, int copy) {
  if (copy == 16) load_tile_by<T, CH, kL, 16>(tile, row0, st, t0, len, width);
  else if (copy == 8) load_tile_by<T, CH, kL, 8>(tile, row0, st, t0, len, width);
  else if (copy == 4) load_tile_by<T, CH, kL, 4>(tile, row0, st, t0, len, width);
  else if constexpr (sizeof(T) == 2) load_tile_by<T, CH, kL, 2>(tile, row0, st, t0, len, width);
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
// Into the shared memory of the cluster's CTA `rank`, at this CTA's address `p`.
__device__ __forceinline__ void store_remote(float4 *p, uint32_t rank, float4 v) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(at)
               : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(v.x), "f"(v.y),
               "f"(v.z), "f"(v.w)
               : "memory");
}

int launch_recur_fwd(const RecurCall &c, int dtype, cudaStream_t s);
int launch_recur_bwd(const RecurCall &c, int dtype, cudaStream_t s);
// CTAs along the tokens that the gradient of this size runs with (rows of
// `partial` per sequence).
int recur_bwd_rows(int64_t batch, int64_t tokens, int channels, int sm_count);

}  // namespace la
