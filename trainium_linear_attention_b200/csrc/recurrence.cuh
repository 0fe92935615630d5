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

#include "pairs.cuh"
#include "token_tiles.cuh"

namespace la {

struct RecurCall {
  TokenView x, gate, input_gate;     // input_gate.p null: none
  const float *log_decay = nullptr;  // null: a = sigmoid(gate)
  const float *init = nullptr;       // null, or (batch, channels)
  const void *lengths = nullptr;     // null, or one per sequence
  int lengths64 = 0;                 // int64 (else int32)
  TokenSizes sizes;
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
constexpr int kRecurMaxCluster = 8;


// The floor of 1 - a^2 under a root or a division, where it meets a zero.
constexpr float kBetaFloor = 1e-36f;
constexpr float kExpMost = 8.5070592e37f;  // 2^126, whose reciprocal is still normal

// exp(z) - 1 for z <= 0, to a relative 2^-23: z = n ln 2 + f with |f| <= ln 2 / 2,
// exp(z) - 1 = 2^n (exp(f) - 1) + (2^n - 1), exp(f) - 1 = f + f^2 q(f).  q is the
// Chebyshev fit of degree 4 on that interval (2.4e-8 of exp(f) - 1).  On the
// FMA pipe: the special-function unit is as busy as memory without it.
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
  const float2 s = make_float2(__uint_as_float(__float_as_uint(t.x) * (1u << 23) + 0x3F800000u),
                               __uint_as_float(__float_as_uint(t.y) * (1u << 23) + 0x3F800000u));
  return __ffma2_rn(s, p, __fadd2_rn(s, two(-1.f)));
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
//
// kOneRoot: beta u as one root, beta^2 / sqrt(beta^2 p^2) with p = 1 + exp(-i), for a
// loop that the special-function unit bounds (8 x 32768 x 1024 in bf16: 392 us, with two
// functions 412; fp32 gains nothing).  p^2 overflows from an input gate of -44.36 down, and
// u is then 0: the caller takes tokens with such gates without it.
constexpr float kOneRootLeast = -44.f;
template <typename T, bool kDecay, bool kInput, bool kGrad, bool kOneRoot>
__device__ __forceinline__ Token token_of(float2 g, float2 i, float2 lambda) {
  static_assert(!kOneRoot || (kDecay && kInput && !kGrad), "");
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
    if constexpr (!kOneRoot) u = rcp_two<T>(pu);
    if constexpr (kGrad) y.uc = __fmul2_rn(min_nan(eu, kExpMost), u);
  }
  if constexpr (kDecay) {
    y.am1 = expm1_neg(__fmul2_rn(lambda, y.s));
    float2 w;
    const float2 v = beta_squared(y.am1, w);
    if constexpr (kOneRoot) {
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
  __syncwarp();  // (one lane may have been issuing copies)
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

// Channels of a CTA, CTAs along the tokens and warps of a CTA for a size.  A CTA for
// every SM comes from narrower channel groups, and only then from clusters along
// the tokens, each of whose CTAs has tokens of its own (l for each of its parts):
// a cluster's exchange at every step costs more than an idle SM (16384 x 2048 in
// 69 us by 128 CTAs of 16 channels, in 85 by 256 in clusters of two).  One CTA of 16
// warps on most SMs beats two of 8 on some, where instructions bound it (`heavy`: 8 x
// 32768 x 1024 by 128 CTAs of 64 channels and 16 warps in 385 us, by 256 of 32 and 8
// in 429; the gradient of 4 x 4096 x 1024 in 71 and 73); where memory does, all SMs'
// loads count (8 x 8192 x 1024 without a decay: 84 and 72).  `roomy`: 16 warps' tiles
// fit (bf16).  Many short sequences take CTAs of 2 warps, more of which start
// together (64 x 64 x 1024 in 13.5 us against 17.2; 512 tokens in 66 against 59).
struct RecurShape {
  int ch, cluster, warps;
};
inline RecurShape recur_shape(const TokenSizes &z, int sm_count, int l, int widest, bool heavy,
                              bool roomy) {
  RecurShape s{widest, 1, 8};
  auto ctas = [&] { return z.batch * ((z.channels + s.ch - 1) / s.ch) * s.cluster; };
  auto tokens = [&] { return (int64_t)s.cluster * (64 / s.ch) * l * 8; };  // of 8 warps' step
  const int64_t enough = heavy && roomy ? sm_count * 4 / 5 : sm_count;
  while (s.ch > 16 && ctas() < enough) s.ch /= 2;
  while (s.cluster < kRecurMaxCluster && ctas() * 2 <= sm_count && z.tokens > tokens()) s.cluster *= 2;
  if (s.cluster == 1 && ctas() > 2 * sm_count && z.tokens <= tokens()) s.warps = 2;
  if (heavy && roomy && s.cluster == 1 && ctas() <= sm_count && z.tokens > tokens()) s.warps = 16;
  return s;
}

struct RecurLaunch {
  TileLaunch tile;
  int cluster;  // CTAs along the tokens
};

// (TMA kernels write pairs of channels.)
inline Fetch recur_fetch(const RecurCall &p, const TokenView *const *views, int n, int size, int l,
                         TileLaunch *launch) {
  const Fetch f = fetch_of(views, n, p.sizes, size, l, launch);
  return f == Fetch::kTma && !p.pairs ? Fetch::kAsync : f;
}

template <class Kernel>
int launch_clusters(Kernel kernel, const RecurCall &p, const RecurLaunch &l, const TileMaps &maps,
                    int threads, int smem, cudaStream_t s) {
  const int64_t grid = p.sizes.batch * ((p.sizes.channels + l.tile.ch - 1) / l.tile.ch) * l.cluster;
  if (grid > INT32_MAX) return LA_ERR_UNSUPPORTED;
  const int st = allow_dynamic_smem((const void *)kernel, smem);
  if (st != LA_OK) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(threads);
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
int recur_bwd_rows(const TokenSizes &z, int sm_count);

}  // namespace la
