// Gradient of the gated linear recurrence.
//
// With H_t the gradient of h_t, summed over all that h_t reaches:
//   H_t = dh_t + a_{t+1} H_{t+1}        (the last one: + the final state's gradient)
//   dx_t = H_t beta_t u_t               d(input gate)_t = H_t beta_t x_t u_t (1 - u_t)
//   with a decay, beta = sqrt(1 - a^2):
//     d(log a)_t = a_t H_t (h_{t-1} - a_t u_t x_t / beta_t)
//     d(gate)_t = d(log a)_t lambda s_t (1 - s_t),  d(lambda) = sum_t d(log a)_t s_t
//   without: d(gate)_t = H_t (h_{t-1} - u_t x_t) s_t (1 - s_t)
//   d(initial state) = a_0 H_0
//
// The forward pass' tiles, clusters and summaries, walked from the last tile
// to the first (14 bytes per element in bf16 with both gates, against about
// 70 instructions).  h is not saved but computed again, in fp32, from the
// state before each tile that the forward pass left (1/16 byte per element and
// byte of a float, against two for h rounded to bf16): a thread's summary has
// both chains, E for the state and R for the gradient, under one product A.
// d(lambda) is summed over a CTA's tokens and written as one row per CTA; a
// second kernel adds the rows in a fixed order.
#include "column_sum.cuh"
#include "recurrence.cuh"

namespace la {
namespace {

constexpr int kL = 8;  // tokens of a thread and step

template <typename T, int CH, bool kDecay, bool kInput>
__global__ void __launch_bounds__(kRecurThreads, 2) recur_bwd_kernel(const RecurCall p,
                                                                   const int cluster,
                                                                   const int copy) {
  using Tile = RecurTile<T, CH, kL>;
  constexpr int kIn = kInput ? 4 : 3;
  constexpr int kPairs = Tile::kPairs, kSlots = Tile::kSlots, kTok = Tile::kTokens;
  static_assert(kTok % kRecurCheck == 0, "tiles start at saved states");
  extern __shared__ __align__(16) uint8_t smem[];
  T *tiles = (T *)smem;                                  // [2][kIn][kElems]
  __shared__ float4 sums[2][kSlots][kPairs];             // (A, A, R, R) of a pair
  __shared__ float2 sums_e[2][kSlots][kPairs];           // (E, E)
  __shared__ float4 csums[2][kRecurMaxCluster][kPairs];  // (A, A, R, R) of the cluster's CTAs

  column_sum_may_start();
  const int rank = cluster > 1 ? (int)cluster_rank() : 0;
  const int groups = (p.channels + CH - 1) / CH;
  const int64_t unit = blockIdx.x / cluster;
  const int64_t ib = unit / groups;
  const int c0 = (int)(unit % groups) * CH;
  const int width = min(CH, p.channels - c0);
  const int64_t len = recur_length(p.lengths, p.lengths64, ib, p.tokens);
  const int pair = threadIdx.x % kPairs, slot = threadIdx.x / kPairs;
  const int c = c0 + 2 * pair;
  const bool live = c < p.channels, second = c + 1 < p.channels;

  const T *rows[4] = {(const T *)p.x.p + ib * p.x.sb + c0, (const T *)p.gate.p + ib * p.gate.sb + c0,
                      (const T *)p.d_out.p + ib * p.d_out.sb + c0,
                      kInput ? (const T *)p.input_gate.p + ib * p.input_gate.sb + c0 : nullptr};
  const int64_t st[4] = {p.x.st, p.gate.st, p.d_out.st, p.input_gate.st};
  const int64_t blocks = (len + kTok - 1) / kTok;
  const int64_t steps = (blocks + cluster - 1) / cluster;
  auto block_of = [&](int64_t i) { return blocks - 1 - (i * cluster + rank); };  // < 0: none
  auto fetch = [&](int64_t i, int buf) {
    if (i < steps) {
#pragma unroll
      for (int n = 0; n < kIn; ++n)
        load_tile<T, CH, kL>(tiles + (buf * kIn + n) * Tile::kElems, rows[n], st[n],
                             block_of(i) * kTok, len, width, copy);
    }
    copy_commit();
  };

  float2 lambda = two(0.f), carry = two(0.f), d_lambda = two(0.f);
  if (live) {
    if (kDecay) lambda = make_float2(p.log_decay[c], second ? p.log_decay[c + 1] : 0.f);
    if (p.d_final) {
      const float *h = p.d_final + ib * p.channels + c;
      carry = make_float2(h[0], second ? h[1] : 0.f);
    }
  }
  if (cluster > 1) cluster_arrive();
  fetch(0, 0);
  fetch(1, 1);
  if (cluster > 1) cluster_wait();  // the peers run before their shared memory is written

  const bool pairs = p.pairs;
  const int64_t n_check = (p.tokens + kRecurCheck - 1) / kRecurCheck;
  const int64_t first = ib * p.tokens * p.channels + c;
  for (int64_t i = 0; i < steps; ++i) {
    const int buf = (int)(i & 1);
    const T *xs = tiles + buf * kIn * Tile::kElems;
    const T *gs = xs + Tile::kElems, *ds = gs + Tile::kElems, *us = ds + Tile::kElems;
    const int64_t block = block_of(i);
    const int64_t t0 = block * kTok + slot * kL;
    const int inside = block < 0 ? 0 : (int)max64(0, min64(kL, len - t0));
    float2 start = two(0.f);  // the state before the tile
    if (block >= 0 && live) {
      const float *h = p.check + (ib * n_check + block * (kTok / kRecurCheck)) * p.channels + c;
      start = make_float2(h[0], second ? h[1] : 0.f);
    }
    copy_wait<1>();
    __syncthreads();
    // bu = beta u; tokens outside the sequence (zero in the tile) keep state and gradient
    float2 am1[kL], bu[kL], s[kL], sc[kL], uc[kL];
    float2 sum = two(kDecay ? 0.f : 1.f), e = two(0.f), r = two(0.f);
#pragma unroll
    for (int k = 0; k < kL; ++k) {
      const int at = Tile::at(slot * kL + k) + 2 * pair;
      float2 g = load_two(gs + at);
      if (k >= inside) g = two(kDecay ? -INFINITY : INFINITY);
      const Gates y = gates_of<T, kInput>(g, kInput ? load_two(us + at) : two(0.f));
      float2 beta2;
      decay_of<T, kDecay>(y, lambda, am1[k], bu[k], beta2);
      if (kInput) bu[k] = __fmul2_rn(bu[k], y.u), uc[k] = y.uc;
      s[k] = y.s, sc[k] = y.sc;
      e = __ffma2_rn(bu[k], load_two(xs + at), __ffma2_rn(am1[k], e, e));
      sum = kDecay ? __fadd2_rn(sum, y.s) : __fmul2_rn(sum, y.s);
    }
#pragma unroll
    for (int k = kL - 1; k >= 0; --k) {
      r = __fadd2_rn(r, load_two(ds + Tile::at(slot * kL + k) + 2 * pair));
      r = __ffma2_rn(am1[k], r, r);
    }
    if (kDecay) {
      sum = __fmul2_rn(sum, lambda);
      sum = make_float2(Fn<T>::exp(sum.x), Fn<T>::exp(sum.y));
    }
    sums[buf][slot][pair] = make_float4(sum.x, sum.y, r.x, r.y);
    sums_e[buf][slot][pair] = e;
    __syncthreads();

    float2 h = start, g = carry;  // the state before this thread's tokens, the gradient behind
    float2 a = two(1.f), a_own = two(1.f), r_own = two(0.f);
    r = cluster == 1 ? carry : two(0.f);
#pragma unroll
    for (int j = kSlots - 1; j >= 0; --j) {
      if (j == slot) a_own = a, r_own = r;
      const float4 v = sums[buf][j][pair];
      r = __ffma2_rn(make_float2(v.x, v.y), r, make_float2(v.z, v.w));
      a = __fmul2_rn(a, make_float2(v.x, v.y));
    }
    if (cluster == 1) {
      g = r_own;
      carry = r;
    } else {
      if (slot < cluster)
        store_remote(&csums[buf][rank][pair], (uint32_t)slot, make_float4(a.x, a.y, r.x, r.y));
      cluster_arrive();
    }
    for (int j = 0; j < slot; ++j) {
      const float4 v = sums[buf][j][pair];
      h = __ffma2_rn(make_float2(v.x, v.y), h, sums_e[buf][j][pair]);
    }
    float2 before[kL];
#pragma unroll
    for (int k = 0; k < kL; ++k) {
      before[k] = h;
      const float2 x = load_two(xs + Tile::at(slot * kL + k) + 2 * pair);
      h = __ffma2_rn(bu[k], x, __ffma2_rn(am1[k], h, h));
    }
    if (cluster > 1) {
      cluster_wait();
      for (int j = 0; j < cluster; ++j) {
        if (j == rank) g = carry;
        const float4 v = csums[buf][j][pair];
        carry = __ffma2_rn(make_float2(v.x, v.y), carry, make_float2(v.z, v.w));
      }
      g = __ffma2_rn(a_own, g, r_own);
    }
    const int64_t o = first + (t0 + kL - 1) * p.channels;
    T *dx = (T *)p.dx + o, *dg = (T *)p.d_gate + o, *di = kInput ? (T *)p.d_input + o : nullptr;
#pragma unroll
    for (int k = kL - 1; k >= 0; --k) {
      const int at = Tile::at(slot * kL + k) + 2 * pair;
      const float2 x = load_two(xs + at);
      const float2 hh = __fadd2_rn(g, load_two(ds + at));
      g = __ffma2_rn(am1[k], hh, hh);  // a H
      const float2 dxk = __fmul2_rn(hh, bu[k]);
      float2 dgk, dik;
      if constexpr (kInput) dik = __fmul2_rn(__fmul2_rn(dxk, x), uc[k]);
      if constexpr (kDecay) {
        float2 beta2 = __fmul2_rn(make_float2(-am1[k].x, -am1[k].y), __fadd2_rn(am1[k], two(2.f)));
        beta2 = make_float2(Fn<T>::rcp(max_nan(beta2.x, kBetaFloor)),
                            Fn<T>::rcp(max_nan(beta2.y, kBetaFloor)));
        // a u x / beta = a (bu x) / beta^2
        float2 w = __fmul2_rn(__fmul2_rn(bu[k], x), beta2);
        w = __ffma2_rn(am1[k], w, w);
        const float2 d_log = __fmul2_rn(g, __fadd2_rn(before[k], make_float2(-w.x, -w.y)));
        const float2 ds_ = __fmul2_rn(d_log, s[k]);
        d_lambda = __fadd2_rn(d_lambda, ds_);
        dgk = __fmul2_rn(__fmul2_rn(ds_, lambda), sc[k]);
      } else {
        // bu = (1 - s) u: H (h - u x) s (1 - s) = H s ((1 - s) h - bu x)
        const float2 bx = __fmul2_rn(bu[k], x);
        dgk = __fmul2_rn(__fmul2_rn(hh, s[k]),
                         __ffma2_rn(sc[k], before[k], make_float2(-bx.x, -bx.y)));
      }
      if (live && k < inside) {
        store_two(dx, dxk, pairs, second);
        store_two(dg, dgk, pairs, second);
        if constexpr (kInput) store_two(di, dik, pairs, second);
      }
      dx -= p.channels, dg -= p.channels;
      if (kInput) di -= p.channels;
    }
    __syncthreads();  // the tile is read
    fetch(i + 2, buf);
  }
  if (p.d_init && rank == 0 && slot == 0 && live)
    store_two(p.d_init + ib * p.channels + c, carry, pairs, second);
  for (int64_t t = len + rank * kSlots + slot; t < p.tokens && live; t += cluster * kSlots) {
    const int64_t o = first + t * p.channels;
    store_two((T *)p.dx + o, two(0.f), pairs, second);
    store_two((T *)p.d_gate + o, two(0.f), pairs, second);
    if (kInput) store_two((T *)p.d_input + o, two(0.f), pairs, second);
  }
  if (kDecay && p.partial) {
    __syncthreads();
    sums_e[0][slot][pair] = d_lambda;
    __syncthreads();
    if (slot == 0 && live) {
      float2 v = two(0.f);
#pragma unroll
      for (int j = 0; j < kSlots; ++j) v = __fadd2_rn(v, sums_e[0][j][pair]);
      store_two(p.partial + (ib * cluster + rank) * p.channels + c, v, pairs, second);
    }
  }
}

struct Shape {
  int ch, cluster;
};

// As in the forward pass: two CTAs per SM, 32 channels where 64 leave SMs idle.
Shape shape_of(int64_t batch, int64_t tokens, int channels, int sm_count) {
  auto cluster_for = [&](int ch, int tile) {
    const int64_t units = batch * ((channels + ch - 1) / ch);
    int k = 1;
    while (k < kRecurMaxCluster && units * k * 2 <= 2 * sm_count && tokens > (int64_t)k * tile) k *= 2;
    return k;
  };
  const int wide = cluster_for(64, RecurTile<float, 64, kL>::kTokens);
  if (batch * ((channels + 63) / 64) * wide <= sm_count && channels > 32)
    return {32, cluster_for(32, RecurTile<float, 32, kL>::kTokens)};
  return {64, wide};
}

template <typename T, int CH, bool kDecay, bool kInput>
int launch(const RecurCall &p, int cluster, cudaStream_t s) {
  using Tile = RecurTile<T, CH, kL>;
  const int smem = 2 * (kInput ? 4 : 3) * Tile::kBytes;
  auto kernel = recur_bwd_kernel<T, CH, kDecay, kInput>;
  const int st = allow_dynamic_smem((const void *)kernel, smem);
  if (st != LA_OK) return st;
  int copy = 16;
  for (const TokenView *v : {&p.x, &p.gate, &p.d_out, &p.input_gate})
    if (v->p && copy_bytes(*v, sizeof(T)) < copy) copy = copy_bytes(*v, sizeof(T));
  const int64_t grid = p.batch * ((p.channels + CH - 1) / CH) * cluster;
  if (grid > INT32_MAX) return LA_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kRecurThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  cudaLaunchKernelEx(&cfg, kernel, p, cluster, copy);
  return check_launch();
}

template <typename T, bool kDecay, bool kInput>
int launch_by_size(const RecurCall &p, const Shape &shape, cudaStream_t s) {
  if (shape.ch == 32) return launch<T, 32, kDecay, kInput>(p, shape.cluster, s);
  return launch<T, 64, kDecay, kInput>(p, shape.cluster, s);
}

template <typename T>
int launch_typed(const RecurCall &p, const Shape &sh, cudaStream_t s) {
  if (p.log_decay)
    return p.input_gate.p ? launch_by_size<T, true, true>(p, sh, s)
                          : launch_by_size<T, true, false>(p, sh, s);
  return p.input_gate.p ? launch_by_size<T, false, true>(p, sh, s)
                        : launch_by_size<T, false, false>(p, sh, s);
}

}  // namespace

int recur_bwd_rows(int64_t batch, int64_t tokens, int channels, int sm_count) {
  return shape_of(batch, tokens, channels, sm_count).cluster;
}

int launch_recur_bwd(const RecurCall &p, int dtype, cudaStream_t s) {
  DeviceInfo info;
  const int st = current_device_info(&info);
  if (st != LA_OK) return st;
  const Shape sh = shape_of(p.batch, p.tokens, p.channels, info.sm_count);
  return dtype == LA_DTYPE_FLOAT32 ? launch_typed<float>(p, sh, s)
                                   : launch_typed<__nv_bfloat16>(p, sh, s);
}

}  // namespace la
