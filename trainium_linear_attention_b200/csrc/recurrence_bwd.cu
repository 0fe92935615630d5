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
// The forward pass' tiles, warps and summaries, walked from the last tokens to the
// first: a summary is (A, R), a H in front = A (a H behind) + R.  14.5 bytes per
// element in bf16 with both gates, against 75 instructions.  h is not saved but
// computed again, in fp32, from the state that the forward pass left every 16
// tokens (a quarter of a byte per element, against two for an h rounded to
// bf16); those states keep the forward chain out of the walk: with one state per
// CTA's tile, handed on from warp to warp against the gradient's direction, 4 x
// 4096 x 1024 took 125 us instead of 71 (52% of the copy rate; no unit above 61%, the wait
// for tiles comes first: 128 CTAs on 148 SMs, 16 warps on each).
// d(lambda) is summed over a CTA's tokens and written as one row per CTA; a second
// kernel adds the rows in a fixed order.
#include <type_traits>

#include "column_sum.cuh"
#include "recurrence.cuh"
#include "tc_kernels.cuh"

namespace la {
namespace {

constexpr int kL = 8;       // tokens of a thread and step
constexpr int kStages = 2;  // tiles of a warp (with 3 the training step takes 106 us, not 103)

template <int kWarps>
struct Exchange {
  // What the warp behind hands to each warp: without a cluster a H (in xy), else the
  // summary (A, A, R, R) of the CTA's tokens behind its own.
  float4 behind[kWarps][32];
  float4 csums[2][kRecurMaxCluster][32];  // summaries of the cluster's CTAs
  float2 sums[kWarps][32];
  uint64_t full[kStages][kWarps], handed[kWarps], arrived[2];
  int abort;
};

template <typename T, bool kDecay, bool kInput, Fetch kF, int kWarps>
__global__ void __launch_bounds__(32 * kWarps, 16 / kWarps)
recur_bwd_kernel(const RecurCall p, const RecurLaunch l, const __grid_constant__ TileMaps maps) {
  constexpr int kIn = kInput ? 4 : 3, kLast = kWarps - 1;
  static_assert(kRecurCheck == 2 * kL, "every other part starts at a saved state");
  extern __shared__ __align__(1024) uint8_t smem[];
  column_sum_may_start();
  const int cluster = l.cluster, ch = l.tile.ch, half = ch / 2, parts = 64 / ch;
  const int channels = p.sizes.channels;
  const int elems = tile_elems<kF>(kL, ch);
  Exchange<kWarps> &ex = *(Exchange<kWarps> *)(smem + kStages * kIn * kWarps * elems * sizeof(T));
  const int rank = cluster > 1 ? (int)cluster_rank() : 0;
  const int groups = (channels + ch - 1) / ch;
  const int64_t ib = blockIdx.x / cluster / groups;
  const int c0 = (int)(blockIdx.x / cluster % groups) * ch;
  const int len = (int)sequence_length(p.lengths, p.lengths64, ib, p.sizes.tokens);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int pair = lane & (half - 1), part = lane / half;
  const int c = c0 + 2 * pair;
  const bool live = c < channels, second = c + 1 < channels;

  const TokenView *views[4] = {&p.x, &p.gate, &p.d_out, &p.input_gate};
  WarpTiles<T, kL, kIn, kStages, kF> tiles{
      (T *)smem + warp * kIn * elems, kWarps * kIn * elems, elems, &ex.full[0][warp], kWarps,
      views, maps.m, ib, c0, ch, min(ch, channels - c0), l.tile.copy, p.sizes, 0};
  const int rows = parts * kL;            // tokens of a warp and step
  const int block_rows = kWarps * rows;
  const int blocks = (len + block_rows - 1) / block_rows;
  const int steps = (blocks + cluster - 1) / cluster;
  auto block_of = [&](int i) { return blocks - 1 - (i * cluster + rank); };  // < 0: none
  auto fetch = [&](int i, int stage) {
    tiles.fetch(block_of(i) * block_rows + warp * rows, i < steps ? len : 0, stage);
  };

  float2 lambda = two(0.f), carry = two(0.f), d_lambda = two(0.f);
  if (live) {
    if (kDecay) lambda = make_float2(p.log_decay[c], second ? p.log_decay[c + 1] : 0.f);
    if (p.d_final) {
      const float *h = p.d_final + ib * channels + c;
      carry = make_float2(h[0], second ? h[1] : 0.f);
    }
  }
  if (threadIdx.x == 0) {
    for (int w = 0; w < kWarps; ++w) {
      for (int j = 0; j < kStages; ++j) tc::mbar_init(&ex.full[j][w], 1);
      tc::mbar_init(&ex.handed[w], 1);
    }
    for (int j = 0; j < 2; ++j) tc::mbar_init(&ex.arrived[j], 1);
    ex.abort = 0;
    tc::fence_barrier_init();
  }
  __syncthreads();
  if (cluster > 1) cluster_arrive();
#pragma unroll
  for (int j = 0; j < kStages; ++j) fetch(j, j);
  if (cluster > 1) cluster_wait();  // the peers' barriers are there before they are counted on

  const bool pairs = kF == Fetch::kTma || p.pairs;
  const int64_t n_check = (p.sizes.tokens + kRecurCheck - 1) / kRecurCheck;
  const int64_t origin = ib * p.sizes.tokens * channels + c;
  // The saved state at or before this thread's tokens of a step; loaded a step ahead.
  auto saved = [&](int i) {
    const int t0 = block_of(i) * block_rows + warp * rows + part * kL;
    if (t0 < 0 || t0 >= len || !live) return two(0.f);
    const float *v = p.check + (ib * n_check + t0 / kRecurCheck) * channels + c;
    return make_float2(v[0], second ? v[1] : 0.f);
  };
  float2 start = saved(0);
  // Without a cluster the chain starts at the warp with the last token: the first
  // step's warps behind it have nothing to do, and they and it are not handed anything then.
  const int last = cluster > 1 ? kLast : max(len - 1, 0) % block_rows / rows;
  int stage = 0;
  for (int i = 0; i < steps; ++i) {
    const int buf = i & 1;
    if (i == 0 && warp > last) {
      start = saved(1);
      fetch(kStages, 0);
      stage = 1;
      continue;
    }
    const T *xs = tiles.tile(stage, 0), *gs = tiles.tile(stage, 1), *ds = tiles.tile(stage, 2),
            *us = tiles.tile(stage, kIn - 1);
    const int block = block_of(i);
    const int row0 = block * block_rows + warp * rows, t0 = row0 + part * kL;
    const bool whole = tiles.whole(row0, len);
    float2 h = start;
    start = saved(i + 1);
    // tokens outside the sequence keep the state and the gradient
    tiles.wait(row0, len, stage, kDecay ? -INFINITY : INFINITY, &ex.abort);
    float2 am1[kL], bu[kL], s[kL], sc[kL], uc[kL];
    float2 a = two(kDecay ? 0.f : 1.f), e = two(0.f), r = two(0.f);
#pragma unroll
    for (int k = 0; k < kL; ++k) {
      const int at = 64 * k + 2 * lane;
      const Token y = token_of<T, kDecay, kInput, true, false>(
          load_two(gs + at), kInput ? load_two(us + at) : two(0.f), lambda);
      am1[k] = y.am1, bu[k] = y.bu, s[k] = y.s, sc[k] = y.sc;
      if (kInput) uc[k] = y.uc;
      e = __ffma2_rn(bu[k], load_two(xs + at), __ffma2_rn(am1[k], e, e));
      a = kDecay ? __fadd2_rn(a, y.s) : __fmul2_rn(a, y.s);
    }
#pragma unroll
    for (int k = kL - 1; k >= 0; --k) {
      r = __fadd2_rn(r, load_two(ds + 64 * k + 2 * lane));
      r = __ffma2_rn(am1[k], r, r);
    }
    if (kDecay) {
      a = __fmul2_rn(a, lambda);
      a = make_float2(Fn<T>::exp(a.x), Fn<T>::exp(a.y));
    }
    {  // an odd part's state comes through the part before
      const float2 ao = shuffle_up(a, half), eo = shuffle_up(e, half);
      if (part & 1) h = __ffma2_rn(ao, h, eo);
    }
    const Summary rest = join_parts<true>(a, r, half, lane);
    float2 g;  // a H of the token behind this thread's
    const int next = warp == 0 ? kLast : warp - 1;
    float2 ap = two(1.f), rp = two(0.f);  // of the CTA's warps behind (with a cluster)
    if (cluster == 1) {
      if (warp < last || i > 0) {
        tc::mbar_wait(&ex.handed[warp], (uint32_t)(warp < last ? i : i - 1) & 1, &ex.abort);
        const float4 v = ex.behind[warp][pair];
        carry = make_float2(v.x, v.y);
      }
      g = carry;
      carry = __ffma2_rn(a, carry, r);
      if (part == 0) *(float2 *)&ex.behind[next][pair] = carry;
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&ex.handed[next]);
    } else {
      if (warp < kLast) {
        tc::mbar_wait(&ex.handed[warp], (uint32_t)i & 1, &ex.abort);
        const float4 v = ex.behind[warp][pair];
        ap = make_float2(v.x, v.y), rp = make_float2(v.z, v.w);
      }
      const float2 at = __fmul2_rn(a, ap), rt = __ffma2_rn(a, rp, r);
      const float4 sum = make_float4(at.x, at.y, rt.x, rt.y);
      if (warp > 0) {
        if (part == 0) ex.behind[next][pair] = sum;
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&ex.handed[next]);
      } else {  // the CTA's summary, to all of the cluster
        if (lane == 0)
          tc::mbar_arrive_expect_tx(&ex.arrived[buf], cluster * half * sizeof(float4));
        if (part == 0)
          for (int j = 0; j < cluster; ++j)
            store_remote(&ex.csums[buf][rank][pair], &ex.arrived[buf], (uint32_t)j, sum);
      }
    }
    float2 before[kL];
#pragma unroll
    for (int k = 0; k < kL; ++k) {
      before[k] = h;
      const float2 x = load_two(xs + 64 * k + 2 * lane);
      h = __ffma2_rn(bu[k], x, __ffma2_rn(am1[k], h, h));
    }
    if (cluster > 1) {
      tc::mbar_wait(&ex.arrived[buf], (uint32_t)(i >> 1) & 1, &ex.abort);
      for (int j = 0; j < cluster; ++j) {
        if (j == rank) g = carry;
        const float4 v = ex.csums[buf][j][pair];
        carry = __ffma2_rn(make_float2(v.x, v.y), carry, make_float2(v.z, v.w));
      }
      g = __ffma2_rn(ap, g, rp);
    }
    g = __ffma2_rn(rest.a, g, rest.e);
    const int64_t o = origin + (int64_t)t0 * channels;
    T *dx = (T *)p.dx + o, *dg = (T *)p.d_gate + o, *di = kInput ? (T *)p.d_input + o : nullptr;
    auto finish = [&](auto all) {
#pragma unroll
      for (int k = kL - 1; k >= 0; --k) {
        const int at = 64 * k + 2 * lane;
        const float2 x = load_two(xs + at);
        const float2 hh = __fadd2_rn(g, load_two(ds + at));
        g = __ffma2_rn(am1[k], hh, hh);  // a H
        const float2 dxk = __fmul2_rn(hh, bu[k]), b = __fmul2_rn(bu[k], x);
        float2 dgk, dik = two(0.f);
        if constexpr (kInput) dik = __fmul2_rn(__fmul2_rn(dxk, x), uc[k]);
        if constexpr (kDecay) {
          // a u x / beta = a (b / beta^2)
          float2 w;
          beta_squared(am1[k], w);
          w = __fmul2_rn(b, rcp_two<T>(w));
          w = __ffma2_rn(am1[k], w, w);
          const float2 d_log = __fmul2_rn(g, __ffma2_rn(w, two(-1.f), before[k]));
          const float2 ds_ = __fmul2_rn(d_log, s[k]);
          d_lambda = __fadd2_rn(d_lambda, ds_);
          dgk = __fmul2_rn(__fmul2_rn(ds_, lambda), sc[k]);
        } else {
          // H (h - u x) s (1 - s) = H s ((1 - s) h - b)
          dgk = __fmul2_rn(__fmul2_rn(hh, s[k]),
                           __ffma2_rn(b, two(-1.f), __fmul2_rn(sc[k], before[k])));
        }
        if (all || (block >= 0 && t0 + k < len)) {
          const int64_t at_k = (int64_t)k * channels;
          store_two(dx + at_k, dxk, all || pairs, second);
          store_two(dg + at_k, dgk, all || pairs, second);
          if constexpr (kInput) store_two(di + at_k, dik, all || pairs, second);
        }
      }
    };
    if (live) {
      if (pairs && whole) finish(std::true_type{});
      else finish(std::false_type{});
    }
    __syncwarp();  // the rows are read
    fetch(i + kStages, stage);
    if (++stage == kStages) stage = 0;
  }
  if (p.d_init && rank == 0 && warp == 0 && part == 0 && live)
    store_two(p.d_init + ib * channels + c, carry, pairs, second);
  const int slots = kWarps * parts;
  for (int64_t t = len + rank * slots + warp * parts + part; t < p.sizes.tokens && live; t += cluster * slots) {
    const int64_t o = origin + t * channels;
    store_two((T *)p.dx + o, two(0.f), pairs, second);
    store_two((T *)p.d_gate + o, two(0.f), pairs, second);
    if (kInput) store_two((T *)p.d_input + o, two(0.f), pairs, second);
  }
  if (kDecay && p.partial) {
    for (int d = half; d < 32; d *= 2) {
      d_lambda.x += __shfl_xor_sync(0xffffffffu, d_lambda.x, d);
      d_lambda.y += __shfl_xor_sync(0xffffffffu, d_lambda.y, d);
    }
    __syncthreads();
    if (part == 0) ex.sums[warp][pair] = d_lambda;
    __syncthreads();
    if (warp == 0 && part == 0 && live) {
      float2 v = two(0.f);
#pragma unroll
      for (int j = 0; j < kWarps; ++j) v = __fadd2_rn(v, ex.sums[j][pair]);
      store_two(p.partial + (ib * cluster + rank) * channels + c, v, channels % 2 == 0, second);
    }
  }
  if (ex.abort) {
    if (l.tile.err) *l.tile.err = tc::kErrTimeout;
    const uint64_t since = tc::globaltimer();  // copies in flight still write into this CTA
    while (tc::globaltimer() - since < tc::kWaitTimeoutNs) __nanosleep(1000);
  }
}

// (The rows of `partial` may not go by the inputs' alignment: the shape is that of 16
// warps' tiles whether they are used or not.)
RecurShape shape_of(const TokenSizes &z, int sm_count) {
  return recur_shape(z, sm_count, kL, 32, true, true);
}

template <typename T, bool kDecay, bool kInput, Fetch kF, int kWarps = 8>
int launch(const RecurCall &p, RecurLaunch l, cudaStream_t s) {
  constexpr int kIn = kInput ? 4 : 3;
  const TokenView *views[4] = {&p.x, &p.gate, &p.d_out, &p.input_gate};
  TileMaps maps;
  for (int n = 0; kF == Fetch::kTma && n < kIn; ++n)
    if (!tile_map(&maps.m[n], *views[n], p.sizes, sizeof(T) == 4 ? LA_DTYPE_FLOAT32 : LA_DTYPE_BFLOAT16,
                  l.tile.ch, kL))
      return LA_ERR_CUDA;
  const int smem = kStages * kIn * kWarps * tile_elems<kF>(kL, l.tile.ch) * (int)sizeof(T) +
                   (int)sizeof(Exchange<kWarps>);
  return launch_clusters(recur_bwd_kernel<T, kDecay, kInput, kF, kWarps>, p, l, maps, 32 * kWarps, smem, s);
}

template <typename T, bool kDecay, bool kInput>
int launch_by_fetch(const RecurCall &p, const RecurShape &shape, cudaStream_t s) {
  RecurLaunch l{{shape.ch, 0, device_error_word()}, shape.cluster};
  const TokenView *views[4] = {&p.x, &p.gate, &p.d_out, &p.input_gate};
  const Fetch f = recur_fetch(p, views, 4, sizeof(T), kL, &l.tile);
  if constexpr (sizeof(T) == 2) {
    if (f == Fetch::kTma && shape.warps == 16)
      return launch<T, kDecay, kInput, Fetch::kTma, 16>(p, l, s);
    if (f == Fetch::kShifted) return launch<T, kDecay, kInput, Fetch::kShifted>(p, l, s);
  }
  if (shape.warps == 2)
    return f == Fetch::kTma ? launch<T, kDecay, kInput, Fetch::kTma, 2>(p, l, s)
                            : launch<T, kDecay, kInput, Fetch::kAsync, 2>(p, l, s);
  return f == Fetch::kTma ? launch<T, kDecay, kInput, Fetch::kTma>(p, l, s)
                          : launch<T, kDecay, kInput, Fetch::kAsync>(p, l, s);
}

template <typename T>
int launch_typed(const RecurCall &p, const RecurShape &sh, cudaStream_t s) {
  if (p.log_decay)
    return p.input_gate.p ? launch_by_fetch<T, true, true>(p, sh, s)
                          : launch_by_fetch<T, true, false>(p, sh, s);
  return p.input_gate.p ? launch_by_fetch<T, false, true>(p, sh, s)
                        : launch_by_fetch<T, false, false>(p, sh, s);
}

}  // namespace

int recur_bwd_rows(const TokenSizes &z, int sm_count) { return shape_of(z, sm_count).cluster; }

int launch_recur_bwd(const RecurCall &p, int dtype, cudaStream_t s) {
  DeviceInfo info;
  const int st = current_device_info(&info);
  if (st != LA_OK) return st;
  const RecurShape sh = shape_of(p.sizes, info.sm_count);
  return dtype == LA_DTYPE_FLOAT32 ? launch_typed<float>(p, sh, s)
                                   : launch_typed<__nv_bfloat16>(p, sh, s);
}

}  // namespace la
