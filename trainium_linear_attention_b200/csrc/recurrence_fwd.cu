// Gated linear recurrence: prompts.
//
// Bound by memory and, nearly as much, by its instructions: x and the gates are
// read once and h is written once (8 bytes per element in bf16 with both gates),
// against 36 instructions and 4 of the special-function unit, which does 16 a cycle
// and SM.  A channel's sequence is a chain, and channels x batch are too few
// chains for the SMs, so a CTA takes 64, 32 or 16 channels and its lanes and warps
// neighbouring groups of kL tokens.  A thread
//   1. turns its tokens of two channels into (a - 1, b), kept in registers, and
//      folds them to a summary (A, E): h_out = A h_in + E,
//   2. gets h_in: the summaries of the warp's other parts by shuffles, the state
//      from the warp before, which it hands on to the next one at once,
//   3. walks its tokens once more from h_in, and writes them.
// Warps fetch their own tiles by TMA two steps ahead and wait for nothing but
// them and the warp before: no barrier over the CTA.  With too few channels for the
// SMs a cluster of up to 8 CTAs along the tokens shares a channel group; its CTAs'
// summaries cross distributed shared memory once per step.  Inputs that TMA cannot
// address come by cp.async, or element by element.  The sums have one fixed
// order.
//
// A CTA has 2, 8 or 16 warps (recur_shape says when).
//
// 8 x 32768 x 1024 in 392 us (5.5 TB/s, 83% of the copy rate), 16384 x 2048 in 61
// (128 CTAs: 67%), 4 x 4096 x 1024 in 34 (60%; 62% of the issue slots, 59% of the
// special-function unit's), in fp32 55 (74%).  What it took, for the first of these: one
// barrier-bound form with cp.async 873 us, fewer instructions (one root for beta and u, no selects)
// 663, TMA 524, the hand-over from warp to warp 451, tiles that any channel width reads
// without bank conflicts and stores without predicates 421, 16 warps with one chain of
// hand-overs for an SM 385 (392 with input gates below -44).
#include "recurrence.cuh"
#include "tc_kernels.cuh"

namespace la {
namespace {

constexpr int kL = 16;       // tokens of a thread and step
constexpr int kStages = 2;   // tiles of a warp

template <int kWarps>
struct Exchange {
  // What the warp before hands to each warp: without a cluster the state (in
  // xy), else the summary (A, A, E, E) of the CTA's tokens before its own.
  float4 before[kWarps][32];
  float4 csums[2][kRecurMaxCluster][32];  // summaries of the cluster's CTAs
  uint64_t full[kStages][kWarps], handed[kWarps], arrived[2];
  int abort;
};

// beta u x of a thread's tokens, of any input gates, in the place of its x and input gates
// (two fp32 values for each pair).  Out of the way of the loop that reads them back.
__device__ __noinline__ void any_input_gates(__nv_bfloat16 *xs, const __nv_bfloat16 *gs,
                                             __nv_bfloat16 *us, float2 lambda) {
#pragma unroll 1
  for (int k = 0; k < kL; ++k, xs += 64, gs += 64, us += 64) {
    const Token y = token_of<__nv_bfloat16, true, true, false, false>(load_two(gs), load_two(us), lambda);
    const float2 b = __fmul2_rn(y.bu, load_two(xs));
    *(float *)xs = b.x;
    *(float *)us = b.y;
  }
}

template <typename T, bool kDecay, bool kInput, Fetch kF, int kWarps>
__global__ void __launch_bounds__(32 * kWarps, 16 / kWarps)
recur_fwd_kernel(const RecurCall p, const RecurLaunch l, const __grid_constant__ TileMaps maps) {
  constexpr int kIn = kInput ? 3 : 2, kLast = kWarps - 1;
  extern __shared__ __align__(1024) uint8_t smem[];
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

  const TokenView *views[3] = {&p.x, &p.gate, &p.input_gate};
  WarpTiles<T, kL, kIn, kStages, kF> tiles{
      (T *)smem + warp * kIn * elems, kWarps * kIn * elems, elems, &ex.full[0][warp], kWarps,
      views, maps.m, ib, c0, ch, min(ch, channels - c0), l.tile.copy, p.sizes, 0};
  const int rows = parts * kL;                      // tokens of a warp and step
  const int step = cluster * kWarps * rows;    // of all
  const int steps = (len + step - 1) / step;
  const int first = (rank * kWarps + warp) * rows;
  auto fetch = [&](int i, int stage) { tiles.fetch(i * step + first, i < steps ? len : 0, stage); };

  float2 lambda = two(0.f), carry = two(0.f);
  if (live) {
    if (kDecay) lambda = make_float2(p.log_decay[c], second ? p.log_decay[c + 1] : 0.f);
    if (p.init) {
      const float *h = p.init + ib * channels + c;
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
  T *out = (T *)p.out + ib * p.sizes.tokens * channels + c;
  const int64_t n_check = (p.sizes.tokens + kRecurCheck - 1) / kRecurCheck;
  int stage = 0;
  for (int i = 0; i < steps; ++i) {
    const int buf = i & 1;
    T *const xs = tiles.tile(stage, 0), *const gs = tiles.tile(stage, 1),
            *const us = tiles.tile(stage, kIn - 1);
    const int row0 = i * step + first, t0 = row0 + part * kL;
    if (cluster == 1 && row0 >= len) break;  // (nobody waits for the last step's other warps)
    const bool whole = tiles.whole(row0, len);
    // tokens beyond the sequence keep the state
    tiles.wait(row0, len, stage, kDecay ? -INFINITY : INFINITY, &ex.abort);
    float2 am1[kL], b[kL];
    float2 a = two(kDecay ? 0.f : 1.f), e = two(0.f);
    constexpr bool kOneRoot = kDecay && kInput && sizeof(T) == 2;
    Least least;  // of the input gates
#pragma unroll
    for (int k = 0; k < kL; ++k) {
      const int at = 64 * k + 2 * lane;
      if constexpr (kOneRoot)
        if (k % 2) least.take(us + at - 64, us + at);
      const Token y = token_of<T, kDecay, kInput, false, kOneRoot>(
          load_two(gs + at), kInput ? load_two(us + at) : two(0.f), lambda);
      am1[k] = y.am1;
      b[k] = __fmul2_rn(y.bu, load_two(xs + at));
      e = __fadd2_rn(__ffma2_rn(am1[k], e, e), b[k]);
      a = kDecay ? __fadd2_rn(a, y.s) : __fmul2_rn(a, y.s);
    }
    if (kDecay) {
      a = __fmul2_rn(a, lambda);
      a = make_float2(Fn<T>::exp(a.x), Fn<T>::exp(a.y));
    }
    if constexpr (kOneRoot) {
      if (least.below(kOneRootLeast)) {  // nearly closed input gates
        any_input_gates(xs + 2 * lane, gs + 2 * lane, us + 2 * lane, lambda);
        e = two(0.f);
#pragma unroll
        for (int k = 0; k < kL; ++k) {
          const int at = 64 * k + 2 * lane;
          b[k] = make_float2(*(const float *)(xs + at), *(const float *)(us + at));
          e = __fadd2_rn(__ffma2_rn(am1[k], e, e), b[k]);
        }
        if (kF == Fetch::kTma) tc::fence_proxy_async_smem();  // (ahead of the next copy into it)
      }
    }
    __syncwarp();  // the rows are read
    fetch(i + kStages, stage);
    if (++stage == kStages) stage = 0;

    const Summary own = join_parts<false>(a, e, half, lane);
    float2 h;  // the state before this thread's tokens
    if (cluster == 1) {
      if (warp > 0 || i > 0) {
        tc::mbar_wait(&ex.handed[warp], (uint32_t)(warp > 0 ? i : i - 1) & 1, &ex.abort);
        const float4 v = ex.before[warp][pair];
        carry = make_float2(v.x, v.y);
      }
      h = __ffma2_rn(own.a, carry, own.e);
      carry = __ffma2_rn(a, carry, e);
      const int next = warp == kLast ? 0 : warp + 1;
      if (part == 0) *(float2 *)&ex.before[next][pair] = carry;
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&ex.handed[next]);
    } else {
      float2 ap = two(1.f), ep = two(0.f);  // of the CTA's warps before
      if (warp > 0) {
        tc::mbar_wait(&ex.handed[warp], (uint32_t)i & 1, &ex.abort);
        const float4 v = ex.before[warp][pair];
        ap = make_float2(v.x, v.y), ep = make_float2(v.z, v.w);
      }
      e = __ffma2_rn(a, ep, e);
      a = __fmul2_rn(a, ap);
      const float4 sum = make_float4(a.x, a.y, e.x, e.y);
      if (warp < kLast) {
        if (part == 0) ex.before[warp + 1][pair] = sum;
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&ex.handed[warp + 1]);
      } else {  // the CTA's summary, to all of the cluster
        if (lane == 0)
          tc::mbar_arrive_expect_tx(&ex.arrived[buf], cluster * half * sizeof(float4));
        if (part == 0)
          for (int j = 0; j < cluster; ++j)
            store_remote(&ex.csums[buf][rank][pair], &ex.arrived[buf], (uint32_t)j, sum);
      }
      tc::mbar_wait(&ex.arrived[buf], (uint32_t)(i >> 1) & 1, &ex.abort);
      for (int j = 0; j < cluster; ++j) {
        if (j == rank) h = carry;
        const float4 v = ex.csums[buf][j][pair];
        carry = __ffma2_rn(make_float2(v.x, v.y), carry, make_float2(v.z, v.w));
      }
      h = __ffma2_rn(ap, h, ep);
      h = __ffma2_rn(own.a, h, own.e);
    }
    static_assert(kL == kRecurCheck, "every thread saves the state before its tokens");
    if (p.check && live && t0 < len)
      store_two(p.check + (ib * n_check + t0 / kRecurCheck) * channels + c, h, pairs, second);
    T *dst = out + (int64_t)t0 * channels;
    if (!live) continue;
    if (pairs && whole) {
#pragma unroll
      for (int k = 0; k < kL; ++k) {
        h = __fadd2_rn(__ffma2_rn(am1[k], h, h), b[k]);
        store_two(dst + (int64_t)k * channels, h, true, true);
      }
    } else {
#pragma unroll
      for (int k = 0; k < kL; ++k) {
        h = __fadd2_rn(__ffma2_rn(am1[k], h, h), b[k]);
        if (t0 + k < len) store_two(dst + (int64_t)k * channels, h, pairs, second);
      }
    }
  }
  // by the warp with the last token; with a cluster all warps have folded all summaries
  const int last = cluster > 1 ? kLast : max(len - 1, 0) % step / rows;
  if (p.final_state && rank == 0 && warp == last && part == 0 && live)
    store_two(p.final_state + ib * channels + c, carry, pairs, second);
  // zeros behind the sequence
  const int slots = kWarps * parts;
  for (int64_t t = len + rank * slots + warp * parts + part; t < p.sizes.tokens && live; t += cluster * slots)
    store_two(out + t * channels, two(0.f), pairs, second);
  if (ex.abort) {
    if (l.tile.err) *l.tile.err = tc::kErrTimeout;
    const uint64_t since = tc::globaltimer();  // copies in flight still write into this CTA
    while (tc::globaltimer() - since < tc::kWaitTimeoutNs) __nanosleep(1000);
  }
}

template <typename T, bool kDecay, bool kInput, Fetch kF, int kWarps = 8>
int launch(const RecurCall &p, RecurLaunch l, cudaStream_t s) {
  constexpr int kIn = kInput ? 3 : 2;
  const TokenView *views[3] = {&p.x, &p.gate, &p.input_gate};
  TileMaps maps;
  for (int n = 0; kF == Fetch::kTma && n < kIn; ++n)
    if (!tile_map(&maps.m[n], *views[n], p.sizes, sizeof(T) == 4 ? LA_DTYPE_FLOAT32 : LA_DTYPE_BFLOAT16,
                  l.tile.ch, kL))
      return LA_ERR_CUDA;
  const int smem = kStages * kIn * kWarps * tile_elems<kF>(kL, l.tile.ch) * (int)sizeof(T) +
                   (int)sizeof(Exchange<kWarps>);
  return launch_clusters(recur_fwd_kernel<T, kDecay, kInput, kF, kWarps>, p, l, maps, 32 * kWarps, smem, s);
}

template <typename T, bool kDecay, bool kInput>
int launch_by_fetch(const RecurCall &p, cudaStream_t s) {
  DeviceInfo info;
  const int st = current_device_info(&info);
  if (st != LA_OK) return st;
  RecurLaunch l{{0, 0, device_error_word()}, 1};
  const TokenView *views[3] = {&p.x, &p.gate, &p.input_gate};
  const Fetch f = recur_fetch(p, views, 3, sizeof(T), kL, &l.tile);
  const RecurShape shape =
      recur_shape(p.sizes, info.sm_count, kL, 64, kDecay, f == Fetch::kTma && sizeof(T) == 2);
  l.tile.ch = shape.ch, l.cluster = shape.cluster;
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
int launch_typed(const RecurCall &p, cudaStream_t s) {
  if (p.log_decay)
    return p.input_gate.p ? launch_by_fetch<T, true, true>(p, s) : launch_by_fetch<T, true, false>(p, s);
  return p.input_gate.p ? launch_by_fetch<T, false, true>(p, s) : launch_by_fetch<T, false, false>(p, s);
}

}  // namespace

int launch_recur_fwd(const RecurCall &p, int dtype, cudaStream_t s) {
  return dtype == LA_DTYPE_FLOAT32 ? launch_typed<float>(p, s) : launch_typed<__nv_bfloat16>(p, s);
}

}  // namespace la
