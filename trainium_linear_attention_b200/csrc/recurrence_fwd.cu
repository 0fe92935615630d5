// Gated linear recurrence: prompts, and single tokens.
//
// Bound by memory: x and the gates read once, h written once (8 bytes per
// element in bf16 with both gates), against about 30 instructions.  A sequence
// of one channel is a chain, so the parallel work is channels x batch, too few
// for a long prompt: a CTA takes 64 (or 32) channels and, at each step, a tile of
// neighbouring tokens, and a cluster of up to 8 CTAs along the tokens shares a
// channel group.  Per step every thread
//   1. turns kL tokens of two channels into (a - 1, b), kept in registers, and
//      folds them to a summary (A, E): h_out = A h_in + E,
//   2. reads the summaries of the CTA's other threads (shared memory) and of the
//      cluster's other CTAs (distributed shared memory, one cluster barrier),
//   3. walks its tokens once more from its own h_in, and writes them.
// So inputs are read once, nothing waits for another cluster, and the sums have
// one fixed order.  The tiles are fetched two steps ahead with cp.async.
#include "recurrence.cuh"

namespace la {
namespace {

constexpr int kL = 16;  // tokens of a thread and step

template <typename T, int CH, bool kDecay, bool kInput>
__global__ void __launch_bounds__(kRecurThreads, 2) recur_fwd_kernel(const RecurCall p,
                                                                   const int cluster,
                                                                   const int copy) {
  using Tile = RecurTile<T, CH, kL>;
  constexpr int kIn = kInput ? 3 : 2;
  constexpr int kPairs = Tile::kPairs, kSlots = Tile::kSlots, kTok = Tile::kTokens;
  extern __shared__ __align__(16) uint8_t smem[];
  T *tiles = (T *)smem;  // [2][kIn][kElems]
  __shared__ float4 sums[2][kSlots][kPairs];             // (A, A, E, E) of a pair
  __shared__ float4 csums[2][kRecurMaxCluster][kPairs];  // of the cluster's CTAs

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

  const T *rows[3] = {(const T *)p.x.p + ib * p.x.sb + c0, (const T *)p.gate.p + ib * p.gate.sb + c0,
                      kInput ? (const T *)p.input_gate.p + ib * p.input_gate.sb + c0 : nullptr};
  const int64_t st[3] = {p.x.st, p.gate.st, p.input_gate.st};
  const int64_t step = (int64_t)cluster * kTok;
  const int64_t steps = (len + step - 1) / step;
  auto fetch = [&](int64_t i, int buf) {
    if (i < steps) {
#pragma unroll
      for (int n = 0; n < kIn; ++n)
        load_tile<T, CH, kL>(tiles + (buf * kIn + n) * Tile::kElems, rows[n], st[n],
                             i * step + rank * kTok, len, width, copy);
    }
    copy_commit();
  };

  float2 lambda = two(0.f), carry = two(0.f);
  if (live) {
    if (kDecay) lambda = make_float2(p.log_decay[c], second ? p.log_decay[c + 1] : 0.f);
    if (p.init) {
      const float *h = p.init + ib * p.channels + c;
      carry = make_float2(h[0], second ? h[1] : 0.f);
    }
  }
  if (cluster > 1) cluster_arrive();
  fetch(0, 0);
  fetch(1, 1);
  if (cluster > 1) cluster_wait();  // the peers run before their shared memory is written

  const bool pairs = p.pairs;
  T *out = (T *)p.out + ib * p.tokens * p.channels + c;
  const int64_t n_check = (p.tokens + kRecurCheck - 1) / kRecurCheck;
  for (int64_t i = 0; i < steps; ++i) {
    const int buf = (int)(i & 1);
    const T *xs = tiles + buf * kIn * Tile::kElems;
    const T *gs = xs + Tile::kElems, *us = gs + Tile::kElems;
    const int64_t t0 = i * step + rank * kTok + slot * kL;
    copy_wait<1>();
    __syncthreads();
    // tokens beyond the sequence (zero in the tile) keep the state: an infinite
    // gate of the sign that forgets nothing
    const int inside = (int)max64(0, min64(kL, len - t0));
    float2 am1[kL], b[kL];
    float2 sum = two(kDecay ? 0.f : 1.f), e = two(0.f);
#pragma unroll
    for (int k = 0; k < kL; ++k) {
      const int at = Tile::at(slot * kL + k) + 2 * pair;
      float2 g = load_two(gs + at);
      if (k >= inside) g = two(kDecay ? -INFINITY : INFINITY);
      const Gates y = gates_of<T, kInput>(g, kInput ? load_two(us + at) : two(0.f));
      float2 beta, beta2;
      decay_of<T, kDecay>(y, lambda, am1[k], beta, beta2);
      if (kInput) beta = __fmul2_rn(beta, y.u);
      b[k] = __fmul2_rn(beta, load_two(xs + at));
      e = __fadd2_rn(__ffma2_rn(am1[k], e, e), b[k]);
      sum = kDecay ? __fadd2_rn(sum, y.s) : __fmul2_rn(sum, y.s);
    }
    if (kDecay) {
      sum = __fmul2_rn(sum, lambda);
      sum = make_float2(Fn<T>::exp(sum.x), Fn<T>::exp(sum.y));
    }
    sums[buf][slot][pair] = make_float4(sum.x, sum.y, e.x, e.y);
    __syncthreads();
    fetch(i + 2, buf);

    float2 h = carry;  // the state before this thread's tokens
    if (cluster == 1) {
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
        if (j == slot) h = carry;
        const float4 v = sums[buf][j][pair];
        carry = __ffma2_rn(make_float2(v.x, v.y), carry, make_float2(v.z, v.w));
      }
    } else {
      float2 a = two(1.f), a_own = two(1.f), e_own = two(0.f);
      e = two(0.f);
#pragma unroll
      for (int j = 0; j < kSlots; ++j) {
        if (j == slot) a_own = a, e_own = e;
        const float4 v = sums[buf][j][pair];
        e = __ffma2_rn(make_float2(v.x, v.y), e, make_float2(v.z, v.w));
        a = __fmul2_rn(a, make_float2(v.x, v.y));
      }
      if (slot < cluster)
        store_remote(&csums[buf][rank][pair], (uint32_t)slot, make_float4(a.x, a.y, e.x, e.y));
      cluster_arrive();
      cluster_wait();
      for (int j = 0; j < cluster; ++j) {
        if (j == rank) h = carry;
        const float4 v = csums[buf][j][pair];
        carry = __ffma2_rn(make_float2(v.x, v.y), carry, make_float2(v.z, v.w));
      }
      h = __ffma2_rn(a_own, h, e_own);
    }
    if (p.check && live && inside > 0 && (t0 & (kRecurCheck - 1)) == 0)
      store_two(p.check + (ib * n_check + t0 / kRecurCheck) * p.channels + c, h, pairs, second);
    T *dst = out + t0 * p.channels;
#pragma unroll
    for (int k = 0; k < kL; ++k) {
      h = __fadd2_rn(__ffma2_rn(am1[k], h, h), b[k]);
      if (live && k < inside) store_two(dst, h, pairs, second);
      dst += p.channels;
    }
  }
  if (p.final_state && rank == 0 && slot == 0 && live)
    store_two(p.final_state + ib * p.channels + c, carry, pairs, second);
  // zeros behind the sequence
  for (int64_t t = len + rank * kSlots + slot; t < p.tokens && live; t += cluster * kSlots)
    store_two(out + t * p.channels, two(0.f), pairs, second);
}

template <typename T, int CH, bool kDecay, bool kInput>
int launch(const RecurCall &p, int cluster, cudaStream_t s) {
  using Tile = RecurTile<T, CH, kL>;
  const int smem = 2 * (kInput ? 3 : 2) * Tile::kBytes;
  auto kernel = recur_fwd_kernel<T, CH, kDecay, kInput>;
  const int st = allow_dynamic_smem((const void *)kernel, smem);
  if (st != LA_OK) return st;
  int copy = copy_bytes(p.x, sizeof(T)) < copy_bytes(p.gate, sizeof(T)) ? copy_bytes(p.x, sizeof(T))
                                                                        : copy_bytes(p.gate, sizeof(T));
  if (kInput && copy_bytes(p.input_gate, sizeof(T)) < copy) copy = copy_bytes(p.input_gate, sizeof(T));
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
int launch_by_size(const RecurCall &p, cudaStream_t s) {
  DeviceInfo info;
  const int st = current_device_info(&info);
  if (st != LA_OK) return st;
  // Two CTAs per SM, by as many CTAs along the tokens as they have tiles for;
  // 32 channels where that leaves SMs idle.
  auto cluster_for = [&](int ch, int tokens) {
    const int64_t units = p.batch * ((p.channels + ch - 1) / ch);
    int k = 1;
    while (k < kRecurMaxCluster && units * k * 2 <= 2 * info.sm_count && p.tokens > (int64_t)k * tokens)
      k *= 2;
    return k;
  };
  const int wide = cluster_for(64, RecurTile<T, 64, kL>::kTokens);
  const int64_t ctas = p.batch * ((p.channels + 63) / 64) * wide;
  if (ctas <= info.sm_count && p.channels > 32)
    return launch<T, 32, kDecay, kInput>(p, cluster_for(32, RecurTile<T, 32, kL>::kTokens), s);
  return launch<T, 64, kDecay, kInput>(p, wide, s);
}

template <typename T>
int launch_typed(const RecurCall &p, cudaStream_t s) {
  if (p.log_decay)
    return p.input_gate.p ? launch_by_size<T, true, true>(p, s) : launch_by_size<T, true, false>(p, s);
  return p.input_gate.p ? launch_by_size<T, false, true>(p, s) : launch_by_size<T, false, false>(p, s);
}

}  // namespace

int launch_recur_fwd(const RecurCall &p, int dtype, cudaStream_t s) {
  return dtype == LA_DTYPE_FLOAT32 ? launch_typed<float>(p, s) : launch_typed<__nv_bfloat16>(p, s);
}

}  // namespace la
