// Causal convolution of each channel with 2 to 4 taps, an activation, and its
// gradient.
//
//   z_t = bias + sum_j w_j x_{t - taps + 1 + j},   y = z, or z sigmoid(z)
//   dz = dy, or dy sigmoid(z) (1 + z (1 - sigmoid(z)))
//   dx_t = sum_j w_j dz_{t + taps - 1 - j},  dw_j = sum_t dz_t x_{t - taps + 1 + j}
//
// Bound by memory: x read and y written once (4 bytes per element in bf16),
// the gradient also reads dy (6).  A warp takes 64 channels, a pair for each lane,
// and walks a run of tokens with the taps' window in registers; it fetches its
// tiles of 16 tokens itself, two ahead, by TMA where the rows allow it (token_tiles.cuh).
// The tokens before and behind a run are read twice, the second time from the
// caches.  The gradient computes z again instead of keeping it.  Its walk meets dz_t
// once and adds it to the taps' sums that are still open, so that dx, dw and the
// bias' gradient come from one pass; the sums over tokens are joined over the
// CTA's warps in shared memory, written as one row per CTA, and the rows added by a
// second kernel in a fixed order.
//
// 4 x 4096 x 1024 with SiLU in 18.2 us (56% of the copy rate), its gradient in 34 (45%):
// 26 and 55 instructions of a warp for its 64 channels of a token.  No unit bounds it (44%
// of the issue slots, half of the special-function unit's forward): a warp's run is 8
// tiles, the first of which it waits for, and 256 CTAs are two on some SMs and one on
// others.  In fp32 26.5 us (77%) and 49 (63%).
#include <type_traits>

#include "column_sum.cuh"
#include "short_conv.cuh"
#include "tc_kernels.cuh"

namespace la {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kL = 16;       // tokens of a tile
// Tiles of a warp (4 x 4096 x 1024, a training step: 51.9 us with 2, 53.3 with 3; 1023
// wide 79 and 104: fewer CTAs fit).
constexpr int kStages = 2;
// Tokens of a warp's run: many, since a run's ends are read twice and the sums of a
// gradient's CTA are written once, but fewer where that leaves SMs without a CTA (4
// x 4096 x 1024 by 256 CTAs of 128-token runs, 512 of 64, 1024 of 32: the gradient
// in 34, 38 and 39 us, the forward pass in 19 each).  The same for both passes; the
// workspace's size goes by it.
constexpr int kMostRun = 128;
constexpr int64_t kEnoughCtas = 222;  // one and a half for each of a B200's SMs
int64_t blocks_of(const TokenSizes &z, int run) {
  return max64(1, (z.tokens + (int64_t)run * kWarps - 1) / ((int64_t)run * kWarps));
}
int run_of(const TokenSizes &z) {
  int run = kMostRun;
  while (run > kL && z.batch * ((z.channels + 63) / 64) * blocks_of(z, run) < kEnoughCtas) run /= 2;
  return run;
}

// A pair of a sequence's channels at single tokens, those before the first among them.
template <typename T, int kTaps>
struct Row {
  const T *x;
  const T *init;   // null, or the kTaps - 1 rows before
  int64_t st;
  int channels, len;
  bool wide, second;  // pairs start at their own size; there is a second channel
  __device__ __forceinline__ float2 at(const T *p) const { return pair_at(p, wide, second); }
  __device__ __forceinline__ float2 load(int t) const {
    if (t >= 0) return t < len ? at(x + t * st) : two(0.f);
    return init && t >= -(kTaps - 1) ? at(init + (int64_t)(t + kTaps - 1) * channels) : two(0.f);
  }
};

template <int kTaps>
struct Weights {
  float2 w[kTaps], b;
  template <typename TW>
  __device__ __forceinline__ void load_as(const ConvCall &p, int c, bool second) {
    const TW *src = (const TW *)p.weight + (int64_t)c * kTaps;
#pragma unroll
    for (int j = 0; j < kTaps; ++j)
      w[j] = make_float2(to_f32(src[j]), second ? to_f32(src[kTaps + j]) : 0.f);
    b = two(0.f);
    if (p.bias) {
      const TW *bias = (const TW *)p.bias + c;
      b = make_float2(to_f32(bias[0]), second ? to_f32(bias[1]) : 0.f);
    }
  }
  __device__ __forceinline__ void load(const ConvCall &p, int c, bool second) {
    if (p.weight_dtype == LA_DTYPE_FLOAT32) load_as<float>(p, c, second);
    else load_as<__nv_bfloat16>(p, c, second);
  }
};

// The warps' mbarriers, behind the tiles.
struct Bars {
  uint64_t full[kStages][kWarps];
  int abort;
};
template <int kIn, Fetch kF, typename T>
__device__ __forceinline__ Bars &start_bars(uint8_t *smem) {
  Bars &bars = *(Bars *)(smem + kStages * kIn * kWarps * tile_elems<kF>(kL, 64) * sizeof(T));
  if (threadIdx.x == 0) {
    for (int j = 0; j < kStages; ++j)
      for (int w = 0; w < kWarps; ++w) tc::mbar_init(&bars.full[j][w], 1);
    bars.abort = 0;
    tc::fence_barrier_init();
  }
  __syncthreads();
  return bars;
}
__device__ __forceinline__ void end_bars(Bars &bars, int *err) {
  if (!bars.abort) return;
  if (err) *err = tc::kErrTimeout;
  const uint64_t since = tc::globaltimer();  // copies in flight still write into this CTA
  while (tc::globaltimer() - since < tc::kWaitTimeoutNs) __nanosleep(1000);
}

// A CTA: 64 channels, kWarps runs of `run` tokens (a multiple of kL).
template <typename T, int kTaps, bool kSilu, Fetch kF>
__global__ void __launch_bounds__(kThreads, 4)
conv_fwd_kernel(const ConvCall p, const TileLaunch l, const __grid_constant__ TileMaps maps,
                const int run, const int columns, const int blocks) {
  extern __shared__ __align__(1024) uint8_t smem[];
  Bars &bars = start_bars<1, kF, T>(smem);
  const int channels = p.sizes.channels;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int c0 = blockIdx.x % columns * 64, c = c0 + 2 * lane;
  const int64_t ib = blockIdx.x / columns / blocks;
  const int t0 = (blockIdx.x / columns % blocks * kWarps + warp) * run;
  const int end = min(t0 + run, (int)p.sizes.tokens);
  const int len = (int)sequence_length(p.lengths, p.lengths64, ib, p.sizes.tokens);
  const int whole = min(end, len);
  constexpr int kElems = tile_elems<kF>(kL, 64);
  const TokenView *views[1] = {&p.x};
  WarpTiles<T, kL, 1, kStages, kF> tiles{
      (T *)smem + warp * kElems, kWarps * kElems, kElems, &bars.full[0][warp], kWarps, views, maps.m, ib,
      c0, 64, min(64, channels - c0), l.copy, p.sizes, 0};
  // Whole tiles, and the one that the run or the sequence ends in.
  auto fetch = [&](int t, int stage) { tiles.fetch(t, whole, stage); };
#pragma unroll
  for (int j = 0; j < kStages; ++j) fetch(t0 + j * kL, j);

  const bool live = c < channels, second = c + 1 < channels;
  Row<T, kTaps> row{(const T *)p.x.p + ib * p.x.sb + c,
                    p.init ? (const T *)p.init + ib * (kTaps - 1) * channels + c : nullptr,
                    p.x.st, channels, live ? len : 0, p.wide_in, second};
  if (!live) row.init = nullptr;
  if (p.final_state && t0 == 0 && live) {
    T *dst = (T *)p.final_state + ib * (kTaps - 1) * channels + c;
#pragma unroll
    for (int j = 0; j < kTaps - 1; ++j)
      store_two(dst + (int64_t)j * channels, row.load(len - (kTaps - 1) + j), p.wide_out, second);
  }
  Weights<kTaps> w;
  w.load(p, live ? c : 0, second);
  float2 x[kTaps];  // the window; the last one is the token's own
#pragma unroll
  for (int j = 0; j < kTaps - 1; ++j) x[j + 1] = row.load(t0 - (kTaps - 1) + j);
  T *out = (T *)p.out + (ib * p.sizes.tokens + t0) * channels + c;
  auto token = [&](float2 in) {
#pragma unroll
    for (int j = 0; j < kTaps - 1; ++j) x[j] = x[j + 1];
    x[kTaps - 1] = in;
    float2 z = w.b;
#pragma unroll
    for (int j = 0; j < kTaps; ++j) z = __ffma2_rn(w.w[j], x[j], z);
    if constexpr (kSilu) z = __fmul2_rn(z, sigmoid_two<T>(z));
    return z;
  };
  int t = t0, stage = 0;
  for (; t + kL <= whole; t += kL) {
    tiles.wait(t, whole, stage, 0.f, &bars.abort);
    const T *in = tiles.tile(stage, 0) + 2 * lane;
    if (p.wide_out && live) {
#pragma unroll
      for (int k = 0; k < kL; ++k) store_two(out + (int64_t)k * channels, token(load_two(in + 64 * k)), true, true);
    } else {
#pragma unroll
      for (int k = 0; k < kL; ++k) {
        const float2 y = token(load_two(in + 64 * k));
        if (live) store_two(out + (int64_t)k * channels, y, false, second);
      }
    }
    out += (int64_t)kL * channels;
    __syncwarp();  // the tile is read
    fetch(t + kStages * kL, stage);
    if (++stage == kStages) stage = 0;
  }
  for (; t < end; t += kL) {  // where the sequence or the tensor ends
    if (t < len) tiles.wait(t, whole, stage, 0.f, &bars.abort);
    const T *in = tiles.tile(stage, 0) + 2 * lane;
    const int left = min(kL, end - t);
#pragma unroll 4
    for (int k = 0; k < left; ++k, out += channels) {
      float2 y = two(0.f);
      if (t + k < len) y = token(load_two(in + 64 * k));
      if (live) store_two(out, y, p.wide_out, second);
    }
  }
  end_bars(bars, l.err);
}

// The same.
template <typename T, int kTaps, bool kSilu, Fetch kF>
__global__ void __launch_bounds__(kThreads, 3)
conv_bwd_kernel(const ConvCall p, const TileLaunch l, const __grid_constant__ TileMaps maps,
                const int run, const int columns, const int blocks) {
  constexpr int kSums = kTaps + 1;
  __shared__ float2 part[kWarps][kSums][32];
  extern __shared__ __align__(1024) uint8_t smem[];
  column_sum_may_start();
  Bars &bars = start_bars<2, kF, T>(smem);
  const int channels = p.sizes.channels;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int c0 = blockIdx.x % columns * 64, c = c0 + 2 * lane;
  const int sums_row = blockIdx.x / columns;
  const int64_t ib = sums_row / blocks;
  const int t0 = (sums_row % blocks * kWarps + warp) * run;
  const int end = min(t0 + run, (int)p.sizes.tokens);
  const int len = (int)sequence_length(p.lengths, p.lengths64, ib, p.sizes.tokens);
  const bool first = t0 == 0;  // also ends the initial state's rows
  // Whole tiles: all tokens the run's own, none of their dx reached by the final
  // state's gradient.
  const int whole = min(end, p.d_final ? len - (kTaps - 1) : len);
  constexpr int kElems = tile_elems<kF>(kL, 64);
  const TokenView *views[2] = {&p.x, &p.d_out};
  WarpTiles<T, kL, 2, kStages, kF> tiles{
      (T *)smem + warp * 2 * kElems, kWarps * 2 * kElems, kElems, &bars.full[0][warp], kWarps, views,
      maps.m, ib, c0, 64, min(64, channels - c0), l.copy, p.sizes, 0};
  // Whole tiles, and those that the run, its neighbour's first tokens or the sequence
  // end in.
  const int reach = min(len, end + kTaps - 1);
  auto fetch = [&](int t, int stage) { tiles.fetch(t, reach, stage); };
#pragma unroll
  for (int j = 0; j < kStages; ++j) fetch(t0 + j * kL, j);

  const bool live = c < channels, second = c + 1 < channels;
  Row<T, kTaps> row{(const T *)p.x.p + ib * p.x.sb + c,
                    p.init && live ? (const T *)p.init + ib * (kTaps - 1) * channels + c : nullptr,
                    p.x.st, channels, live ? len : 0, p.wide_in, second};
  float2 sums[kSums] = {};
  Weights<kTaps> w;
  w.load(p, live ? c : 0, second);
  float2 x[kTaps], open[kTaps] = {};  // the window; dx of its tokens so far
#pragma unroll
  for (int j = 0; j < kTaps - 1; ++j) x[j + 1] = row.load(t0 - (kTaps - 1) + j);
  T *dx = (T *)p.dx + ib * p.sizes.tokens * channels + c;
  // Takes a token's x and dy; open[0] is then the gradient of the window's oldest.  Behind
  // the sequence there is no z, and its window's values are not multiplied by a zero.
  auto token = [&](float2 in, float2 g, auto own, auto inside) {
#pragma unroll
    for (int j = 0; j < kTaps - 1; ++j) x[j] = x[j + 1], open[j] = open[j + 1];
    x[kTaps - 1] = in;
    open[kTaps - 1] = two(0.f);
    if (!inside) return;
    if constexpr (kSilu) {
      float2 z = w.b;
#pragma unroll
      for (int j = 0; j < kTaps; ++j) z = __ffma2_rn(w.w[j], x[j], z);
      // s (1 + z (1 - s)) = s + z s (1 - s)
      const float2 s = sigmoid_two<T>(z);
      g = __fmul2_rn(g, __ffma2_rn(__fmul2_rn(z, s), __ffma2_rn(s, two(-1.f), two(1.f)), s));
    }
#pragma unroll
    for (int j = 0; j < kTaps; ++j) {
      open[j] = j == kTaps - 1 ? __fmul2_rn(w.w[j], g) : __ffma2_rn(w.w[j], g, open[j]);
      if (own) sums[j] = __ffma2_rn(g, x[j], sums[j]);
    }
    if (own) sums[kTaps] = __fadd2_rn(sums[kTaps], g);
  };
  int t = t0, stage = 0;
  for (; t + kL <= whole; t += kL) {
    tiles.wait(t, reach, stage, 0.f, &bars.abort);
    const T *in = tiles.tile(stage, 0) + 2 * lane, *up = tiles.tile(stage, 1) + 2 * lane;
    T *dst = dx + (int64_t)(t - (kTaps - 1)) * channels;
    auto tile = [&](auto wide) {
#pragma unroll
      for (int k = 0; k < kL; ++k) {
        token(load_two(in + 64 * k), load_two(up + 64 * k), std::true_type{}, std::true_type{});
        if (!live) continue;
        if (k >= kTaps - 1 || t > t0)
          store_two(dst + (int64_t)k * channels, open[0], wide, second);
        else if (first && p.d_init)  // (else the run before stores it)
          store_two((T *)p.d_init + (ib * (kTaps - 1) + k) * channels + c, open[0], wide, second);
      }
    };
    if (p.wide_out) tile(std::true_type{});
    else tile(std::false_type{});
    __syncwarp();  // the tile is read
    fetch(t + kStages * kL, stage);
    if (++stage == kStages) stage = 0;
  }
  if (t0 < p.sizes.tokens || first) {
    for (; t < end + kTaps - 1; t += kL) {
      const int left = min(kL, end + kTaps - 1 - t);
      tiles.wait(t, reach, stage, 0.f, &bars.abort);  // (x and dy beyond it are zero)
      const T *in = tiles.tile(stage, 0) + 2 * lane, *up = tiles.tile(stage, 1) + 2 * lane;
#pragma unroll 1
      for (int k = 0; k < left; ++k) {
        const int now = t + k, at = now - (kTaps - 1);  // whose dx is complete
        token(load_two(in + 64 * k), load_two(up + 64 * k), now < end, now < len);
        if (!live || (at < t0 && !first)) continue;
        const int back = at - (len - (kTaps - 1));  // its row of the final state
        if (p.d_final && back >= 0 && back < kTaps - 1) {
          const T *d = (const T *)p.d_final + (ib * (kTaps - 1) + back) * channels + c;
          open[0] = __fadd2_rn(open[0], pair_at(d, p.wide_in, second));
        }
        if (at >= 0)
          store_two(dx + (int64_t)at * channels, open[0], p.wide_out, second);
        else if (p.d_init)
          store_two((T *)p.d_init + (ib * (kTaps - 1) + at + kTaps - 1) * channels + c, open[0],
                    p.wide_out, second);
      }
      __syncwarp();  // the tile is read
      fetch(t + kStages * kL, stage);
      if (++stage == kStages) stage = 0;
    }
  }
  if (p.partial) {
#pragma unroll
    for (int j = 0; j < kSums; ++j) part[warp][j][lane] = sums[j];
    __syncthreads();
    float *dst = p.partial + (int64_t)sums_row * channels * kSums;
    for (int i = threadIdx.x; i < kSums * 64; i += kThreads) {
      const int j = i / 64, channel = c0 + i % 64;
      if (channel >= channels) continue;
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        const float2 v = part[k][j][i % 64 / 2];
        sum += i & 1 ? v.y : v.x;
      }
      if (j < kTaps) dst[(int64_t)channel * kTaps + j] = sum;
      else dst[(int64_t)channels * kTaps + channel] = sum;
    }
  }
  end_bars(bars, l.err);
}

template <typename T, Fetch kF, int kIn>
int make_maps(TileMaps *maps, const ConvCall &p) {
  const TokenView *views[2] = {&p.x, &p.d_out};
  for (int n = 0; kF == Fetch::kTma && n < kIn; ++n)
    if (!tile_map(&maps->m[n], *views[n], p.sizes,
                  sizeof(T) == 4 ? LA_DTYPE_FLOAT32 : LA_DTYPE_BFLOAT16, 64, kL))
      return LA_ERR_CUDA;
  return LA_OK;
}
template <typename T, Fetch kF, int kIn>
constexpr int tile_bytes() {
  return kStages * kIn * kWarps * tile_elems<kF>(kL, 64) * (int)sizeof(T) + (int)sizeof(Bars);
}

template <typename T, int kTaps, bool kSilu, Fetch kF>
int launch(const ConvCall &p, const TileLaunch &l, bool grad, cudaStream_t s) {
  const int columns = (p.sizes.channels + 63) / 64, run = run_of(p.sizes);
  const int64_t blocks = blocks_of(p.sizes, run);
  if (blocks > INT32_MAX / p.sizes.batch / columns) return LA_ERR_UNSUPPORTED;
  const unsigned grid = (unsigned)(blocks * p.sizes.batch * columns);
  TileMaps maps;
  int st = grad ? make_maps<T, kF, 2>(&maps, p) : make_maps<T, kF, 1>(&maps, p);
  if (st != LA_OK) return st;
  const int smem = grad ? tile_bytes<T, kF, 2>() : tile_bytes<T, kF, 1>();
  auto kernel = grad ? conv_bwd_kernel<T, kTaps, kSilu, kF> : conv_fwd_kernel<T, kTaps, kSilu, kF>;
  if ((st = allow_dynamic_smem((const void *)kernel, smem)) != LA_OK) return st;
  kernel<<<grid, kThreads, smem, s>>>(p, l, maps, run, columns, (int)blocks);
  return check_launch();
}
template <typename T, int kTaps, Fetch kF>
int by_silu(const ConvCall &p, const TileLaunch &l, bool grad, cudaStream_t s) {
  return p.silu ? launch<T, kTaps, true, kF>(p, l, grad, s) : launch<T, kTaps, false, kF>(p, l, grad, s);
}
template <typename T, Fetch kF>
int by_taps(const ConvCall &p, const TileLaunch &l, bool grad, cudaStream_t s) {
  if (p.taps == 2) return by_silu<T, 2, kF>(p, l, grad, s);
  if (p.taps == 3) return by_silu<T, 3, kF>(p, l, grad, s);
  return by_silu<T, 4, kF>(p, l, grad, s);
}

template <typename T>
int run_conv(ConvCall p, bool grad, cudaStream_t s) {
  constexpr int size = sizeof(T);
  const TokenView *views[2] = {&p.x, &p.d_out};
  TileLaunch l{64, 0, device_error_word()};
  const Fetch f = fetch_of(views, 2, p.sizes, size, kL, &l);
  auto at = [&](std::initializer_list<const void *> q) {
    uintptr_t bits = (uintptr_t)p.sizes.channels * size;
    for (const void *v : q) bits |= (uintptr_t)v;
    return bits % (2 * size) == 0;
  };
  p.wide_in = row_bytes(p.x, size) >= 2 * size && row_bytes(p.d_out, size) >= 2 * size &&
              at({p.init, p.d_final});
  p.wide_out = at({p.out, p.final_state, p.dx, p.d_init});
  if (f == Fetch::kTma) return by_taps<T, Fetch::kTma>(p, l, grad, s);
  if constexpr (size == 2) {
    if (f == Fetch::kShifted) return by_taps<T, Fetch::kShifted>(p, l, grad, s);
  }
  return by_taps<T, Fetch::kAsync>(p, l, grad, s);
}

}  // namespace

int64_t conv_partial_rows(const TokenSizes &z) { return z.batch * blocks_of(z, run_of(z)); }

int launch_conv_fwd(const ConvCall &p, int dtype, cudaStream_t s) {
  return dtype == LA_DTYPE_FLOAT32 ? run_conv<float>(p, false, s)
                                   : run_conv<__nv_bfloat16>(p, false, s);
}

int launch_conv_bwd(const ConvCall &p, int dtype, cudaStream_t s) {
  return dtype == LA_DTYPE_FLOAT32 ? run_conv<float>(p, true, s)
                                   : run_conv<__nv_bfloat16>(p, true, s);
}

}  // namespace la
