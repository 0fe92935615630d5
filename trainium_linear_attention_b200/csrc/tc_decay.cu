// Linear attention with a decay for each head on tcgen05 tensor cores (sm_100a):
// bf16 q/k/v with widths that are multiples of 8 up to 128.
//
// One CTA walks one (role, head, segment, 64 columns of v) in tiles of 128
// tokens (the roles and the recurrence: decay.cuh).  Per tile, with S the
// state before it, A, B, V the role's tiles, t a token's place in the walk:
//
//   scores = A B^T                       tcgen05 M=128 N=128 K=DK  -> TMEM
//   P      = intra lambda^(ti-tj) scores, tj <= ti   CUDA cores, bf16 over scores
//   O1     = A S                         M=128 N=64 K=DK  (S as a bf16 copy in smem)
//   O2     = P V                         M=128 N=64 K=128 (A = P in TMEM)
//   out    = inter lambda^(ti+e0) O1 + O2               epilogue, rounded once
//   V'     = inc lambda^(len-e0-tj) V, as two bf16 terms hi + lo    CUDA cores
//   U      = B^T [V'hi V'lo]             M=128 N=128 K=128 (, a third term N=64)
//   S      = lambda^len S + U_hi + U_lo  fp32 in registers of the state warps
//
// The decay never multiplies an accumulator in TMEM: it is on the rows of P and
// V' (operands), on O1's rows and on the state's registers, so U, the scores
// and O2 of a tile depend on the tile alone and only O1 waits for the state.
// Roundings: P and the copy of S to bf16 (half a step, 2^-8, like the output), and
// V' to hi + lo: off by 2^-14.8 at most (lo rounds what hi and the weight's own first
// term leave), 2^-17.8 in the mean square.  That is enough for a state that the
// outputs read through its bf16 copy, and stacked along N the second term costs no
// further MMA and no second read of B.  A final state, or its gradient, is asked for
// in fp32: kernels of their own (kExact) then give V' a third term, added onto the
// second's columns, in the tiles that have not decayed below 2^-10 by the walk's end
// (older ones are off by 2^-24.8 of what entered, less than half a step of fp32).
// The state is then 1e-7 off in the 2-norm, with two terms 4.2e-6, and the fp32
// formula 2.2e-7.  What it costs: 16 heads of 16384 x 128 in 121 us (two terms
// 116), 128 heads of 8192 x 64 in 111 (103), 64 heads of 2048 x 64 in 33 (26), 15
// heads of 1000 x 64 / 128 in 21 (16), where the slow heads take it in every tile.
// Kept out: the third term in place of hi once that is formed (41 us for 64 heads of
// 2048), in the same step as the others (35), exact products as four terms (34).
// With DK < 128, M = 128 holds B^T more than once (descriptor stride 0), and the
// state warps of each copy take other columns.
//
// What bounds it.  A tile moves 64 KB at d = 64 and its MMAs read ~190 KB of
// shared memory (~1,500 cycles); with its 24 warps a tile takes 2,300 to 2,600
// cycles, of which the issue slots (4,800 warp instructions on 4 schedulers)
// and the chain O1, O2 -> epilogue -> next O2 are the largest parts: 128 heads
// of 8192 x 64 in 98 us (5.5 TB/s, 84% of the copy rate), of 16 / 64 in 75 us
// (4.5 TB/s; with 128-byte key rows and three stages 83), 64 heads of 128 in 130
// us (4.1 TB/s: the two slices of v form P twice).  What that chain is sensitive
// to is code size: unrolled loops of P alone made it 1.3 times slower, and the
// code of rare cases inside the loops 5%.  Twice the epilogue or V' warps, O2 in
// two buffers, and tiles prefetched into L2 were measured and are no faster.
//
// Warps: 0 TMA; 1 scores and O1 MMAs (TMEM owner); 2 U; 3 O2; 4.. state (8 warps
// at DK = 128, else 4); 8 warps P; 4 warps V' (8 in the state pass, which has no P
// and epilogue: 16 heads of 16384 x 64 in 46 us instead of 47, their gradients in 92
// instead of 95; 8 with a third term, DK <= 64: 33 us instead of 35); 4 warps
// epilogue.  Every wait is bounded (tc_common.cuh).
#include <type_traits>

#include "decay.cuh"
#include "tc_common.cuh"
#include "tc_kernels.cuh"
#include "tma_host.cuh"

namespace la {
namespace {
using namespace tc;

constexpr int kT = kDecayTile;  // tokens per tile
constexpr int kBlock = kT * 128;  // bytes of 128 tokens x 64 bf16 columns, 128B-swizzled
constexpr float kLog2e = 1.4426950408889634f;

// TMEM columns.  P (two bf16 per column) is written over its scores.
constexpr uint32_t kColScores = 0;  // two buffers of 128
constexpr uint32_t kP1 = 64;        // P of tokens 64 .. 127 of the tile, in the buffer
constexpr uint32_t kColU = 256;     // hi 64, lo 64
constexpr uint32_t kColO1 = 384;
constexpr uint32_t kColO2 = 448;

constexpr int kJoinPitch = 65;  // floats per row of a joined state: rows in other banks

template <int DK, bool kStateOnly, bool kExact>
struct TcLayout {
  // A and B: blocks of 64 columns (128-byte rows), or one of 32 (64-byte rows)
  static constexpr int kKBlocks = DK == 32 ? 1 : DK / 64;
  static constexpr int kKBlock = DK == 32 ? kBlock / 2 : kBlock;
  static constexpr auto kKSwizzle = DK == 32 ? kSwizzle64B : kSwizzle128B;
  static constexpr int kKGroup = DK == 32 ? 512 : 1024;  // bytes of 8 tokens
  static constexpr int kStateWarps = DK == 128 ? 8 : 4;
  static constexpr int kStateCols = DK == 32 ? 16 : 32;  // columns of S per thread
  static constexpr int kWState = 4;
  static constexpr int kWP = kWState + kStateWarps;  // first P warp
  static constexpr int kWV = kStateOnly ? kWP : kWP + 8;
  static constexpr int kVWarps = kStateOnly || (kExact && DK <= 64) ? 8 : 4;
  static constexpr int kWE = kWV + kVWarps;
  static constexpr int kWarps = kStateOnly ? kWE : kWE + 4;
  static constexpr int kThreads = kWarps * 32;
  // stage: A, B (kKBlocks blocks each), V (one block)
  static constexpr uint32_t kOffA = 0;
  static constexpr uint32_t kOffB = kStateOnly ? 0 : kKBlocks * kKBlock;
  static constexpr uint32_t kOffV = kOffB + kKBlocks * kKBlock;
  static constexpr uint32_t kStageBytes = kOffV + kBlock;
  static constexpr uint32_t kSnapBytes = DK * 128;
  // V': two terms of a tile or, kExact, three; of two tiles where the space allows it
  static constexpr int kVpBlocks = !kExact ? (DK <= 64 || kStateOnly ? 4 : 2)
                                   : DK == 32 || (kStateOnly && DK == 64) ? 6
                                   : DK == 64 || kStateOnly               ? 4
                                                                          : 3;
  static constexpr uint32_t kVpBytes = kVpBlocks * kBlock;
  // Whether tiles of three terms, or of two, alternate between two places, and where
  // tile c's are.
  static __device__ __forceinline__ bool vp_two(bool third) {
    return kVpBlocks == 6 || (kVpBlocks == 4 && !third);
  }
  static __device__ __forceinline__ uint32_t vp_at(int c, bool third) {
    return vp_two(third) ? (c & 1) * (kVpBytes / 2) : 0;
  }
  static constexpr int kSnaps = kStateOnly ? 0 : kExact && DK == 128 ? 1 : 2;  // copies of S
  static constexpr int kUBufs = kStateOnly ? 2 : 1;
  static constexpr uint32_t kFixed = kVpBytes + kSnaps * kSnapBytes + 512;
  static constexpr int kStages = (227 * 1024 - 1024 - (int)kFixed) / (int)kStageBytes > 6
                                     ? 6
                                     : (227 * 1024 - 1024 - (int)kFixed) / (int)kStageBytes;
  static constexpr uint32_t kOffVp = kStages * kStageBytes;  // V' hi, lo, the third term
  static constexpr uint32_t kOffSnap = kOffVp + kVpBytes;    // bf16 copies of S
  static constexpr uint32_t kOffBar = kOffSnap + kSnaps * kSnapBytes;
  static constexpr uint32_t kSmem = kOffBar + 512 + 1024;  // + alignment
  static constexpr int kJoinBytes = DK * kJoinPitch * 4;  // a joined state, from kOffVp on
  // Whether it reaches beyond V' into the copies of S, as with DK = 128 its last two
  // rows do: a state warp then may write its copy only once all have read theirs.
  static constexpr bool kJoinOverCopies = kJoinBytes > (int)kVpBytes;
  static_assert(kStateOnly || kJoinBytes <= (int)(kVpBytes + kSnaps * kSnapBytes), "joined state");
  static_assert(kStages >= 2 && kSmem <= 227 * 1024, "shared memory budget");
  static_assert(kSmem > 114 * 1024, "one CTA per SM (all TMEM columns)");
};

enum Bar {
  kFull = 0,
  kEmpty = kFull + 6,
  kSReady = kEmpty + 6,
  kPReady = kSReady + 2,
  kSnapReady = kPReady + 2,
  kRead = kSnapReady + 2,  // O1 formed: the copy of S is free
  kVpReady = kRead + 2,
  kUReady = kVpReady + 2,  // alternate tiles: V' may run a tile ahead of its readers
  kUFree = kUReady + 2,
  kOReady = kUFree + 2,
  kOFree = kOReady + 2,
  kDone = kOFree + 2,
  kThird = kDone + 3,  // the third term of V', where it has one; alternate tiles
  kNumBars = kThird + 2
};
static_assert(8 * kNumBars + 8 <= 512, "barrier area");

constexpr int kMaxMaps = 8;  // four tensors, in boxes of 64 columns and of 32

struct TcRole {
  int a, b, v;  // which tensor map
  __nv_bfloat16 *out;
  int64_t ob, oh, ot;
  const float *init;
  float *states, *final_state;
  int da, dvo, transposed, reverse;
  float intra, inter, inc;
};

struct TcParams {
  CUtensorMap map[kMaxMaps];
  TcRole role[kDecayMaxRoles];
  const float *log_decay;
  int *err;
  int64_t heads, n;
  // heads [0, whole) are walked by one CTA per role and slice, the others in
  // segments; a state pass walks all but the last of those
  int64_t whole, seg_len;
  int lead;  // 0, or the tiles of the first of two parts (decay.cuh)
  int roles, slices, segments, orders;
};

__device__ __forceinline__ void tma_load_4d(void *smem_dst, const CUtensorMap *map, uint64_t *bar,
                                            int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// 2^x by the hardware approximation (relative error ~2^-22); only ahead of a
// rounding to bf16.
__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t hfma2_bf16(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}

__device__ __forceinline__ bool wait_teardown(uint64_t *bar, uint32_t parity) {
  const uint64_t t0 = globaltimer();
  while (!mbar_try_wait(bar, parity))
    if (globaltimer() - t0 > kWaitTimeoutNs) return false;
  return true;
}

template <int DK, bool kStateOnly, bool kLead, bool kExact>
__global__ void __launch_bounds__(TcLayout<DK, kStateOnly, kExact>::kThreads, 1)
decay_tc_kernel(const __grid_constant__ TcParams p) {
  using L = TcLayout<DK, kStateOnly, kExact>;
  constexpr int kStages = L::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t sb = smem_u32(smem);
  uint64_t *bars = (uint64_t *)(smem + L::kOffBar);
  uint32_t *tmem_slot = (uint32_t *)(smem + L::kOffBar + 8 * kNumBars);
  volatile int *abort_flag = (volatile int *)(smem + L::kOffBar + 8 * kNumBars + 4);

  // roles fastest, then slices: CTAs that read the same tokens run together;
  // whole heads first, so that the shorter walks of the split ones end the grid
  uint32_t id = blockIdx.x;
  const TcRole &role = p.role[id % p.roles];
  id /= p.roles;
  const int c0 = (int)(id % p.slices) * kDecaySlice;
  id /= p.slices;
  const bool split = kStateOnly || id >= p.whole;
  if (split && !kStateOnly) id -= (uint32_t)p.whole;
  const int segments = split ? p.segments : 1;
  const int order = split ? (int)(id % p.orders) : 0;
  const int64_t head_at = split ? id / p.orders : 0;  // of the split heads
  const int64_t bh = split ? p.whole + head_at : id;
  const int64_t seg_len = split ? p.seg_len : p.n;
  if (c0 >= role.dvo) return;
  const int ib = (int)(bh / p.heads), ih = (int)(bh % p.heads);
  const bool rev = role.reverse != 0;
  const int e0 = rev ? 0 : 1;
  // two parts without a state pass: a kernel of its own, since its few instructions
  // more made the other walks 2 to 4% slower
  const int pre = kLead && order > 0 ? p.lead : 0;  // tiles walked for the state alone
  const bool joins = !kStateOnly && !kLead && order > 0;
  const int64_t part = (int64_t)p.lead * kT;
  const int64_t t0 = !kLead ? (int64_t)(rev ? segments - 1 - order : order) * seg_len
                     : rev && order == 0 ? (p.n + kT - 1) / kT * kT - part : 0;
  const int64_t t1 = !kLead ? min64(p.n, t0 + seg_len) : rev || order > 0 ? p.n : part;
  const int tiles = (int)((t1 - t0 + kT - 1) / kT);
  const bool want_final =
      kStateOnly || (role.final_state != nullptr && order == segments - 1);
  // tiles whose U is needed: the last one's only for the final state
  const int outs = tiles - pre;  // tiles of the output
  const int updates = want_final ? tiles : (tiles > 0 ? tiles - 1 : 0);
  const float g = p.log_decay[ih];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // first token of the walk's tile c; its tokens: 128 but for the ragged tile,
  // which is the walk's last, in a reversed walk its first
  auto tile_start = [&](int c) { return t0 + (int64_t)(rev ? tiles - 1 - c : c) * kT; };
  const int ragged = rev ? 0 : tiles - 1;
  const int ragged_len = (int)(t1 - t0) - (tiles - 1) * kT;
  // Where the final state is written, the first tile whose V' has three terms: from
  // there on lambda^(tokens to the walk's end) is above 2^-10.  (The first of two
  // parts does as a whole walk would, so that its outputs have the same bits.)
  int third_from = INT32_MAX;
  if (kExact && role.final_state != nullptr && (want_final || kLead) &&
      (g != 0.f || role.inc != 1.f)) {  // (weights of one need no more)
    const int64_t reach = (int64_t)fminf(6.94f / fabsf(g), 2e9f);
    if (!rev)
      third_from = (int)((max64(0, p.n - kT - t0 - reach) + kT - 1) / kT);
    else if (reach >= t0)
      third_from = (int)max64(0, tiles - 1 - (reach - t0) / kT);
  }

  if (threadIdx.x == 0) {
    for (int i = 0; i < kNumBars; ++i) {
      const bool per_state_warp = i == kSnapReady || i == kSnapReady + 1 ||
                                  i == kUFree || i == kUFree + 1;
      const bool per_v_warp = i == kVpReady || i == kVpReady + 1 || i == kThird || i == kThird + 1;
      const bool per_four = i == kOFree || i == kOFree + 1;
      const bool per_p_warp = i == kPReady || i == kPReady + 1;
      const bool stage_empty = i >= kEmpty && i < kEmpty + 6;
      mbar_init(&bars[i], per_state_warp ? L::kStateWarps
                          : per_v_warp   ? L::kVWarps
                          : per_four     ? 4
                          : per_p_warp   ? 8
                          : stage_empty  ? (kStateOnly ? 1 : 2)
                                         : 1);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  // The state that a later segment starts with, joined by the whole CTA in the
  // space of V' and the copies of S:
  //   lambda^(tokens so far) init + sum_o lambda^(tokens from o's end on) states_o
  float *joined = (float *)(smem + L::kOffVp);
  if (joins) {
    constexpr int kEach = (DK * 64 + L::kThreads - 1) / L::kThreads;
    const int64_t per_head = (int64_t)role.da * role.dvo;
    // neighbouring threads read neighbouring addresses: columns first, or rows
    // where the states are stored transposed
    int64_t at[kEach];
    float sum[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int i = threadIdx.x + e * L::kThreads;
      const int row = role.transposed ? i % DK : i / 64, col = role.transposed ? i / DK : i % 64;
      const bool in = i < DK * 64 && row < role.da && c0 + col < role.dvo;
      at[e] = !in              ? -1
              : role.transposed ? (int64_t)(c0 + col) * role.da + row
                                : (int64_t)row * role.dvo + c0 + col;
      sum[e] = 0.f;
    }
    int after = 0;  // tokens from the end of segment o to this one's start
    grid_dependency_wait();  // the state pass has written its states
#pragma unroll 2
    for (int o = order - 1; o >= 0; --o) {
      const float keep = decay_pow(g, after);
      const float *src = role.states + (head_at * segments + o) * per_head;
#pragma unroll
      for (int e = 0; e < kEach; ++e)
        if (at[e] >= 0) sum[e] = fmaf(keep, __ldcg(src + at[e]), sum[e]);
      after += segment_tokens(o, rev, segments, seg_len, p.n);
    }
    if (role.init) {
      const float keep = decay_pow(g, after);
#pragma unroll
      for (int e = 0; e < kEach; ++e)
        if (at[e] >= 0) sum[e] = fmaf(keep, role.init[bh * per_head + at[e]], sum[e]);
    }
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int i = threadIdx.x + e * L::kThreads;
      const int row = role.transposed ? i % DK : i / 64, col = role.transposed ? i / DK : i % 64;
      if (i < DK * 64) joined[row * kJoinPitch + col] = sum[e];
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0) {
      const CUtensorMap *ma = &p.map[role.a], *mb = &p.map[role.b], *mv = &p.map[role.v];
      if (!kStateOnly) prefetch_tmap(ma);
      prefetch_tmap(mb);
      prefetch_tmap(mv);
      int c = 0;
      for (; c < tiles; ++c) {
        const int s = c % kStages;
        if (c >= kStages && !mbar_wait(&bars[kEmpty + s], ((c / kStages) - 1) & 1, abort_flag))
          break;
        const int y = (int)tile_start(c);
        uint8_t *st = smem + s * L::kStageBytes;
        const bool with_a = !kStateOnly && (!kLead || c >= pre);
        mbar_arrive_expect_tx(&bars[kFull + s],
                              kStateOnly || with_a ? L::kStageBytes : L::kStageBytes - L::kOffB);
#pragma unroll
        for (int b = 0; b < L::kKBlocks; ++b) {
          tma_load_4d(st + L::kOffB + b * L::kKBlock, mb, &bars[kFull + s], 64 * b, y, ih, ib);
          if (with_a)
            tma_load_4d(st + L::kOffA + b * L::kKBlock, ma, &bars[kFull + s], 64 * b, y, ih, ib);
        }
        tma_load_4d(st + L::kOffV, mv, &bars[kFull + s], c0, y, ih, ib);
      }
      // every issued copy must land before the CTA can exit
      for (int i = c - kStages < 0 ? 0 : c - kStages; i < c; ++i)
        wait_teardown(&bars[kFull + i % kStages], (i / kStages) & 1);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------- scores and O1 = A S
    // Three warps issue MMAs: one instruction of a warp takes ten cycles and more
    // here, so a tile's 24 to 32 MMAs with their waits are too long for one.
    if constexpr (!kStateOnly) {
      constexpr uint32_t id_s = make_idesc_bf16(128, 128, false, false);
      constexpr uint32_t id_o = make_idesc_bf16(128, 64, false, true);
      const int k_steps = (role.da + 15) / 16;  // the columns beyond are zero
      const uint64_t a0 = make_sdesc(sb + L::kOffA, 16, L::kKGroup, L::kKSwizzle);
      const uint64_t b0 = make_sdesc(sb + L::kOffB, 16, L::kKGroup, L::kKSwizzle);
      const uint64_t s0 = make_sdesc(sb + L::kOffSnap, 16, 1024, kSwizzle128B);
      int ss = pre % kStages, sp = (pre / kStages) & 1;  // stage of the next scores, its phase
      auto issue_scores = [&](int c) -> bool {
        if (!mbar_wait_warp(&bars[kFull + ss], sp, abort_flag)) return false;
        // the buffer: P of tile c - 2 has been read by P V
        if (c >= 2 && !mbar_wait_warp(&bars[kOReady + (c & 1)], ((c - 2) / 2) & 1, abort_flag))
          return false;
        tc_fence_after();
        const uint64_t at = (uint64_t)(ss * (L::kStageBytes >> 4));
        const uint32_t d = tmem + kColScores + (c & 1) * 128;
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < DK / 16; ++kk) {  // 32 bytes along the rows
            const uint64_t step = at + (uint64_t)((kk / 4) * (L::kKBlock >> 4) + (kk % 4) * 2);
            if (kk < k_steps) umma_ss(d, a0 + step, b0 + step, id_s, kk > 0);
          }
          umma_commit(&bars[kSReady + (c & 1)]);
        }
        __syncwarp();
        if (++ss == kStages) ss = 0, sp ^= 1;
        return true;
      };
      // behind tiles walked for the state alone a stage's phase tells the first tile
      // from those before it only once they are done: when the state is ready
      bool ok = outs > 0 &&
                (!kLead || pre == 0 || mbar_wait_warp(&bars[kSnapReady], 0, abort_flag)) && issue_scores(0);
      int rs = pre % kStages;  // stage of tile c
      for (int c = 0; ok && c < outs; ++c) {
        const int b = c & 1;
        // the next tile's scores go first if nothing holds them up
        const bool early =
            c + 1 < outs &&
            __all_sync(0xffffffffu,
                       mbar_test_wait(&bars[kFull + ss], sp) &&
                           (c == 0 || mbar_test_wait(&bars[kOReady + (b ^ 1)], ((c - 1) / 2) & 1)));
        if (early && !issue_scores(c + 1)) break;
        if (!mbar_wait_warp(&bars[kSnapReady + b], (c / 2) & 1, abort_flag)) break;
        if (c > 0 && !mbar_wait_warp(&bars[kOFree + (b ^ 1)], ((c - 1) / 2) & 1, abort_flag)) break;
        tc_fence_after();
        const uint64_t at = (uint64_t)(rs * (L::kStageBytes >> 4));
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < DK / 16; ++kk)
            if (kk < k_steps)
              umma_ss(tmem + kColO1,
                      a0 + at + (uint64_t)((kk / 4) * (L::kKBlock >> 4) + (kk % 4) * 2),
                      s0 + (uint64_t)(c % L::kSnaps * (L::kSnapBytes >> 4) + kk * (2048 >> 4)), id_o,
                      kk > 0);
          umma_commit(&bars[kRead + b]);
        }
        __syncwarp();
        if (++rs == kStages) rs = 0;
        if (c + 1 < outs && !early && !issue_scores(c + 1)) break;
      }
      if (elect_one()) umma_commit(&bars[kDone]);
      __syncwarp();
      if (lane == 0) wait_teardown(&bars[kDone], 0);
      __syncwarp();
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------ U = B^T V'
    constexpr uint32_t id_u = make_idesc_bf16(128, 128, true, true);
    // A = B^T: M's 128 rows are two blocks of 64 columns, or with DK < 128 the
    // same columns over again
    const uint64_t a0 =
        make_sdesc(sb + L::kOffB, DK == 128 ? kBlock : 0, L::kKGroup, L::kKSwizzle);
    const uint64_t b0 = make_sdesc(sb + L::kOffVp, kBlock, 1024, kSwizzle128B);
    int us = 0, up = 0;  // stage and its phase
    for (int c = 0; c < updates; ++c) {
      const bool third = kExact && c >= third_from;
      if (!mbar_wait_warp(&bars[kFull + us], up, abort_flag)) break;
      if (!mbar_wait_warp(&bars[kVpReady + (c & 1)], (c / 2) & 1, abort_flag)) break;
      // the columns: U of tile c - 1 (with two buffers c - 2) is in registers
      if (c >= L::kUBufs) {
        const int u = c - L::kUBufs;
        if (!mbar_wait_warp(&bars[kUFree + (u & 1)], (u / 2) & 1, abort_flag)) break;
      }
      tc_fence_after();
      const uint32_t d = tmem + kColU + (c % L::kUBufs) * 128;
      const uint64_t da = a0 + (uint64_t)(us * (L::kStageBytes >> 4));
      const uint64_t db = b0 + (uint64_t)(L::vp_at(c, third) >> 4);
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < kT / 16; ++kk) {
          umma_ss(d, da + (uint64_t)(kk * (2 * L::kKGroup >> 4)),
                  db + (uint64_t)(kk * (2048 >> 4)), id_u, kk > 0);
        }
        if (!third) umma_commit(&bars[kUReady + (c & 1)]);
      }
      __syncwarp();
      if (third) {  // onto the second's columns
        if (!mbar_wait_warp(&bars[kThird + (c & 1)], ((c - third_from) / 2) & 1, abort_flag)) break;
        tc_fence_after();
        constexpr uint32_t id_third = make_idesc_bf16(128, 64, true, true);
        if (elect_one()) {
#pragma unroll 1
          for (int kk = 0; kk < kT / 16; ++kk)
            umma_ss(d + 64, da + (uint64_t)(kk * (2 * L::kKGroup >> 4)),
                    db + (uint64_t)((2 * kBlock >> 4) + kk * (2048 >> 4)), id_third, true);
          umma_commit(&bars[kUReady + (c & 1)]);
        }
        __syncwarp();
      }
      if (++us == kStages) us = 0, up ^= 1;
    }
    if (elect_one()) umma_commit(&bars[kDone + 1]);
    __syncwarp();
    if (lane == 0) wait_teardown(&bars[kDone + 1], 0);
    __syncwarp();
  } else if (warp == 3) {
    // ------------------------------------------------------------ O2 = P V
    if constexpr (!kStateOnly) {
      constexpr uint32_t id_o = make_idesc_bf16(128, 64, false, true);
      const uint64_t v0 = make_sdesc(sb + L::kOffV, 16, 1024, kSwizzle128B);
      int vs = pre % kStages, vp = (pre / kStages) & 1;  // stage and its phase
      for (int c = 0; c < outs; ++c) {
        const int b = c & 1;
        // (with tiles before the output's P first: it is behind the scores)
        if (kLead && !mbar_wait_warp(&bars[kPReady + b], (c / 2) & 1, abort_flag)) break;
        if (!mbar_wait_warp(&bars[kFull + vs], vp, abort_flag)) break;
        if (!kLead && !mbar_wait_warp(&bars[kPReady + b], (c / 2) & 1, abort_flag)) break;
        // the columns: O2 of tile c - 1 has been read out
        if (c > 0 && !mbar_wait_warp(&bars[kOFree + (b ^ 1)], ((c - 1) / 2) & 1, abort_flag)) break;
        tc_fence_after();
        const uint64_t dv = v0 + (uint64_t)(vs * (L::kStageBytes >> 4));
        const uint32_t buf = tmem + kColScores + b * 128;
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < kT / 16; ++kk)
            umma_ts(tmem + kColO2, buf + (kk / 4) * kP1 + (kk % 4) * 8,
                    dv + (uint64_t)(kk * (2048 >> 4)), id_o, kk > 0);
          umma_commit(&bars[kOReady + b]);
        }
        __syncwarp();
        if (++vs == kStages) vs = 0, vp ^= 1;
      }
      if (elect_one()) umma_commit(&bars[kDone + 2]);
      __syncwarp();
      if (lane == 0) wait_teardown(&bars[kDone + 2], 0);
      __syncwarp();
    }
  } else if (warp >= L::kWState && warp < L::kWP) {
    // ------------------------------------------------------------ state
    // A thread owns kCols columns of one row of S; where TMEM's lanes hold the
    // rows more than once, each copy's warps take other columns.
    constexpr int kCols = L::kStateCols;
    const int wq = warp & 3;  // TMEM lane quarter
    const int row = DK == 32 ? lane : DK == 64 ? (wq & 1) * 32 + lane : wq * 32 + lane;
    const int part = DK == 32 ? wq : DK == 64 ? wq >> 1 : (warp - L::kWState) >> 2;
    const int col = c0 + part * kCols;
    float st[kCols];
    const int64_t per_head = (int64_t)role.da * role.dvo;
    const bool mine = row < role.da;
    const int cols = mine ? min(kCols, role.dvo - col) : 0;  // may be negative
#pragma unroll
    for (int i = 0; i < kCols; ++i) st[i] = 0.f;
    if constexpr (kStateOnly) {
      grid_dependents_launch();
    } else if (joins) {
      const float *src = joined + row * kJoinPitch + part * kCols;
#pragma unroll
      for (int i = 0; i < kCols; ++i) st[i] = src[i];
      // V' may take the space, and the copies of S what lies in theirs
      if constexpr (L::kJoinOverCopies) named_barrier_sync(1, L::kStateWarps * 32 + L::kVWarps * 32);
      else named_barrier_arrive(1, L::kStateWarps * 32 + L::kVWarps * 32);
    } else if (role.init) {
      const int64_t step = role.transposed ? role.da : 1;
      const float *src = role.init + bh * per_head + (role.transposed ? (int64_t)col * role.da + row
                                                                      : (int64_t)row * role.dvo + col);
#pragma unroll
      for (int i = 0; i < kCols; ++i)
        if (i < cols) st[i] = src[i * step];
    }
    const float keep_full = decay_pow(g, kT), keep_ragged = decay_pow(g, ragged_len);
    const uint64_t minus2 = f2pack(-1.f, -1.f);
    const uint32_t copy_row = sb + L::kOffSnap + sw128_offset(row, part * (kCols / 8));
    int stage = 0;
#pragma unroll 1
    for (int c = 0;; ++c) {
      if (!kStateOnly && (!kLead || c >= pre) && c < tiles) {  // the copy of S that tile c reads
        const int at = c - pre, b = at & 1, read = at - L::kSnaps;
        if (read >= 0) mbar_wait(&bars[kRead + (read & 1)], (read / 2) & 1, abort_flag);
        __syncwarp();
        const uint32_t dst = copy_row + (L::kSnaps > 1 ? b * L::kSnapBytes : 0);
#pragma unroll
        for (int q = 0; q < kCols / 8; ++q)
          st_shared_v4(dst ^ (16 * q), pack_bf16(st[8 * q], st[8 * q + 1]),
                       pack_bf16(st[8 * q + 2], st[8 * q + 3]),
                       pack_bf16(st[8 * q + 4], st[8 * q + 5]),
                       pack_bf16(st[8 * q + 6], st[8 * q + 7]));
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[kSnapReady + b]);
      }
      if (c >= updates) break;
      const float keep = c == ragged ? keep_ragged : keep_full;
      const uint64_t keep2 = f2pack(keep, keep);
      mbar_wait(&bars[kUReady + (c & 1)], (c / 2) & 1, abort_flag);
      // B and V of the tile's stage have been read by U (and V')
      if (warp == L::kWState && lane == 0) {
        mbar_arrive(&bars[kEmpty + stage]);
        if (kLead && c < pre) mbar_arrive(&bars[kEmpty + stage]);  // for the epilogue
      }
      if (++stage == kStages) stage = 0;
      __syncwarp();
      tc_fence_after();
      const uint32_t urow = taddr(tmem, wq * 32, kColU + (c % L::kUBufs) * 128 + part * kCols);
#pragma unroll
      for (int q = 0; q < kCols / 8; ++q) {
        uint32_t hi[8], lo[8];
        tmem_ld8(urow + 8 * q, hi);
        tmem_ld8(urow + 64 + 8 * q, lo);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const uint64_t u =
              ffma2(f2pack(__uint_as_float(lo[i]), __uint_as_float(lo[i + 1])), minus2,
                    f2pack(__uint_as_float(hi[i]), __uint_as_float(hi[i + 1])));
          f2unpack(ffma2(keep2, f2pack(st[8 * q + i], st[8 * q + i + 1]), u), st[8 * q + i],
                   st[8 * q + i + 1]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[kUFree + (c & 1)]);
    }
    if (want_final) {
      float *dst = (kStateOnly ? role.states + (head_at * segments + order) * per_head
                               : role.final_state + bh * per_head) +
                   (int64_t)row * role.dvo + col;
#pragma unroll
      for (int i = 0; i < kCols; ++i)
        if (i < cols) dst[i] = st[i];
    }
  } else if (!kStateOnly && warp >= L::kWP && warp < L::kWV) {
    // ------------------------------------------------------------ P
    // Two warps per lane quarter, 64 columns each; P takes the first 32 TMEM
    // columns of its own half, so no warp writes what another still reads.
    const int half = (warp - L::kWP) >> 2;
    const int wq = warp & 3;
    // finite, so that 0 * g2 = 0 (e^-6900 is zero like e^-inf)
    const float g2 = fmaxf(g * kLog2e, -1e4f);
    const int sign = rev ? -1 : 1;
    // lambda^lag over 16 columns j0 + t: f = lambda^(i-j0-15) times w = lambda^(15-t),
    // in a reversed walk lambda^(j0-i) * lambda^t.  Off the diagonal both powers
    // are non-negative; on it the first reaches -15, which fp32 holds while
    // |g| <= 4, and the columns with lag < 0 are cut from the packed words.  The two
    // are multiplied before they meet the score, which lambda^15 alone (e^-60) could
    // take below fp32's range.
    const bool mild = g >= -4.f && g <= 4.f;
    const int off = rev ? 0 : 15;
    const int row_lag = (wq * 32 + lane - 64 * half) * sign;  // lag of the warp's first column
    uint64_t w2[8];
    uint32_t cut[2][8];
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const int n0 = rev ? 2 * t : 15 - 2 * t, n1 = rev ? 2 * t + 1 : 14 - 2 * t;
      w2[t] = f2pack(decay_pow(g, n0) * role.intra, decay_pow(g, n1) * role.intra);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int lag = rev ? 16 * q - lane + 2 * t : lane - 16 * q - 2 * t;
        cut[q][t] = (lag >= 0 ? 0xFFFFu : 0u) | (lag - sign >= 0 ? 0xFFFF0000u : 0u);
      }
    }
    // the warp's two blocks of 32 columns: before, on or beyond the diagonal
    const int side0 = (2 * half - wq) * sign, side1 = (2 * half + 1 - wq) * sign;
    auto walk = [&](auto is_mild) {
      for (int c = 0; c < outs; ++c) {
        const uint32_t srow0 = taddr(tmem, wq * 32, kColScores + (c & 1) * 128 + half * 64);
        mbar_wait(&bars[kSReady + (c & 1)], (c / 2) & 1, abort_flag);
        __syncwarp();
        tc_fence_after();
        // Rolled, like the other loops here: the warps of a scheduler run six
        // different ones, and where those did not fit its instruction cache
        // together the kernel took 1.3 times as long.
#pragma unroll 1
        for (int ch = 0; ch < 2; ++ch) {
          const int side = ch ? side1 : side0;
          if (side > 0) {  // beyond the diagonal
            uint32_t z[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) z[i] = 0;
            tmem_st16(srow0 + 16 * ch, z);
            continue;
          }
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int lag = row_lag - sign * (32 * ch + 16 * q);  // of the first column
            uint32_t x[16], pk[8];
            tmem_ld16(srow0 + 32 * ch + 16 * q, x);
            tmem_wait_ld();
            if (decltype(is_mild)::value || side < 0) {
              // (below -15 every column is cut)
              const float f = ex2_approx((float)max(lag - off, -15) * g2);
              const uint64_t f2 = f2pack(f, f);
#pragma unroll
              for (int t = 0; t < 8; ++t)
                pk[t] = pack_bf16x2(
                    fmul2(f2pack(__uint_as_float(x[2 * t]), __uint_as_float(x[2 * t + 1])),
                          fmul2(w2[t], f2)));
            } else {  // strong decays: each column its own power
              float l = (float)lag;
#pragma unroll
              for (int t = 0; t < 8; ++t) {
                const float y0 = __uint_as_float(x[2 * t]) * (role.intra * ex2_approx(l * g2));
                l -= (float)sign;
                const float y1 = __uint_as_float(x[2 * t + 1]) * (role.intra * ex2_approx(l * g2));
                l -= (float)sign;
                pk[t] = pack_bf16(y0, y1);
              }
            }
            if (side == 0) {
#pragma unroll
              for (int t = 0; t < 8; ++t) pk[t] &= cut[q][t];
            }
            tmem_st8(srow0 + 16 * ch + 8 * q, pk);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[kPReady + (c & 1)]);
      }
    };
    // (two loops, so that the rare one's code does not lie inside the other)
    if (mild) walk(std::true_type{});
    else walk(std::false_type{});
  } else if (warp >= L::kWV && warp < L::kWE) {
    // ------------------------------------------------------------ V' = hi + lo
    const int j = ((warp - L::kWV) & 3) * 32 + lane;  // token of the tile
    constexpr uint32_t kPart = 512 / L::kVWarps;      // bytes of its row
    const uint32_t q0 = (uint32_t)((warp - L::kWV) >> 2) * kPart;
    // tokens from this one to the tile's end; in a reversed walk the tile ends at
    // its first token, and the state there decays once more
    const float w_full = role.inc * decay_pow(g, rev ? j + 1 : kT - 1 - j);
    const float w_ragged = role.inc * decay_pow(g, rev ? j + 1 : ragged_len - 1 - j);
    const uint32_t row = sb + sw128_offset(j, 0);
    int s = 0, phase = 0;
    if (joins) named_barrier_sync(1, L::kStateWarps * 32 + L::kVWarps * 32);
    for (int c = 0; c < updates; ++c) {
      const float w = c == ragged ? w_ragged : w_full;
      // w as two bf16 terms; with x * w_hi rounded to hi, the rest of that
      // product is a bf16 value and fma gives it exactly: three packed
      // instructions per two values.  They leave -lo, which the state warps
      // subtract.
      const uint32_t w_hi = pack_bf16(w, w);
      const float rest = bf16lo(w_hi) - w;
      const uint32_t minus_hi = w_hi ^ 0x80008000u, minus_lo = pack_bf16(rest, rest);
      mbar_wait(&bars[kFull + s], phase, abort_flag);
      // U of the tile that used this place before has been formed
      const bool third = kExact && c >= third_from;
      const int u = c - (L::vp_two(third) ? 2 : 1);
      if (u >= 0) mbar_wait(&bars[kUReady + (u & 1)], (u / 2) & 1, abort_flag);
      __syncwarp();
      const uint32_t src = row + s * L::kStageBytes + L::kOffV,
                     dst = row + L::kOffVp + L::vp_at(c, third);
#pragma unroll 2
      for (uint32_t q = q0; q < q0 + kPart; q += 16) {  // a piece of the row: its swizzle is an xor
        uint32_t x[4], hi[4], lo[4];
        ld_shared_v4(src ^ q, x[0], x[1], x[2], x[3]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          hi[i] = hmul2_bf16(x[i], w_hi);
          lo[i] = hfma2_bf16(x[i], minus_lo, hfma2_bf16(x[i], minus_hi, hi[i]));
        }
        st_shared_v4(dst ^ q, hi[0], hi[1], hi[2], hi[3]);
        st_shared_v4((dst ^ q) + kBlock, lo[0], lo[1], lo[2], lo[3]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[kVpReady + (c & 1)]);
      if (third) {
        // what the two leave of w x (fma: to 2^-32 of it), rounded to bf16, while they
        // are on their way into U; negative, like lo
        const uint64_t w2 = f2pack(w, w);
#pragma unroll 2
        for (uint32_t q = q0; q < q0 + kPart; q += 16) {
          uint32_t x[4], hi[4], lo[4];
          ld_shared_v4(src ^ q, x[0], x[1], x[2], x[3]);
          ld_shared_v4((dst ^ q) + kBlock, lo[0], lo[1], lo[2], lo[3]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            hi[i] = hmul2_bf16(x[i], minus_hi);
            const uint64_t left = ffma2(f2pack(bf16lo(x[i]), bf16hi(x[i])), w2,
                                        f2pack(bf16lo(hi[i]), bf16hi(hi[i])));
            x[i] = pack_bf16x2(fadd2(left, f2pack(bf16lo(lo[i]), bf16hi(lo[i])))) ^ 0x80008000u;
          }
          st_shared_v4((dst ^ q) + 2 * kBlock, x[0], x[1], x[2], x[3]);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[kThird + (c & 1)]);
      }
      if (++s == kStages) s = 0, phase ^= 1;
    }
  } else if (!kStateOnly && warp >= L::kWE) {
    // ------------------------------------------------------------ epilogue
    const int wq = warp & 3;
    const int r = wq * 32 + lane;
    const float f_full = role.inter * decay_pow(g, (rev ? kT - 1 - r : r) + e0);
    const float f_ragged = role.inter * decay_pow(g, (rev ? ragged_len - 1 - r : r) + e0);
    const int odd = lane & 1;
    const int row0 = r & ~1;
    const int64_t ot = role.ot;
    // columns from this lane's first on, a multiple of 8
    const int columns = role.dvo - c0 - 16 * odd;
    __nv_bfloat16 *dst = role.out + ib * role.ob + ih * role.oh + (tile_start(pre) + row0) * ot + c0 +
                         16 * odd;
    const int64_t tile_step = (rev ? -kT : kT) * ot;
    const uint32_t o1 = taddr(tmem, wq * 32, kColO1), o2 = taddr(tmem, wq * 32, kColO2);
    auto walk = [&](auto is_wide) {
      int stage = pre % kStages;
      for (int c = 0; c < outs; ++c, dst += tile_step) {
        const int len = c + pre == ragged ? ragged_len : kT;
        const float f = c + pre == ragged ? f_ragged : f_full;
        const uint64_t f2 = f2pack(f, f);
        mbar_wait(&bars[kRead + (c & 1)], (c / 2) & 1, abort_flag);
        mbar_wait(&bars[kOReady + (c & 1)], (c / 2) & 1, abort_flag);
        // the tile's scores, A S and P V are done with its stage
        if (wq == 0 && lane == 0) mbar_arrive(&bars[kEmpty + stage]);
        if (++stage == kStages) stage = 0;
        __syncwarp();
        tc_fence_after();
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {  // 32 columns
          uint32_t w[16];
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            uint32_t x[16], y[16];
            tmem_ld16(o1 + 32 * h + 16 * q, x);
            tmem_ld16(o2 + 32 * h + 16 * q, y);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 8; ++i)
              w[8 * q + i] = pack_bf16x2(
                  ffma2(f2pack(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), f2,
                        f2pack(__uint_as_float(y[2 * i]), __uint_as_float(y[2 * i + 1]))));
          }
          if (h == 1) {  // O is in registers
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars[kOFree + (c & 1)]);
          }
          // neighbouring lanes exchange 32-byte pieces: a store instruction then
          // writes 64 bytes of 16 rows, not 32 bytes of 32 (the row-per-lane form
          // took 173 us where whole pieces took 151: 64 heads of 128, N = 8192)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t send = odd ? w[i] : w[8 + i];
            const uint32_t recv = __shfl_xor_sync(0xffffffffu, send, 1);
            if (odd) w[i] = recv;
            else w[8 + i] = recv;
          }
          const int left = columns - 32 * h;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (row0 + i >= len) continue;
            __nv_bfloat16 *at = dst + 32 * h + i * ot;
            if constexpr (decltype(is_wide)::value) {
              if (left >= 16)
                asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(at),
                             "r"(w[8 * i]), "r"(w[8 * i + 1]), "r"(w[8 * i + 2]),
                             "r"(w[8 * i + 3]), "r"(w[8 * i + 4]), "r"(w[8 * i + 5]),
                             "r"(w[8 * i + 6]), "r"(w[8 * i + 7])
                             : "memory");
            } else {
              if (left > 0)
                *(uint4 *)at = make_uint4(w[8 * i], w[8 * i + 1], w[8 * i + 2], w[8 * i + 3]);
              if (left > 8)
                *(uint4 *)(at + 8) =
                    make_uint4(w[8 * i + 4], w[8 * i + 5], w[8 * i + 6], w[8 * i + 7]);
            }
          }
        }
      }
    };
    // 32-byte stores where every piece is whole and 32-byte aligned
    if (((uintptr_t)role.out & 31) == 0 && role.ob % 16 == 0 && role.oh % 16 == 0 &&
        ot % 16 == 0 && role.dvo % 16 == 0)
      walk(std::true_type{});
    else
      walk(std::false_type{});
  }

  // ---------------------------------------------------------------- teardown
  // The issuers have seen their last MMA complete before they get here.
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (threadIdx.x == 0 && *abort_flag) atomicExch(p.err, kErrTimeout);
}

// 4-D map (width, tokens, heads, batch) with a box of 64 or 32 columns x 128
// tokens; outside reads as zero.
bool make_map(CUtensorMap *map, const DecayView &x, int width, int box_cols, const DecayCall &c) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t one = (cuuint64_t)width * 2;  // a dimension of one entry has no stride
  cuuint64_t gdim[4] = {(cuuint64_t)width, (cuuint64_t)c.n, (cuuint64_t)c.heads,
                        (cuuint64_t)c.batch};
  cuuint64_t gstride[3] = {c.n > 1 ? (cuuint64_t)x.st * 2 : one,
                           c.heads > 1 ? (cuuint64_t)x.sh * 2 : one,
                           c.batch > 1 ? (cuuint64_t)x.sb * 2 : one};
  cuuint32_t box[4] = {(cuuint32_t)box_cols, kT, 1, 1};
  cuuint32_t estride[4] = {1, 1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(x.p), gdim, gstride, box,
            estride, CU_TENSOR_MAP_INTERLEAVE_NONE,
            box_cols == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DK, bool kStateOnly, bool kLead, bool kExact>
int launch_t(const TcParams &p, int64_t grid, cudaStream_t s) {
  using L = TcLayout<DK, kStateOnly, kExact>;
  auto kernel = decay_tc_kernel<DK, kStateOnly, kLead, kExact>;
  if (allow_dynamic_smem((const void *)kernel, (int)L::kSmem) != LA_OK) return LA_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(L::kThreads);
  cfg.dynamicSmemBytes = L::kSmem;
  cfg.stream = s;
  // behind a state pass of its own call, whose CTAs let it start early: it waits
  // where it reads the states
  cudaLaunchAttribute pdl;
  pdl.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &pdl;
  cfg.numAttrs = !kStateOnly && !kLead && p.segments > 1 ? 1 : 0;
  cudaLaunchKernelEx(&cfg, kernel, p);
  return check_launch();
}

template <bool kStateOnly, bool kLead, bool kExact>
int launch_width(const TcParams &p, int da, int64_t grid, cudaStream_t s) {
  if (da <= 32) return launch_t<32, kStateOnly, kLead, kExact>(p, grid, s);
  return da <= 64 ? launch_t<64, kStateOnly, kLead, kExact>(p, grid, s)
                  : launch_t<128, kStateOnly, kLead, kExact>(p, grid, s);
}

template <bool kStateOnly>
int launch(const DecayCall &c, cudaStream_t s) {
  TcParams p;
  // first: it binds the device's context to a thread that has none yet (an
  // autograd worker), which encoding a tensor map needs
  p.err = device_error_word();
  if (!p.err) return LA_ERR_CUDA;
  int maps = 0, da = 0, slices = 1;
  struct {
    DecayView x;
    int width, box;
  } known[kMaxMaps];
  auto map_of = [&](const DecayView &x, int width, int box) {
    for (int i = 0; i < maps; ++i) {
      const DecayView &y = known[i].x;
      if (y.p == x.p && y.sb == x.sb && y.sh == x.sh && y.st == x.st &&
          known[i].width == width && known[i].box == box)
        return i;
    }
    if (maps == kMaxMaps || !make_map(&p.map[maps], x, width, box, c)) return -1;
    known[maps].x = x;
    known[maps].width = width;
    known[maps].box = box;
    return maps++;
  };
  for (int r = 0; r < c.roles; ++r)
    if (c.role[r].da > da) da = c.role[r].da;
  const int box = da <= 32 ? 32 : 64;
  for (int r = 0; r < c.roles; ++r) {
    const DecayRole &f = c.role[r];
    TcRole &t = p.role[r];
    t.a = kStateOnly ? 0 : map_of(f.a, f.da, box);
    t.b = map_of(f.b, f.da, box);
    t.v = map_of(f.v, f.dvo, 64);
    if (t.a < 0 || t.b < 0 || t.v < 0) return LA_ERR_CUDA;
    t.out = (__nv_bfloat16 *)f.out.p;
    t.ob = f.out.sb, t.oh = f.out.sh, t.ot = f.out.st;
    t.init = f.init, t.states = f.states, t.final_state = f.final_state;
    t.da = f.da, t.dvo = f.dvo;
    t.transposed = f.transposed, t.reverse = f.reverse;
    t.intra = f.intra, t.inter = f.inter, t.inc = f.inc;
    const int n = (f.dvo + kDecaySlice - 1) / kDecaySlice;
    if (n > slices) slices = n;
  }
  p.log_decay = c.log_decay;
  p.heads = c.heads, p.n = c.n;
  p.whole = c.whole, p.seg_len = c.seg_len, p.lead = c.lead;
  p.roles = c.roles, p.slices = slices, p.segments = c.segments;
  p.orders = kStateOnly ? c.segments - 1 : c.segments;
  const int64_t walks =
      (kStateOnly ? 0 : c.whole) + (c.batch * c.heads - c.whole) * (int64_t)p.orders;
  const int64_t grid = walks * slices * c.roles;
  if (grid > INT32_MAX) return LA_ERR_UNSUPPORTED;
  bool exact = false;  // a state is asked for
  for (int r = 0; r < c.roles; ++r) exact = exact || c.role[r].final_state;
  if constexpr (!kStateOnly) {
    if (c.lead > 0)
      return exact ? launch_width<false, true, true>(p, da, grid, s)
                   : launch_width<false, true, false>(p, da, grid, s);
  }
  return exact ? launch_width<kStateOnly, false, true>(p, da, grid, s)
               : launch_width<kStateOnly, false, false>(p, da, grid, s);
}

}  // namespace

bool decay_tc_view(const DecayView &x, int width, const DecayCall &c) {
  return width % 8 == 0 && ((uintptr_t)x.p & 15) == 0 &&
         (c.n <= 1 || (x.st % 8 == 0 && x.st >= width)) &&
         (c.heads <= 1 || (x.sh % 8 == 0 && x.sh > 0)) &&
         (c.batch <= 1 || (x.sb % 8 == 0 && x.sb > 0));
}

int launch_decay_state_tc(const DecayCall &c, cudaStream_t s) { return launch<true>(c, s); }
int launch_decay_output_tc(const DecayCall &c, cudaStream_t s) { return launch<false>(c, s); }

}  // namespace la
