// Linear attention with a decay for each head on CUDA cores (fp32 math): every
// width up to 128, fp32 inputs, and bf16 inputs that TMA cannot address.
//
// One CTA walks one (head, segment, 64 columns of v) in tiles of 64 tokens, laid
// in shared memory in the order of the walk (a reversed walk is the same code).
// Per tile, with t the token's place in the walk:
//   P   = intra * lambda^(ti - tj) (A B^T), tj <= ti
//   out = inter * lambda^(ti + e0) A S + P V
//   S   = lambda^len S + (inc * lambda^(len - e0 - tj) B)^T V
// (e0 = 1, or 0 for a reversed walk).  All is fp32.  Groups of 64 threads compute
// the products side by side: the scores, A S, the state (64 rows of it a group, in
// registers, with a copy in shared memory for A S) and, one tile behind, P V,
// which starts from A S, both scaled by then; two barriers a tile, the next tile's
// copies in flight.  A thread holds 8 x 8 results: a 128-bit shared load returns
// 512 bytes to a warp, four cycles, so 16 of them feed 256 FMAs a thread at an
// even rate; with 4 x 4 results (8 loads per 64 FMAs) the loads were the bound and
// a tile took 12 us.  Scores above the diagonal, and P V's zero blocks, are left
// out by blocks of 8 and 16.  The FMAs are packed pairs (scalar ones: 260 against
// 237 us).  Measured: 7.1 us per tile of 64 columns, 12.6 of 128 (8 heads of
// 2048 x 64 unsplit 236 us, in 16 segments 35); the FMA pipe and the shared
// memory are each busy half the time, the rest is the two warps per scheduler
// waiting for their own instructions and for the slowest group at the barriers.
// The state pass has the state's product only; the groups share a tile's tokens.
#include "decay.cuh"
#include "tc_common.cuh"

namespace la {
namespace {

using tc::f2pack;
using tc::ffma2;

constexpr int kC = 64;   // tokens per tile
constexpr int kDv = kDecaySlice;
constexpr int kRow = kDv + 4;       // floats per row of 64: 16-byte rows, banks spread
constexpr int kBuf = kC * kRow;     // one 64 x 64 buffer
constexpr int kStateThreads = 256;  // of the state pass

template <int DK>
struct SimtLayout {
  static constexpr int kThreads = 192 + DK;      // scores 64, read-out 64, P V 64, state DK
  static constexpr int kStages = DK == 64 ? 2 : 1;  // tiles of A and B (227 KB hold no more)
  static constexpr int kVs = kStages + 1;
  static constexpr int kRowA = DK + 4;
  static constexpr int kTileA = kC * kRowA;
  static constexpr int kA = 0;
  static constexpr int kB = kA + kStages * kTileA;
  static constexpr int kV = kB + kStages * kTileA;
  static constexpr int kP = kV + kVs * kBuf;
  static constexpr int kO = kP + kBuf;           // 16 float4 of each read-out thread
  static constexpr int kS = kO + kC * kDv;
  static constexpr int kPow = kS + DK * kRow;
  static constexpr int kFloats = kPow + kC + 4;
};

template <int DK>
struct SimtStateLayout {
  static constexpr int kRowA = DK + 4;
  static constexpr int kTileA = kC * kRowA;
  static constexpr int kGroups = kStateThreads / DK;  // share a tile's tokens
  static constexpr int kB = 0;
  static constexpr int kV = kB + 2 * kTileA;
  static constexpr int kPow = kV + 2 * kBuf;
  static constexpr int kFloats = kPow + kC + 4;
  static_assert((kGroups - 1) * DK * 64 <= kPow, "partial states take the tiles' place");
};

__device__ __forceinline__ float4 ld4(const float *p) { return *(const float4 *)p; }
__device__ __forceinline__ void fma4(float *acc, float x, const float4 &y) {
  const uint64_t w = f2pack(x, x);
  uint64_t *to = (uint64_t *)acc;
  to[0] = ffma2(w, f2pack(y.x, y.y), to[0]);
  to[1] = ffma2(w, f2pack(y.z, y.w), to[1]);
}
__device__ __forceinline__ float dot4(const float4 &x, const float4 &y, float acc) {
  return fmaf(x.w, y.w, fmaf(x.z, y.z, fmaf(x.y, y.y, fmaf(x.x, y.x, acc))));
}

// Tokens [0, len) x columns [c0, width) of a tile into dst, in the order of the
// walk, zero outside; fp32 rows of 16 bytes by asynchronous copies.
template <typename T, int kCols, int kThreads>
__device__ __forceinline__ void load_tile(float *dst, const T *src, int64_t st, int len, bool rev,
                                          int c0, int width, bool vec) {
  constexpr int kRowFloats = kCols + 4;
  if (vec) {
    constexpr int kPer = kCols / 4;
    for (int i = threadIdx.x; i < kC * kPer; i += kThreads) {
      const int r = i / kPer, c = (i % kPer) * 4;
      const bool in = r < len && c0 + c < width;
      const T *from = in ? src + (rev ? len - 1 - r : r) * st + c0 + c : src;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(
                       (uint32_t)__cvta_generic_to_shared(dst + r * kRowFloats + c)),
                   "l"(from), "r"(in ? 16 : 0)
                   : "memory");
    }
    return;
  }
  for (int i = threadIdx.x; i < kC * kCols; i += kThreads) {
    const int r = i / kCols, c = i % kCols;
    dst[r * kRowFloats + c] = r < len && c0 + c < width
                                  ? to_f32(src[(rev ? len - 1 - r : r) * st + c0 + c]) : 0.f;
  }
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

template <typename T>
__device__ __forceinline__ bool vec_ok(const DecayView &x, int width) {
  return sizeof(T) == 4 && ((uintptr_t)x.p & 15) == 0 && width % 4 == 0 && x.sb % 4 == 0 &&
         x.sh % 4 == 0 && x.st % 4 == 0;
}

// acc[i] += X[row ty + 8 i][k] * Y[k][tx * 4 ..+4, 32 + tx * 4 ..+4], i >= kFrom
template <int kFrom>
__device__ __forceinline__ void product(float (&acc)[8][8], const float *x, int x_row,
                                        const float *y, int k0, int k1) {
#pragma unroll 1
  for (int k = k0; k < k1; k += 4) {
    float4 a[8];
#pragma unroll
    for (int i = kFrom; i < 8; ++i) a[i] = ld4(x + 8 * i * x_row + k);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      const float4 y0 = ld4(y + (k + kk) * kRow), y1 = ld4(y + (k + kk) * kRow + 32);
#pragma unroll
      for (int i = kFrom; i < 8; ++i) {
        const float w = ((const float *)&a[i])[kk];
        fma4(acc[i], w, y0);
        fma4(acc[i] + 4, w, y1);
      }
    }
  }
}

// A tile's tokens [j0, j1) into the state rows h + ty * 4 ..+4 and 32 further
__device__ __forceinline__ void state_update(float (&st)[8][8], const float *b, int b_row,
                                             const float *v, const float *pw, float inc, int len,
                                             int e0, int j0, int j1) {
  const float keep = pw[len];
#pragma unroll
  for (int r = 0; r < 8; ++r)
#pragma unroll
    for (int x = 0; x < 8; ++x) st[r][x] *= keep;
#pragma unroll 4
  for (int j = j0; j < j1; ++j) {
    const float w = inc * pw[max(len - e0 - j, 0)];  // (tokens behind len are zero)
    const float4 x0 = ld4(b + j * b_row), x1 = ld4(b + j * b_row + 32);
    float4 y0 = ld4(v + j * kRow), y1 = ld4(v + j * kRow + 32);
    y0.x *= w; y0.y *= w; y0.z *= w; y0.w *= w;
    y1.x *= w; y1.y *= w; y1.z *= w; y1.w *= w;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      fma4(st[r], ((const float *)&x0)[r], y0);
      fma4(st[r] + 4, ((const float *)&x0)[r], y1);
      fma4(st[r + 4], ((const float *)&x1)[r], y0);
      fma4(st[r + 4] + 4, ((const float *)&x1)[r], y1);
    }
  }
}

__device__ __forceinline__ void store_state(float *dst, const float (&st)[8][8], int row0, int c0,
                                            int da, int dvo) {
#pragma unroll
  for (int r = 0; r < 8; ++r)
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int row = row0 + (r & 3) + (r >> 2) * 32, col = c0 + (x & 3) + (x >> 2) * 32;
      if (row < da && col < dvo) dst[(int64_t)row * dvo + col] = st[r][x];
    }
}

// The tokens of one CTA's walk.
struct SimtWalk {
  int64_t t0, t1;
  int tiles;
  bool rev;
  __device__ SimtWalk(const DecayCall &call, bool rev, int order) : rev(rev) {
    t0 = (int64_t)(rev ? call.segments - 1 - order : order) * call.seg_len;
    t1 = min64(call.n, t0 + call.seg_len);
    tiles = (int)((t1 - t0 + kC - 1) / kC);
  }
  __device__ int64_t base(int c) const { return t0 + (int64_t)(rev ? tiles - 1 - c : c) * kC; }
  __device__ int len(int c) const { return (int)min64(kC, t1 - base(c)); }
};

template <typename T, int DK>
__global__ void __launch_bounds__(SimtLayout<DK>::kThreads, 1)
decay_simt_kernel(const __grid_constant__ DecayCall call, int slices) {
  using L = SimtLayout<DK>;
  extern __shared__ __align__(16) float sm[];
  const DecayRole &role = call.role[blockIdx.z];
  const int order = blockIdx.x / slices, c0 = blockIdx.x % slices * kDv;
  if (c0 >= role.dvo) return;
  const int64_t bh = blockIdx.y;
  const int64_t ib = bh / call.heads, ih = bh % call.heads;
  const SimtWalk walk(call, role.reverse != 0, order);
  const int e0 = walk.rev ? 0 : 1, tiles = walk.tiles;
  const float g = call.log_decay[ih];
  float *pw = sm + L::kPow;
  if (threadIdx.x <= kC) pw[threadIdx.x] = decay_pow(g, threadIdx.x);

  const T *ap = (const T *)role.a.p + ib * role.a.sb + ih * role.a.sh;
  const T *bp = (const T *)role.b.p + ib * role.b.sb + ih * role.b.sh;
  const T *vp = (const T *)role.v.p + ib * role.v.sb + ih * role.v.sh;
  T *op = (T *)role.out.p + ib * role.out.sb + ih * role.out.sh;
  const bool va = vec_ok<T>(role.a, role.da), vb = vec_ok<T>(role.b, role.da);
  const bool vv = vec_ok<T>(role.v, role.dvo), vo = vec_ok<T>(role.out, role.dvo);
  auto load = [&](int c) {
    const int64_t base = walk.base(c);
    const int len = walk.len(c), stage = c % L::kStages;
    load_tile<T, DK, L::kThreads>(sm + L::kA + stage * L::kTileA, ap + base * role.a.st,
                                  role.a.st, len, walk.rev, 0, role.da, va);
    load_tile<T, DK, L::kThreads>(sm + L::kB + stage * L::kTileA, bp + base * role.b.st,
                                  role.b.st, len, walk.rev, 0, role.da, vb);
    load_tile<T, kDv, L::kThreads>(sm + L::kV + c % L::kVs * kBuf, vp + base * role.v.st,
                                   role.v.st, len, walk.rev, c0, role.dvo, vv);
    copies_commit();
  };
  if (tiles > 0) load(0);

  // the seed: the segments before this one, from the last, and the initial state
  {
    const int per_head = role.da * role.dvo;
    constexpr int kPer = (DK * kDv + L::kThreads - 1) / L::kThreads;
    int at[kPer];  // outside the state: its first value, put to zero below
    float seed[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int i = threadIdx.x + e * L::kThreads;
      const int row = role.transposed ? i % DK : i / kDv;
      const int col = c0 + (role.transposed ? i / DK : i % kDv);
      at[e] = row >= role.da || col >= role.dvo ? 0
              : role.transposed ? col * role.da + row : row * role.dvo + col;
      seed[e] = 0.f;
    }
    auto join = [&](const float *src, float keep) {
#pragma unroll
      for (int e = 0; e < kPer; ++e) seed[e] = fmaf(keep, src[at[e]], seed[e]);
    };
    int after = 0;  // tokens from the end of segment o to this one's start
#pragma unroll 2
    for (int o = order - 1; o >= 0; --o) {
      join(role.states + (bh * call.segments + o) * per_head, decay_pow(g, after));
      after += segment_tokens(o, walk.rev, call.segments, call.seg_len, call.n);
    }
    if (role.init) join(role.init + bh * per_head, decay_pow(g, after));
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int i = threadIdx.x + e * L::kThreads;
      const int row = role.transposed ? i % DK : i / kDv;
      const int col = role.transposed ? i / DK : i % kDv;
      if (i < DK * kDv)
        sm[L::kS + row * kRow + col] = row < role.da && c0 + col < role.dvo ? seed[e] : 0.f;
    }
  }

  const int group = threadIdx.x / 64;  // 0 scores, 1 read-out, 3 P V, else state
  const int tx = threadIdx.x & 7, ty = threadIdx.x / 8 & 7;
  const int kd = (role.da + 3) & ~3;
  const int row0 = (group == 2 ? 0 : 64) + ty * 4;  // of the state, in its groups
  alignas(16) float acc[8][8];
  __syncthreads();
  if (group == 2 || group > 3) {
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const float *s = sm + L::kS + (row0 + (r & 3) + (r >> 2) * 32) * kRow + tx * 4;
      *(float4 *)acc[r] = ld4(s);
      *(float4 *)(acc[r] + 4) = ld4(s + 32);
    }
  }

#pragma unroll 1
  for (int c = 0; c <= tiles; ++c) {
    copies_wait();
    __syncthreads();  // tile c is loaded; P, O of tile c - 1 and S are written
    if (L::kStages > 1 && c + 1 < tiles) load(c + 1);
    const float *a = sm + L::kA + c % L::kStages * L::kTileA;
    const float *b = sm + L::kB + c % L::kStages * L::kTileA;
    if (group == 3) {
      if (c > 0) {
        const float *o = sm + L::kO + (threadIdx.x & 63) * 4;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          *(float4 *)acc[i] = ld4(o + (2 * i) * 256);
          *(float4 *)(acc[i] + 4) = ld4(o + (2 * i + 1) * 256);
        }
        const float *x = sm + L::kP + ty * kRow;
        const float *y = sm + L::kV + (c - 1) % L::kVs * kBuf + tx * 4;
        product<0>(acc, x, kRow, y, 0, 16);  // (rows before k see no token k)
        product<2>(acc, x, kRow, y, 16, 32);
        product<4>(acc, x, kRow, y, 32, 48);
        product<6>(acc, x, kRow, y, 48, 64);
        const int len = walk.len(c - 1), col = c0 + tx * 4;
        const int64_t base = walk.base(c - 1);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = ty + 8 * i;
          if (row >= len) continue;
          T *dst = op + (base + (walk.rev ? len - 1 - row : row)) * role.out.st + col;
          if (vo) {
            if (col < role.dvo) *(float4 *)dst = *(const float4 *)acc[i];
            if (col + 32 < role.dvo) *(float4 *)(dst + 32) = *(const float4 *)(acc[i] + 4);
          } else {
#pragma unroll
            for (int x = 0; x < 8; ++x) {
              const int at = (x & 3) + (x >> 2) * 32;
              if (col + at < role.dvo) dst[at] = from_f32<T>(acc[i][x]);
            }
          }
        }
      }
    } else if (c < tiles) {
      if (group == 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int j = 0; j <= i; ++j) acc[i][j] = 0.f;
#pragma unroll 1
        for (int k = 0; k < kd; k += 4) {
          float4 x[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = ld4(a + (ty + 8 * i) * L::kRowA + k);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 y = ld4(b + (tx + 8 * j) * L::kRowA + k);
#pragma unroll
            for (int i = j; i < 8; ++i) acc[i][j] = dot4(x[i], y, acc[i][j]);
          }
        }
      } else if (group == 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int x = 0; x < 8; ++x) acc[i][x] = 0.f;
        product<0>(acc, a + ty * L::kRowA, L::kRowA, sm + L::kS + tx * 4, 0, kd);
      } else if (row0 < role.da) {
        state_update(acc, b + row0, L::kRowA, sm + L::kV + c % L::kVs * kBuf + tx * 4, pw,
                     role.inc, walk.len(c), e0, 0, kC);
      }
    }
    __syncthreads();  // S, P, O and, with one stage, the tile are read
    if (c == tiles) break;
    if (L::kStages == 1 && c + 1 < tiles) load(c + 1);
    if (group == 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int lag = ty + 8 * i - (tx + 8 * j);
          sm[L::kP + (ty + 8 * i) * kRow + tx + 8 * j] =
              j <= i && lag >= 0 ? role.intra * acc[i][j] * pw[max(lag, 0)] : 0.f;
        }
    } else if (group == 1) {
      float *o = sm + L::kO + (threadIdx.x & 63) * 4;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float w = role.inter * pw[min(ty + 8 * i + e0, kC)];
#pragma unroll
        for (int x = 0; x < 8; ++x) acc[i][x] *= w;
        *(float4 *)(o + (2 * i) * 256) = *(const float4 *)acc[i];
        *(float4 *)(o + (2 * i + 1) * 256) = *(const float4 *)(acc[i] + 4);
      }
    } else if (group != 3) {
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        float *s = sm + L::kS + (row0 + (r & 3) + (r >> 2) * 32) * kRow + tx * 4;
        *(float4 *)s = *(const float4 *)acc[r];
        *(float4 *)(s + 32) = *(const float4 *)(acc[r] + 4);
      }
    }
  }
  if ((group == 2 || group > 3) && role.final_state && order == call.segments - 1)
    store_state(role.final_state + bh * role.da * role.dvo, acc, row0, c0 + tx * 4, role.da, role.dvo);
}

// The state that each segment but the last adds: the groups of DK threads share
// a tile's tokens and hold a state each, summed at the end.
template <typename T, int DK>
__global__ void __launch_bounds__(kStateThreads, 2)
decay_simt_state_kernel(const __grid_constant__ DecayCall call, int slices) {
  using L = SimtStateLayout<DK>;
  extern __shared__ __align__(16) float sm[];
  const DecayRole &role = call.role[blockIdx.z];
  const int order = blockIdx.x / slices, c0 = blockIdx.x % slices * kDv;
  if (c0 >= role.dvo) return;
  const int64_t bh = blockIdx.y;
  const int64_t ib = bh / call.heads, ih = bh % call.heads;
  const SimtWalk walk(call, role.reverse != 0, order);
  const int e0 = walk.rev ? 0 : 1;
  const float g = call.log_decay[ih];
  float *pw = sm + L::kPow;
  if (threadIdx.x <= kC) pw[threadIdx.x] = decay_pow(g, threadIdx.x);
  const T *bp = (const T *)role.b.p + ib * role.b.sb + ih * role.b.sh;
  const T *vp = (const T *)role.v.p + ib * role.v.sb + ih * role.v.sh;
  const bool vb = vec_ok<T>(role.b, role.da), vv = vec_ok<T>(role.v, role.dvo);
  auto load = [&](int c) {
    const int64_t base = walk.base(c);
    const int len = walk.len(c);
    load_tile<T, DK, kStateThreads>(sm + L::kB + c % 2 * L::kTileA, bp + base * role.b.st,
                                    role.b.st, len, walk.rev, 0, role.da, vb);
    load_tile<T, kDv, kStateThreads>(sm + L::kV + c % 2 * kBuf, vp + base * role.v.st, role.v.st,
                                     len, walk.rev, c0, role.dvo, vv);
    copies_commit();
  };
  const int group = threadIdx.x / DK, tx = threadIdx.x & 7, ty = threadIdx.x / 8 & 7;
  const int row0 = threadIdx.x % DK / 64 * 64 + ty * 4;
  constexpr int kShare = kC / L::kGroups;
  alignas(16) float st[8][8] = {};
  load(0);
#pragma unroll 1
  for (int c = 0; c < walk.tiles; ++c) {
    copies_wait();
    __syncthreads();  // tile c is loaded, tile c - 1 read
    if (c + 1 < walk.tiles) load(c + 1);
    state_update(st, sm + L::kB + c % 2 * L::kTileA + row0, L::kRowA,
                 sm + L::kV + c % 2 * kBuf + tx * 4, pw, role.inc, walk.len(c), e0,
                 group * kShare, (group + 1) * kShare);
  }
  __syncthreads();
  if (group > 0) {
    float *at = sm + (group - 1) * DK * 64 + threadIdx.x % DK * 4;
#pragma unroll
    for (int i = 0; i < 16; ++i) *(float4 *)(at + i * DK * 4) = *(const float4 *)(st[i / 2] + i % 2 * 4);
  }
  __syncthreads();
  if (group > 0) return;
#pragma unroll 1
  for (int o = 0; o < L::kGroups - 1; ++o) {
    const float *at = sm + o * DK * 64 + threadIdx.x * 4;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float4 x = ld4(at + i * DK * 4);
      float *to = st[i / 2] + i % 2 * 4;
      to[0] += x.x; to[1] += x.y; to[2] += x.z; to[3] += x.w;
    }
  }
  store_state(role.states + (bh * call.segments + order) * role.da * role.dvo, st, row0,
              c0 + tx * 4, role.da, role.dvo);
}

template <typename T, int DK, bool kStateOnly>
int launch_t(const DecayCall &c, int slices, cudaStream_t s) {
  const dim3 grid((unsigned)(slices * (kStateOnly ? c.segments - 1 : c.segments)),
                  (unsigned)(c.batch * c.heads), c.roles);
  const int bytes = (kStateOnly ? SimtStateLayout<DK>::kFloats : SimtLayout<DK>::kFloats) * 4;
  auto kernel = kStateOnly ? decay_simt_state_kernel<T, DK> : decay_simt_kernel<T, DK>;
  if (allow_dynamic_smem((const void *)kernel, bytes) != LA_OK) return LA_ERR_CUDA;
  kernel<<<grid, kStateOnly ? kStateThreads : SimtLayout<DK>::kThreads, bytes, s>>>(c, slices);
  return check_launch();
}

template <bool kStateOnly>
int launch(const DecayCall &c, cudaStream_t s) {
  int da = 0, slices = 1;
  for (int r = 0; r < c.roles; ++r) {
    if (c.role[r].da > da) da = c.role[r].da;
    const int n = (c.role[r].dvo + kDv - 1) / kDv;
    if (n > slices) slices = n;
  }
  if (da > kDecayMaxWidth || slices > kDecayMaxWidth / kDv) return LA_ERR_UNSUPPORTED;
  if (c.dtype == LA_DTYPE_FLOAT32)
    return da <= 64 ? launch_t<float, 64, kStateOnly>(c, slices, s)
                    : launch_t<float, 128, kStateOnly>(c, slices, s);
  return da <= 64 ? launch_t<__nv_bfloat16, 64, kStateOnly>(c, slices, s)
                  : launch_t<__nv_bfloat16, 128, kStateOnly>(c, slices, s);
}

}  // namespace

int launch_decay_state_simt(const DecayCall &c, cudaStream_t s) { return launch<true>(c, s); }
int launch_decay_output_simt(const DecayCall &c, cudaStream_t s) { return launch<false>(c, s); }

}  // namespace la
