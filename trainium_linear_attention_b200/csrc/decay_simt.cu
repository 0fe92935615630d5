// Linear attention with a decay for each head on CUDA cores (fp32 math): every
// width up to 128, fp32 inputs, and bf16 inputs that TMA cannot address.
//
// One CTA of 256 threads walks one (head, segment, 64 columns of v) in tiles
// of 64 tokens.  Everything is held in fp32: the state in registers (a thread
// owns DK / 16 rows x 4 columns) with a copy in shared memory for the read-out,
// A, B, V, the 64 x 64 scores and the powers lambda^0 .. lambda^64.  Per tile,
// with t the token's place in the walk:
//   P   = intra * lambda^(ti - tj) (A B^T), tj <= ti
//   out = inter * lambda^(ti + e0) A S + P V
//   S   = lambda^len S + (inc * lambda^(len - e0 - tj) B)^T V
// (e0 = 1, or 0 for a reversed walk).  Each product is 4x4 register tiles fed
// by 128-bit shared loads (8 per 64 FMAs), so the FMA pipe is the bound: four
// products of 64 x 64 x 64 a tile at d = d_v = 64, 4.2 us at one SM's rate.
// A tile takes 12 us there (24 us per 128 tokens; 8 warps do not hide the loads
// and barriers), 18 at 128 columns: 8 heads of 2048 x 64 in fp32 take 80 us in
// 16 segments, 379 unsplit.
#include "decay.cuh"

namespace la {
namespace {

constexpr int kC = 64;   // tokens per tile
constexpr int kDv = kDecaySlice;
constexpr int kThreads = 256;

template <int DK>
struct SimtLayout {
  static constexpr int kRowA = DK + 4;  // floats per row of A and B: 16-byte rows, banks spread
  static constexpr int kRowV = kDv + 4;
  static constexpr int kA = 0;
  static constexpr int kB = kA + kC * kRowA;
  static constexpr int kV = kB + kC * kRowA;
  static constexpr int kP = kV + kC * kRowV;
  static constexpr int kS = kP + kC * kRowV;
  static constexpr int kPow = kS + DK * kRowV;
  static constexpr int kFloats = kPow + kC + 4;
};

__device__ __forceinline__ float4 ld4(const float *p) { return *(const float4 *)p; }
__device__ __forceinline__ void fma4(float *acc, float x, const float4 &y) {
  acc[0] = fmaf(x, y.x, acc[0]);
  acc[1] = fmaf(x, y.y, acc[1]);
  acc[2] = fmaf(x, y.z, acc[2]);
  acc[3] = fmaf(x, y.w, acc[3]);
}
__device__ __forceinline__ float dot4(const float4 &x, const float4 &y, float acc) {
  return fmaf(x.w, y.w, fmaf(x.z, y.z, fmaf(x.y, y.y, fmaf(x.x, y.x, acc))));
}

// Rows [0, len) x columns [c0, width) of a tile into dst (cols wide, zero
// outside).
template <typename T>
__device__ __forceinline__ void load_tile(float *dst, int row_floats, int cols, const T *src,
                                          int64_t st, int len, int c0, int width, bool vec) {
  if (vec) {  // 16-byte rows of fp32
    const int per_row = cols / 4;
    for (int i = threadIdx.x; i < kC * per_row; i += kThreads) {
      const int r = i / per_row, c = (i % per_row) * 4;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < len && c0 + c < width) x = *(const float4 *)(src + r * st + c0 + c);
      *(float4 *)(dst + r * row_floats + c) = x;
    }
    return;
  }
  for (int i = threadIdx.x; i < kC * cols; i += kThreads) {
    const int r = i / cols, c = i % cols;
    dst[r * row_floats + c] = r < len && c0 + c < width ? to_f32(src[r * st + c0 + c]) : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ bool vec_ok(const DecayView &x, int width) {
  return sizeof(T) == 4 && ((uintptr_t)x.p & 15) == 0 && width % 4 == 0 && x.sb % 4 == 0 &&
         x.sh % 4 == 0 && x.st % 4 == 0;
}

template <typename T, int DK, bool kStateOnly>
__global__ void __launch_bounds__(kThreads)
decay_simt_kernel(const __grid_constant__ DecayCall call, int slices) {
  using L = SimtLayout<DK>;
  constexpr int kR = DK / 16;  // state rows per thread
  extern __shared__ __align__(16) float sm[];
  const DecayRole &role = call.role[blockIdx.z];
  const int slice = blockIdx.x % slices, order = blockIdx.x / slices;
  const int c0 = slice * kDv;
  if (c0 >= role.dvo) return;
  const int64_t bh = blockIdx.y;
  const int64_t ib = bh / call.heads, ih = bh % call.heads;
  const bool rev = role.reverse != 0;
  const int e0 = rev ? 0 : 1;
  const int64_t t0 = (int64_t)(rev ? call.segments - 1 - order : order) * call.seg_len;
  const int64_t t1 = min64(call.n, t0 + call.seg_len);
  const int tiles = (int)((t1 - t0 + kC - 1) / kC);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const float g = call.log_decay[ih];
  float *pw = sm + L::kPow;
  if (threadIdx.x <= kC) pw[threadIdx.x] = decay_pow(g, threadIdx.x);

  const T *ap = kStateOnly ? nullptr : (const T *)role.a.p + ib * role.a.sb + ih * role.a.sh;
  const T *bp = (const T *)role.b.p + ib * role.b.sb + ih * role.b.sh;
  const T *vp = (const T *)role.v.p + ib * role.v.sb + ih * role.v.sh;
  T *op = kStateOnly ? nullptr : (T *)role.out.p + ib * role.out.sb + ih * role.out.sh;
  const bool va = !kStateOnly && vec_ok<T>(role.a, role.da);
  const bool vb = vec_ok<T>(role.b, role.da), vv = vec_ok<T>(role.v, role.dvo);
  const bool vo = !kStateOnly && vec_ok<T>(role.out, role.dvo);

  // state rows ty * kR + r, columns c0 + tx * 4 + x
  float st[kR][4] = {};
  const int64_t per_head = (int64_t)role.da * role.dvo;
  const int64_t state_at = (bh * call.segments + order) * per_head;
  if (!kStateOnly) {
    auto add = [&](const float *src, float keep) {
#pragma unroll
      for (int r = 0; r < kR; ++r)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int row = ty * kR + r, col = c0 + tx * 4 + x;
          if (row < role.da && col < role.dvo)
            st[r][x] = fmaf(keep, st[r][x],
                            src[role.transposed ? (int64_t)col * role.da + row
                                                : (int64_t)row * role.dvo + col]);
        }
    };
    if (role.init) add(role.init + bh * per_head, 0.f);
    for (int o = 0; o < order; ++o)
      add(role.states + (bh * call.segments + o) * per_head,
          decay_pow(g, segment_tokens(o, rev, call.segments, call.seg_len, call.n)));
  }

  for (int c = 0; c < tiles; ++c) {
    const int64_t base = t0 + (int64_t)(rev ? tiles - 1 - c : c) * kC;
    const int len = (int)min64(kC, t1 - base);
    __syncthreads();  // the tile before is read
    if (!kStateOnly) load_tile(sm + L::kA, L::kRowA, DK, ap + base * role.a.st, role.a.st, len, 0,
                               role.da, va);
    load_tile(sm + L::kB, L::kRowA, DK, bp + base * role.b.st, role.b.st, len, 0, role.da, vb);
    load_tile(sm + L::kV, L::kRowV, kDv, vp + base * role.v.st, role.v.st, len, c0, role.dvo, vv);
    if (!kStateOnly) {
#pragma unroll
      for (int r = 0; r < kR; ++r)
        *(float4 *)(sm + L::kS + (ty * kR + r) * L::kRowV + tx * 4) =
            make_float4(st[r][0], st[r][1], st[r][2], st[r][3]);
    }
    __syncthreads();
    if (!kStateOnly) {
      // scores of rows ty * 4 + i, columns tx + 16 * j
      float p[4][4] = {};
#pragma unroll 4
      for (int k = 0; k < DK; k += 4) {
        float4 x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = ld4(sm + L::kA + (ty * 4 + i) * L::kRowA + k);
          y[i] = ld4(sm + L::kB + (tx + 16 * i) * L::kRowA + k);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) p[i][j] = dot4(x[i], y[j], p[i][j]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int lag = rev ? tx + 16 * j - (ty * 4 + i) : ty * 4 + i - (tx + 16 * j);
          sm[L::kP + (ty * 4 + i) * L::kRowV + tx + 16 * j] =
              lag >= 0 && tx + 16 * j < len ? role.intra * p[i][j] * pw[lag] : 0.f;
        }
      __syncthreads();
      float o[4][4] = {};
#pragma unroll 2
      for (int k = 0; k < DK; k += 4) {
        float4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = ld4(sm + L::kA + (ty * 4 + i) * L::kRowA + k);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          const float4 y = ld4(sm + L::kS + (k + kk) * L::kRowV + tx * 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) fma4(o[i], ((const float *)&x[i])[kk], y);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = ty * 4 + i;
        const float w = row < len ? role.inter * pw[(rev ? len - 1 - row : row) + e0] : 0.f;
#pragma unroll
        for (int x = 0; x < 4; ++x) o[i][x] *= w;
      }
#pragma unroll 2
      for (int k = 0; k < kC; k += 4) {
        float4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = ld4(sm + L::kP + (ty * 4 + i) * L::kRowV + k);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          const float4 y = ld4(sm + L::kV + (k + kk) * L::kRowV + tx * 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) fma4(o[i], ((const float *)&x[i])[kk], y);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = ty * 4 + i, col = c0 + tx * 4;
        if (row >= len) continue;
        T *dst = op + (base + row) * role.out.st + col;
        if (vo && col < role.dvo) {
          *(float4 *)dst = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
        } else {
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (col + x < role.dvo) dst[x] = from_f32<T>(o[i][x]);
        }
      }
    }
    // the state after this tile
    const float keep = pw[len];
#pragma unroll
    for (int r = 0; r < kR; ++r)
#pragma unroll
      for (int x = 0; x < 4; ++x) st[r][x] *= keep;
    for (int j = 0; j < len; ++j) {
      const float w = role.inc * pw[len - e0 - (rev ? len - 1 - j : j)];
      float4 y = ld4(sm + L::kV + j * L::kRowV + tx * 4);
      y.x *= w; y.y *= w; y.z *= w; y.w *= w;
#pragma unroll
      for (int r = 0; r < kR; r += 4) {
        const float4 x = ld4(sm + L::kB + j * L::kRowA + ty * kR + r);
        fma4(st[r], x.x, y);
        fma4(st[r + 1], x.y, y);
        fma4(st[r + 2], x.z, y);
        fma4(st[r + 3], x.w, y);
      }
    }
  }
  float *dst = nullptr;
  if (kStateOnly) dst = role.states + state_at;
  else if (role.final_state && order == call.segments - 1) dst = role.final_state + bh * per_head;
  if (dst) {
#pragma unroll
    for (int r = 0; r < kR; ++r)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int row = ty * kR + r, col = c0 + tx * 4 + x;
        if (row < role.da && col < role.dvo) dst[(int64_t)row * role.dvo + col] = st[r][x];
      }
  }
}

template <typename T, int DK, bool kStateOnly>
int launch_t(const DecayCall &c, int slices, cudaStream_t s) {
  auto kernel = decay_simt_kernel<T, DK, kStateOnly>;
  const int bytes = SimtLayout<DK>::kFloats * 4;
  if (allow_dynamic_smem((const void *)kernel, bytes) != LA_OK) return LA_ERR_CUDA;
  const dim3 grid((unsigned)(slices * (kStateOnly ? c.segments - 1 : c.segments)), (unsigned)(c.batch * c.heads), c.roles);
  kernel<<<grid, kThreads, bytes, s>>>(c, slices);
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
