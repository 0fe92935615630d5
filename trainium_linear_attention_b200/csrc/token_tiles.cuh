// Tiles of (batch, tokens, channels) tensors, as warps fetch them.
#pragma once

#include "common.cuh"
#include "pairs.cuh"
#include "tc_common.cuh"
#include "tma_host.cuh"

namespace la {

// A (batch, tokens, channels) tensor with a dense last dimension; strides in
// elements.
struct TokenView {
  const void *p = nullptr;
  int64_t sb = 0, st = 0;
};
struct TokenSizes {
  int64_t batch = 0, tokens = 0;
  int channels = 0;
};

__device__ __forceinline__ int64_t sequence_length(const void *lengths, int is64, int64_t b,
                                                   int64_t tokens) {
  if (!lengths) return tokens;
  const int64_t n = is64 ? ((const int64_t *)lengths)[b] : ((const int32_t *)lengths)[b];
  return n < 0 ? 0 : n < tokens ? n : tokens;
}

// A warp's tile: a lane has two channels and kL neighbouring tokens.  A CTA takes
// `ch` = 64, 32 or 16 channels; the ch / 2 lanes of a "part" share its tokens, the
// 64 / ch parts of a warp have neighbouring groups of kL.  In shared memory token k
// of part p lies at (k * parts + p) * ch: lane l finds its two channels at 64 k +
// 2 l whatever ch is, in other banks than its warp's other lanes.  A warp fetches
// its own tiles and reads no other's.
//
// kTma: rows that start at 16 bytes.  kAsync: at 4 or 8 bytes.  kShifted (bf16): at
// any element; the 16-byte pieces of memory that a row lies in are copied, and its
// elements moved to the row's start when they have arrived.
enum class Fetch { kTma, kAsync, kShifted };

constexpr int kTileMaps = 4;
struct TileMaps {  // (channels, groups of kL tokens, tokens of a group, batch)
  CUtensorMap m[kTileMaps];
};

// Elements of a tile of one tensor.
template <Fetch kF>
__host__ __device__ constexpr int tile_elems(int l, int ch) {
  return 64 * l + (kF == Fetch::kShifted ? 8 * (64 / ch) * l : 0);
}

template <int kN>
__device__ __forceinline__ void copy_async(uint32_t dst, const void *src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(kN),
               "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kN>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kN) : "memory");
}

// Tokens [t0, t0 + 64 / ch * kL) of `row0` (the tensor at this sequence's first
// token and this CTA's first channel); tokens outside [0, len) and channels beyond
// `width` are set to zero and not read.  kN bytes a copy.
template <typename T, int kL, int kN>
__device__ __forceinline__ void copy_tile(T *tile, const T *row0, int64_t st, int t0, int len, int ch,
                                          int width) {
  constexpr int kPer = kN / (int)sizeof(T);  // elements of a copy
  const int lane = threadIdx.x & 31;
  if constexpr (kPer >= 2) {  // a lane's copies are whole rows of 64 apart
    const int at = lane * kPer, q = at % ch;
    int k = at / 64, t = t0 + at % 64 / ch * kL + k;
    const T *src = row0 + (int64_t)t * st + q;
    uint32_t dst = (uint32_t)__cvta_generic_to_shared(tile + at);
    const int bytes = max(0, min(kN, (width - q) * (int)sizeof(T)));
    const int64_t step = st * (kPer / 2);
#pragma unroll
    for (int n = 0; n < kL * 2 / kPer; ++n) {
      const bool in = bytes > 0 && (unsigned)t < (unsigned)len;
      copy_async<kN>(dst, in ? src : row0, in ? bytes : 0);
      src += step, dst += 32 * kN, t += kPer / 2;
    }
  } else {
#pragma unroll 4
    for (int n = lane; n < 64 * kL; n += 32) {
      const int t = t0 + n % 64 / ch * kL + n / 64, q = n % ch;
      const bool in = q < width && (unsigned)t < (unsigned)len;
      copy_async<kN>((uint32_t)__cvta_generic_to_shared(tile + n),
                     in ? row0 + (int64_t)t * st + q : row0, in ? kN : 0);
    }
  }
}

// The same by the 16-byte pieces that the rows lie in, `ch` + 8 elements for each.
// [begin, end): the tensor's memory; pieces that reach beyond it go by elements.
template <int kL>
__device__ __forceinline__ void copy_shifted(__nv_bfloat16 *tile, const __nv_bfloat16 *row0,
                                             int64_t st, int t0, int ch, uintptr_t begin,
                                             uintptr_t end) {
  const int pieces = ch / 8 + 1, parts = 64 / ch;
#pragma unroll 2
  for (int n = threadIdx.x & 31; n < parts * kL * pieces; n += 32) {
    const int r = n / pieces, q = n % pieces;
    const uintptr_t row = (uintptr_t)(row0 + (int64_t)(t0 + r % parts * kL + r / parts) * st);
    const uintptr_t src = (row & ~(uintptr_t)15) + 16 * q;
    __nv_bfloat16 *dst = tile + r * (ch + 8) + 8 * q;
    if (src >= begin && src + 16 <= end) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                       (uint32_t)__cvta_generic_to_shared(dst)),
                   "l"(src)
                   : "memory");
    } else {
      for (int e = 0; e < 8; ++e)
        if (src + 2 * e >= begin && src + 2 * e + 2 <= end) dst[e] = ((const __nv_bfloat16 *)src)[e];
    }
  }
}
// Moves the rows that copy_shifted has brought to where copy_tile puts them.  Rows
// go down in memory, four at a time: none is written before it is read.
template <int kL>
__device__ __forceinline__ void align_shifted(__nv_bfloat16 *tile, const __nv_bfloat16 *row0,
                                              int64_t st, int t0, int ch) {
  const int lane = threadIdx.x & 31, half = ch / 2, part = lane / half, parts = 64 / ch;
  const int column = 2 * (lane & (half - 1));
  const uint32_t shift0 = (uint32_t)((uintptr_t)row0 >> 1) + (uint32_t)(t0 + part * kL) * (uint32_t)st;
  const uint16_t *from = (const uint16_t *)tile + part * (ch + 8) + column;
  uint32_t *to = (uint32_t *)tile + lane;
#pragma unroll 1
  for (int k0 = 0; k0 < kL; k0 += 4) {
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t *p = from + (k0 + i) * parts * (ch + 8) + ((shift0 + (k0 + i) * (uint32_t)st) & 7);
      v[i] = p[0] | (uint32_t)p[1] << 16;
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) to[32 * (k0 + i)] = v[i];
    __syncwarp();
  }
}

// The same out of the way of a loop that copies whole tiles by other means.
template <typename T, int kL>
__device__ __noinline__ void copy_edge(T *tile, const T *row0, int64_t st, int t0, int len, int ch,
                                       int width, int copy) {
  if (copy == 8) copy_tile<T, kL, 8>(tile, row0, st, t0, len, ch, width);
  else copy_tile<T, kL, 4>(tile, row0, st, t0, len, ch, width);
}

// A pair of channels at p, the second of which may be beyond the row; `wide`: pairs
// start at their own size.
template <typename T>
__device__ __forceinline__ float2 pair_at(const T *p, bool wide, bool second) {
  if (wide && second) return load_two(p);
  return make_float2(to_f32(p[0]), second ? to_f32(p[1]) : 0.f);
}
// The same by elements.
template <int kL>
__device__ __noinline__ void load_elements(__nv_bfloat16 *tile, const __nv_bfloat16 *row0, int64_t st,
                                           int t0, int len, int ch, int width) {
  const int lane = threadIdx.x & 31, half = ch / 2, q = 2 * (lane & (half - 1));
  const int first = t0 + lane / half * kL;
  float2 v[kL];
#pragma unroll
  for (int k = 0; k < kL; ++k) {
    v[k] = two(0.f);
    if ((unsigned)(first + k) < (unsigned)len && q < width)
      v[k] = pair_at(row0 + (int64_t)(first + k) * st + q, false, q + 1 < width);
  }
#pragma unroll
  for (int k = 0; k < kL; ++k) store_two(tile + 64 * k + 2 * lane, v[k], true, true);
}
// The tokens of a tile outside [0, len) become `value`.
template <typename T, int kL>
__device__ __noinline__ void fill_outside(T *tile, int t0, int len, int ch, float value) {
  const int lane = threadIdx.x & 31, first = t0 + lane / (ch / 2) * kL;
  for (int k = 0; k < kL; ++k)
    if ((unsigned)(first + k) >= (unsigned)len) store_two(tile + 64 * k + 2 * lane, two(value), true, true);
}

__device__ __forceinline__ void tma_load_4d(void *dst, const CUtensorMap *map, uint64_t *bar, int x,
                                            int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(tc::smem_u32(dst)),
      "l"(map), "r"(tc::smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// What a launch hands a kernel that reads tiles, besides its call.
struct TileLaunch {
  int ch;       // channels of a CTA
  int copy;     // kAsync: bytes of a copy, 4 or 8
  int *err;     // the library's device error word
};

// A warp's ring of kStages tiles of kIn tensors.
template <typename T, int kL, int kIn, int kStages, Fetch kF>
struct WarpTiles {
  T *tiles;                 // the first stage's; stage_elems further on the next one's
  int stage_elems, elems;   // elems: of one tensor's tile
  uint64_t *full;           // kTma: one per stage, `full_step` apart
  int full_step;
  const TokenView *const *views;
  const CUtensorMap *maps;
  int64_t ib;
  int c0, ch, width, copy;
  TokenSizes sizes;
  uint32_t phases;          // kTma: a bit per stage

  __device__ __forceinline__ T *tile(int stage, int n) const {
    return tiles + stage * stage_elems + n * elems;
  }
  __device__ __forceinline__ const T *row0(int n) const {
    return (const T *)views[n]->p + ib * views[n]->sb + c0;
  }
  __device__ __forceinline__ bool whole(int t0, int len) const {
    return t0 >= 0 && t0 + 64 / ch * kL <= len;
  }
  // Starts to fetch the tiles from token t0 on; a sequence of `len` tokens may end in
  // them, or not reach them.
  __device__ __forceinline__ void fetch(int t0, int len, int stage) const {
    if (kF == Fetch::kTma && whole(t0, len)) {
      if ((threadIdx.x & 31) == 0) {
        uint64_t *bar = full + stage * full_step;
        tc::mbar_arrive_expect_tx(bar, kIn * 64 * kL * sizeof(T));
#pragma unroll
        for (int n = 0; n < kIn; ++n)
          tma_load_4d(tile(stage, n), maps + n, bar, c0, t0 / kL, 0, (int)ib);
      }
    } else if (kF == Fetch::kShifted && whole(t0, len)) {
#pragma unroll
      for (int n = 0; n < kIn; ++n) {
        const int64_t st = views[n]->st;
        const uintptr_t begin = (uintptr_t)views[n]->p;
        const uintptr_t end =
            begin + 2 * ((sizes.batch - 1) * views[n]->sb + (sizes.tokens - 1) * st + sizes.channels);
        if constexpr (kF == Fetch::kShifted)
          copy_shifted<kL>(tile(stage, n), row0(n), st, t0, ch, begin, end);
      }
    } else if (kF != Fetch::kShifted && t0 < len && t0 + 64 / ch * kL > 0) {
#pragma unroll
      for (int n = 0; n < kIn; ++n) {
        if constexpr (kF == Fetch::kTma)
          copy_edge<T, kL>(tile(stage, n), row0(n), views[n]->st, t0, len, ch, width, copy);
        else if (copy == 8)
          copy_tile<T, kL, 8>(tile(stage, n), row0(n), views[n]->st, t0, len, ch, width);
        else
          copy_tile<T, kL, 4>(tile(stage, n), row0(n), views[n]->st, t0, len, ch, width);
      }
    }
    if (kF != Fetch::kTma) copy_commit();
  }
  // Waits for what was fetched from t0 on.  Tokens that the sequence does not have are
  // zero, and those of tensor 1 `outside`.
  __device__ __forceinline__ void wait(int t0, int len, int stage, float outside,
                                       volatile int *abort) {
    if (whole(t0, len)) {
      if constexpr (kF == Fetch::kTma) {
        tc::mbar_wait(full + stage * full_step, phases >> stage & 1, abort);
        phases ^= 1u << stage;
        return;
      }
      copy_wait<kStages - 1>();
      __syncwarp();
      if constexpr (kF == Fetch::kShifted) {
#pragma unroll
        for (int n = 0; n < kIn; ++n)
          align_shifted<kL>(tile(stage, n), row0(n), views[n]->st, t0, ch);
      }
      return;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
    const bool none = t0 >= len || t0 + 64 / ch * kL <= 0;
#pragma unroll
    for (int n = 0; n < kIn; ++n) {
      if constexpr (kF == Fetch::kShifted) load_elements<kL>(tile(stage, n), row0(n), views[n]->st, t0, len, ch, width);
      if ((none && kF != Fetch::kShifted) || (n == 1 && outside != 0.f))
        fill_outside<T, kL>(tile(stage, n), t0, len, ch, n == 1 ? outside : 0.f);
    }
    // (ahead of the next copy into these tiles)
    if (kF == Fetch::kTma) tc::fence_proxy_async_smem();
    __syncwarp();
  }
};

// ---- host side ----------------------------------------------------------------------
// The bytes (16 at most) that every row of a tensor starts at.
inline int row_bytes(const TokenView &v, int size) {
  const uint64_t bits = (uint64_t)(uintptr_t)v.p | (uint64_t)(v.sb * size) | (uint64_t)(v.st * size);
  return bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : 2;
}
// Whether TMA can address it: rows at 16 bytes, no broadcast dimension, a whole group.
inline bool tma_view(const TokenView &v, const TokenSizes &s, int size, int l) {
  return row_bytes(v, size) == 16 && v.st >= s.channels && (v.sb > 0 || s.batch == 1) &&
         v.st < ((int64_t)1 << 32) && v.sb < ((int64_t)1 << 37) && s.batch <= INT32_MAX &&
         s.tokens >= l;
}
// (channels, groups of l tokens, tokens of a group, batch), with boxes that fill a
// warp's tile; for the sequences' whole groups only.
inline bool tile_map(CUtensorMap *map, const TokenView &v, const TokenSizes &s, int dtype, int ch,
                     int l) {
  const EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const uint64_t size = dtype == LA_DTYPE_FLOAT32 ? 4 : 2;
  const cuuint64_t st = (cuuint64_t)v.st * size;
  const cuuint64_t dim[4] = {(cuuint64_t)s.channels, (cuuint64_t)(s.tokens / l), (cuuint64_t)l,
                             (cuuint64_t)s.batch};
  const cuuint64_t stride[3] = {st * l, st, s.batch == 1 ? st * l : (cuuint64_t)v.sb * size};
  const cuuint32_t box[4] = {(cuuint32_t)ch, (cuuint32_t)(64 / ch), (cuuint32_t)l, 1};
  const cuuint32_t one[4] = {1, 1, 1, 1};
  return fn(map, dtype == LA_DTYPE_FLOAT32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                           : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
            4, const_cast<void *>(v.p), dim, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// The fetch for all of `views` (null pointers: absent tensors).
inline Fetch fetch_of(const TokenView *const *views, int n, const TokenSizes &s, int size, int l,
                      TileLaunch *launch) {
  bool tma = encode_fn() != nullptr && s.tokens >= l;
  int least = 16;
  for (int i = 0; i < n; ++i) {
    if (!views[i]->p) continue;
    tma = tma && tma_view(*views[i], s, size, l);
    const int bytes = row_bytes(*views[i], size);
    least = bytes < least ? bytes : least;
  }
  launch->copy = least >= 8 ? 8 : 4;
  return tma ? Fetch::kTma : least < 4 ? Fetch::kShifted : Fetch::kAsync;
}

}  // namespace la
