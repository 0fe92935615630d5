// Tiles of (batch, tokens, channels) tensors, as warps fetch them.
#pragma once

#include "common.cuh"
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
// token and this CTA's first channel), all of which the sequence has; channels beyond
// `width` are set to zero and not read.
template <typename T, int kL, int kN>
__device__ __forceinline__ void copy_tile(T *tile, const T *row0, int64_t st, int t0, int ch,
                                          int width) {
  constexpr int kPer = kN / (int)sizeof(T);  // elements of a copy
#pragma unroll 4
  for (int n = threadIdx.x & 31; n < 64 * kL / kPer; n += 32) {
    const int at = n * kPer, k = at / 64, part = at % 64 / ch, q = at % ch;
    const T *src = row0 + (int64_t)(t0 + part * kL + k) * st + q;
    const int bytes = max(0, min(kN, (width - q) * (int)sizeof(T)));
    copy_async<kN>((uint32_t)__cvta_generic_to_shared(tile + at), bytes ? src : row0, bytes);
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

// A tile that the sequence ends in, or that lies beside it: tokens outside [0, len)
// become `outside` and are not read.
template <typename T, int kL>
__device__ __forceinline__ void ragged_tile(T *tile, const T *row0, int64_t st, int t0, int len,
                                            int ch, int width, float outside) {
  const T none = from_f32<T>(outside);
#pragma unroll 8
  for (int at = threadIdx.x & 31; at < 64 * kL; at += 32) {
    const int t = t0 + at % 64 / ch * kL + at / 64, q = at % ch;
    T v = none;
    if (t >= 0 && t < len && q < width) v = row0[(int64_t)t * st + q];
    tile[at] = v;
  }
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
  // Starts to fetch the tiles from token t0 on, all of whose tokens the sequence has.
  __device__ __forceinline__ void fetch(int t0, int stage) const {
    if constexpr (kF == Fetch::kTma) {
      if ((threadIdx.x & 31) == 0) {
        uint64_t *bar = full + stage * full_step;
        tc::mbar_arrive_expect_tx(bar, kIn * 64 * kL * sizeof(T));
#pragma unroll
        for (int n = 0; n < kIn; ++n)
          tma_load_4d(tile(stage, n), maps + n, bar, c0, t0 / kL, 0, (int)ib);
      }
    } else {
#pragma unroll
      for (int n = 0; n < kIn; ++n) {
        const int64_t st = views[n]->st;
        if constexpr (kF == Fetch::kShifted) {
          const uintptr_t begin = (uintptr_t)views[n]->p;
          const uintptr_t end = begin + 2 * ((sizes.batch - 1) * views[n]->sb +
                                             (sizes.tokens - 1) * st + sizes.channels);
          copy_shifted<kL>(tile(stage, n), row0(n), st, t0, ch, begin, end);
        } else if (copy == 8) {
          copy_tile<T, kL, 8>(tile(stage, n), row0(n), st, t0, ch, width);
        } else {
          copy_tile<T, kL, 4>(tile(stage, n), row0(n), st, t0, ch, width);
        }
      }
    }
  }
  // Closes a step's fetches (also where there were none).
  __device__ __forceinline__ void commit() const {
    if constexpr (kF != Fetch::kTma) copy_commit();
  }
  // Waits for what was fetched from t0 on.
  __device__ __forceinline__ void wait(int t0, int stage, volatile int *abort) {
    if constexpr (kF == Fetch::kTma) {
      tc::mbar_wait(full + stage * full_step, phases >> stage & 1, abort);
      phases ^= 1u << stage;
    } else {
      copy_wait<kStages - 1>();
      __syncwarp();
      if constexpr (kF == Fetch::kShifted) {
#pragma unroll
        for (int n = 0; n < kIn; ++n)
          align_shifted<kL>(tile(stage, n), row0(n), views[n]->st, t0, ch);
      }
    }
  }
  // Instead of both, for tiles that the sequence does not fill.  A __syncwarp()
  // follows.
  __device__ __forceinline__ void load_ragged(int t0, int len, int stage, int n, float outside) const {
    ragged_tile<T, kL>(tile(stage, n), row0(n), views[n]->st, t0, len, ch, width, outside);
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
// The fetch for all of `views` (null pointers: absent tensors), and the bytes of a
// copy should it be kAsync.
inline Fetch fetch_of(const TokenView *const *views, int n, const TokenSizes &s, int size, int l,
                      int *copy) {
  bool tma = encode_fn() != nullptr && s.tokens >= l;
  *copy = 16;
  for (int i = 0; i < n; ++i) {
    if (!views[i]->p) continue;
    tma = tma && tma_view(*views[i], s, size, l);
    const int bytes = row_bytes(*views[i], size);
    *copy = bytes < *copy ? bytes : *copy;
  }
  const Fetch f = tma ? Fetch::kTma : *copy < 4 ? Fetch::kShifted : Fetch::kAsync;
  *copy = *copy >= 8 ? 8 : 4;
  return f;
}

}  // namespace la
