#include "column_sum.cuh"

namespace la {
namespace {

// 32 columns x 32 row lanes per CTA.
template <typename T>
__global__ void __launch_bounds__(1024)
column_sum_kernel(const float *partial, int64_t rows, int64_t columns, T *out0, int64_t columns0,
                  T *out1) {
  __shared__ float part[32][33];
  const int x = threadIdx.x & 31, lane = threadIdx.x >> 5;
  int64_t c = (int64_t)blockIdx.x * 32 + x;
  tc::grid_dependency_wait();  // launched behind the kernel that writes the rows
  float sum = 0.f;
  if (c < columns) {
#pragma unroll 8
    for (int64_t r = lane; r < rows; r += 32) sum += partial[r * columns + c];
  }
  part[lane][x] = sum;
  __syncthreads();
  // warp w adds column w over the row lanes
  sum = part[x][lane];
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
  c = (int64_t)blockIdx.x * 32 + lane;
  if (x == 0 && c < columns) {
    if (c < columns0) { if (out0) out0[c] = from_f32<T>(sum); }
    else if (out1) { out1[c - columns0] = from_f32<T>(sum); }
  }
}

}  // namespace

int launch_column_sum(const float *partial, int64_t rows, int64_t columns, void *out0,
                      int64_t columns0, void *out1, int dtype, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((columns + 31) / 32));
  cfg.blockDim = dim3(1024);
  cfg.stream = s;
  cudaLaunchAttribute pdl;
  pdl.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &pdl;
  cfg.numAttrs = 1;
  if (dtype == LA_DTYPE_FLOAT32)
    cudaLaunchKernelEx(&cfg, column_sum_kernel<float>, partial, rows, columns, (float *)out0,
                       columns0, (float *)out1);
  else
    cudaLaunchKernelEx(&cfg, column_sum_kernel<__nv_bfloat16>, partial, rows, columns,
                       (__nv_bfloat16 *)out0, columns0, (__nv_bfloat16 *)out1);
  return check_launch();
}

}  // namespace la
