// Linear layer on compressed weights (include/xksv_cuda.h, part 7): the
// activations' layout changes and the epilogue around a plan's product.
#include <cuda_bf16.h>

#include <algorithm>

#include "kernels.h"
#include "linear_epilogue.cuh"

namespace xksv {
namespace {

constexpr int TS = 32;  // transpose tile

// x [batch, cols] BF16 (rows `stride` apart) -> FP32 [cols, batch].
__global__ void __launch_bounds__(TS * 8) linear_x_kernel(const __nv_bfloat16* __restrict__ x, uint64_t stride,
                                                          uint64_t batch, uint64_t cols, float* __restrict__ xt) {
  __shared__ float tile[TS][TS + 1];
  const uint64_t nb = (batch + TS - 1) / TS, nc = (cols + TS - 1) / TS;
  const uint32_t tx = threadIdx.x % TS, ty = threadIdx.x / TS;
  for (uint64_t k = blockIdx.x; k < nb * nc; k += gridDim.x) {
    const uint64_t b0 = k / nc * TS, c0 = k % nc * TS;
    for (uint32_t i = ty; i < TS; i += 8)
      if (b0 + i < batch && c0 + tx < cols) tile[i][tx] = __bfloat162float(x[(b0 + i) * stride + c0 + tx]);
    __syncthreads();
    for (uint32_t i = ty; i < TS; i += 8)
      if (c0 + i < cols && b0 + tx < batch) xt[(c0 + i) * batch + b0 + tx] = tile[tx][i];
    __syncthreads();
  }
}

// z FP32 [rows of Y, batch] -> y [batch, rows of Y] with the epilogue, over
// the plan's runs of covered rows.
__global__ void __launch_bounds__(TS * 8) linear_y_kernel(const float* __restrict__ z, uint64_t batch,
                                                          const RowRun* __restrict__ runs, uint32_t nruns,
                                                          const Epilogue e) {
  __shared__ float tile[TS][TS + 1];
  const uint64_t nb = (batch + TS - 1) / TS;
  const uint32_t tx = threadIdx.x % TS, ty = threadIdx.x / TS;
  for (uint32_t ri = blockIdx.y; ri < nruns; ri += gridDim.y) {
    const RowRun run = runs[ri];
    const uint64_t nr = (run.rows + TS - 1) / TS;
    for (uint64_t k = blockIdx.x; k < nb * nr; k += gridDim.x) {
      const uint64_t b0 = k % nb * TS, r0 = k / nb * TS;
      for (uint32_t i = ty; i < TS; i += 8)
        if (r0 + i < run.rows && b0 + tx < batch) tile[i][tx] = z[(run.row0 + r0 + i) * batch + b0 + tx];
      __syncthreads();
      for (uint32_t i = ty; i < TS; i += 8)
        if (b0 + i < batch && r0 + tx < run.rows) epilogue_store(e, b0 + i, run.row0 + r0 + tx, tile[tx][i]);
      __syncthreads();
    }
  }
}

}  // namespace

cudaError_t launch_linear_x(const void* x, uint64_t stride, uint64_t batch, uint64_t cols, float* xt, cudaStream_t st) {
  const uint64_t tiles = ((batch + TS - 1) / TS) * ((cols + TS - 1) / TS);
  if (!tiles) return cudaSuccess;
  linear_x_kernel<<<uint32_t(std::min<uint64_t>(tiles, 4096)), TS * 8, 0, st>>>(
      static_cast<const __nv_bfloat16*>(x), stride, batch, cols, xt);
  return cudaGetLastError();
}

cudaError_t launch_linear_y(const float* z, uint64_t batch, const RowRun* runs, uint32_t nruns, uint64_t rows,
                            const Epilogue& e, cudaStream_t st) {
  if (!nruns) return cudaSuccess;
  const uint64_t tiles = ((batch + TS - 1) / TS) * ((rows + TS - 1) / TS);
  const dim3 g(uint32_t(std::min<uint64_t>(tiles, 4096)), std::min<uint32_t>(nruns, 1024));
  linear_y_kernel<<<g, TS * 8, 0, st>>>(z, batch, runs, nruns, e);
  return cudaGetLastError();
}

}  // namespace xksv
