// Epilogue of a linear layer: y = act(z + bias) * mul + residual, FP32,
// rounded once into y.
#pragma once
#include <cuda_bf16.h>

#include "kernels.h"

namespace xksv {

__device__ __forceinline__ float act_apply(uint32_t act, float z) {
  switch (act) {
    case 1: return z > 0.f || z != z ? z : 0.f;  // relu, NaN kept
    case 2: return z / (1.f + expf(-z));         // silu
    case 3: return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
    case 4: return 0.5f * z * (1.f + tanhf(0.79788456080286536f * (z + 0.044715f * z * z * z)));
    default: return z;
  }
}

__device__ __forceinline__ float load_elem(const void* p, uint64_t i, bool f32) {
  return f32 ? static_cast<const float*>(p)[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

__device__ __forceinline__ void epilogue_store(const Epilogue& e, uint64_t b, uint64_t row, float z) {
  if (e.bias) z += load_elem(e.bias, row, e.bias_f32);
  z = act_apply(e.act, z);
  if (e.mul) z *= load_elem(e.mul, b * e.mul_stride + row, e.mul_f32);
  if (e.residual) z += load_elem(e.residual, b * e.residual_stride + row, e.residual_f32);
  if (e.y_f32)
    static_cast<float*>(e.y)[b * e.y_stride + row] = z;
  else
    static_cast<__nv_bfloat16*>(e.y)[b * e.y_stride + row] = __float2bfloat16_rn(z);
}

}  // namespace xksv
