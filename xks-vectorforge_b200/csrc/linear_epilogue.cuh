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

// The epilogue's operands at token b and a row, apart from its arithmetic: a
// caller with several elements reads all of them first (y may be mul or
// residual, so that no read moves past a write by itself).
struct EpilogueOps {
  float bias, mul, residual;
};
__device__ __forceinline__ EpilogueOps epilogue_read(const Epilogue& e, uint64_t b, uint64_t row) {
  return EpilogueOps{e.bias ? load_elem(e.bias, row, e.bias_f32) : 0.f,
                     e.mul ? load_elem(e.mul, b * e.mul_stride + row, e.mul_f32) : 1.f,
                     e.residual ? load_elem(e.residual, b * e.residual_stride + row, e.residual_f32) : 0.f};
}
__device__ __forceinline__ void epilogue_write(const Epilogue& e, uint64_t b, uint64_t row, float z, const EpilogueOps& o) {
  if (e.bias) z += o.bias;
  z = act_apply(e.act, z);
  if (e.mul) z *= o.mul;
  if (e.residual) z += o.residual;
  if (e.y_f32)
    static_cast<float*>(e.y)[b * e.y_stride + row] = z;
  else
    static_cast<__nv_bfloat16*>(e.y)[b * e.y_stride + row] = __float2bfloat16_rn(z);
}
__device__ __forceinline__ void epilogue_store(const Epilogue& e, uint64_t b, uint64_t row, float z) {
  epilogue_write(e, b, row, z, epilogue_read(e, b, row));
}

// Eight elements at index i of a BF16 or FP32 array, 16-byte aligned there.
__device__ __forceinline__ void load8(const void* p, uint64_t i, bool f32, float* v) {
  if (f32) {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    const float4 a = q[0], b = q[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p) + i);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[2 * k] = __uint_as_float(w[k] << 16);
      v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
    }
  }
}

// z[0 .. 7] of token b into y's columns row .. row + 7 (n of them exist):
// 16-byte accesses where every operand allows them (Epilogue::vec, row a
// multiple of 8 past a multiple-of-8 start), else one by one.
__device__ __forceinline__ void epilogue_store8(const Epilogue& e, uint64_t b, uint64_t row, float* z, int n) {
  if (!e.vec || n < 8) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < n) epilogue_store(e, b, row + k, z[k]);
    return;
  }
  float t[8];
  if (e.bias) {
    load8(e.bias, row, e.bias_f32, t);
#pragma unroll
    for (int k = 0; k < 8; ++k) z[k] += t[k];
  }
  if (e.act) {
#pragma unroll
    for (int k = 0; k < 8; ++k) z[k] = act_apply(e.act, z[k]);
  }
  if (e.mul) {
    load8(e.mul, b * e.mul_stride + row, e.mul_f32, t);
#pragma unroll
    for (int k = 0; k < 8; ++k) z[k] *= t[k];
  }
  if (e.residual) {
    load8(e.residual, b * e.residual_stride + row, e.residual_f32, t);
#pragma unroll
    for (int k = 0; k < 8; ++k) z[k] += t[k];
  }
  const uint64_t at = b * e.y_stride + row;
  if (e.y_f32) {
    float4* q = reinterpret_cast<float4*>(static_cast<float*>(e.y) + at);
    q[0] = make_float4(z[0], z[1], z[2], z[3]);
    q[1] = make_float4(z[4], z[5], z[6], z[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(z[2 * k], z[2 * k + 1]);
      w[k] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(e.y) + at) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

}  // namespace xksv
