// Elements of the paged cache's calls, and a position's rotation: what the
// append kernels share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

namespace xksv {
namespace {

struct E4m3 {
  __nv_fp8_storage_t b;
};
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(float x) { return x; }
template <class T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}
template <>
__device__ __forceinline__ __half from_float<__half>(float x) {
  return __float2half_rn(x);
}
template <>
__device__ __forceinline__ float from_float<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ E4m3 from_float<E4m3>(float x) {
  return E4m3{__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3)};
}

// Cosine and sine of position * freq, times `scale`.  The angle is formed in 64
// bits, less its whole turns: an FP32 product would be wrong by radians at far
// positions.
__device__ __forceinline__ void angle_of(int32_t pos, float freq, float scale, float* cs, float* sn) {
  constexpr double kTurn = 6.283185307179586476925286766559, kTurns = 1.0 / kTurn, kHalfTurns = 2.0 / kTurn;
  const double angle = double(pos) * double(freq);
  float sv, cv;
  sincospif(float(fma(-rint(angle * kTurns), kTurn, angle) * kHalfTurns), &sv, &cv);
  *cs = cv * scale;
  *sn = sv * scale;
}

// Eight elements as 32-bit words (E4M3: two, 16-bit types: four, FP32: eight).
template <class T>
struct alignas(sizeof(T) == 1 ? 8 : 16) Eight {
  uint32_t w[sizeof(T) * 2];
};
__device__ __forceinline__ void spread(const Eight<__nv_bfloat16>& a, float* x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(a.w[i] << 16);
    x[2 * i + 1] = __uint_as_float(a.w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void spread(const Eight<__half>& a, float* x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a.w[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void spread(const Eight<float>& a, float* x) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(a.w[i]);
}
__device__ __forceinline__ void gather(const float* x, Eight<__nv_bfloat16>& a) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    a.w[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
}
__device__ __forceinline__ void gather(const float* x, Eight<__half>& a) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 v = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    a.w[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
}
__device__ __forceinline__ void gather(const float* x, Eight<float>& a) {
#pragma unroll
  for (int i = 0; i < 8; ++i) a.w[i] = __float_as_uint(x[i]);
}
__device__ __forceinline__ void gather(const float* x, Eight<E4m3>& a) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i], x[4 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i + 2], x[4 * i + 3]), __NV_SATFINITE, __NV_E4M3);
    a.w[i] = lo | hi << 16;
  }
}

}  // namespace
}  // namespace xksv
