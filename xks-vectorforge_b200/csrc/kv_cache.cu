// Paged key/value cache (include/xksv_cuda.h, part 8): the append of new
// tokens with their position rotation, and the attention of one new token per
// sequence over the cached ones.
//
// This file holds the kernels and their C entries; the cache itself is the
// caller's memory, the handle its geometry and a device status word.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <new>
#include <utility>

#include "kv_cache.h"
#include "kv_index.h"
#include "xksv_types.h"

struct xksv_kv {
  int device = 0, sms = 148;
  xksv_kv_desc d{};
  int* d_status = nullptr;
  int* h_status = nullptr;
};

namespace xksv {
namespace {

// Runs a call on the handle's device, whichever is current.
struct DeviceGuard {
  int before = -1;
  bool ok = false;
  explicit DeviceGuard(int dev) {
    if (cudaGetDevice(&before) != cudaSuccess) return;
    ok = before == dev || cudaSetDevice(dev) == cudaSuccess;
    if (before == dev) before = -1;
  }
  ~DeviceGuard() {
    if (before >= 0) cudaSetDevice(before);
  }
};

// ------------------------------------------------------------- elements ---
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

// --------------------------------------------------------------- append ---
// Bound: memory (every element is read once and written once) for prompts,
// the chain of dependent loads (place -> page -> store) for a few tokens.  A
// CTA takes tokens in turn: a token's page is looked up and its angles are
// computed while its first rows are already being read.  A thread moves 8
// elements (and, rotated in halves, their 8 partners) at a time and keeps its
// place in the row, so that it reads its angles once a token and divides no
// index in the loop.
constexpr int AT = 128;         // threads per token
constexpr int kMaxPairs = 128;  // head_dim <= 256
constexpr int kPerSm = 6;       // CTAs an SM holds (16384 tokens: 71 us; three of 256 threads 83 us)

// cos and sin of a token's angles into shared memory.  The angle is formed in
// 64 bits, less its whole turns: an FP32 product would be wrong by radians at
// far positions.
__device__ __forceinline__ void angles(const xksv_kv_append_args& a, int32_t pos, float* cs, float* sn) {
  constexpr double kTurn = 6.283185307179586476925286766559, kTurns = 1.0 / kTurn, kHalfTurns = 2.0 / kTurn;
  for (uint32_t i = threadIdx.x; i < a.rot_dim / 2; i += AT) {
    const double angle = double(pos) * double(a.inv_freq[i]);
    float sv, cv;
    sincospif(float(fma(-rint(angle * kTurns), kTurn, angle) * kHalfTurns), &sv, &cv);
    cs[i] = cv * a.rot_scale;
    sn[i] = sv * a.rot_scale;
  }
}

// A token's place in the cache (below 2^31: 32-bit division); page -1:
// nothing of it is stored.
__device__ __forceinline__ KvPlace token_place(const AppendArgs& p, int64_t seq, int32_t idx) {
  if (seq < 0 || idx < 0) return KvPlace{-1, 0};  // padding
  const KvPlace at = kv_place(p.a.table, p.a.table_rows, p.a.table_cols, p.a.table_stride, p.c.pages, uint32_t(p.c.page_size), seq, idx);
  if (at.page < 0 && threadIdx.x == 0) atomicOr(p.status, kStatusHeader);
  return at;
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

// Rows of 16-byte pieces (alignment, and rotated pairs that fill them) whose
// heads lie less than 2^31 elements apart.  16384 tokens of 32 + 8 heads of
// 128 in BF16: 71.6 us, 5625 GB/s; 3001 tokens of 20 + 20 heads of 80 in FP16
// 16.7 us; one token 3.1 us.
template <class TI, class TC>
__global__ void __launch_bounds__(AT, kPerSm) kv_append_kernel(const AppendArgs p) {
  __shared__ __align__(16) float cs[2][kMaxPairs], sn[2][kMaxPairs];
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  using In = Eight<TI>;
  using Out = Eight<TC>;
  const uint32_t D = p.c.head_dim, rot = p.a.rot_dim, H = p.c.kv_heads, nq = p.a.q ? p.a.q_heads : 0;
  const bool inter = p.a.flags & XKSV_KV_INTERLEAVED;
  const uint32_t pairs = inter ? 0 : rot / 16;  // threads of a row that hold two pieces
  const uint32_t per = D / 8 - pairs, vper = D / 8;
  const uint32_t rows = nq + H, step = AT / per, vstep = AT / vper;
  // this thread's piece of a query or key row, and the first of its rows; the
  // same for values (a row beyond the last: nothing to do)
  const uint32_t c = threadIdx.x % per, d = c < pairs ? 8 * c : 8 * (c + pairs), half = c < pairs ? rot / 2 : 0;
  const uint32_t row0 = threadIdx.x / per < step ? threadIdx.x / per : rows;
  const uint32_t vd = 8 * (threadIdx.x % vper), vrow0 = threadIdx.x / vper < vstep ? threadIdx.x / vper : H;
  const bool turn = half || (inter && d < rot);
  struct Token {
    int32_t idx, pos;
    int64_t seq;
  };
  auto token = [&](uint64_t t) {
    Token k;
    k.idx = p.a.index[t];
    k.seq = p.a.seq ? int64_t(p.a.seq[t]) : int64_t(t);
    k.pos = p.a.positions ? p.a.positions[t] : int32_t(k.idx);
    return k;
  };
  // head strides fit 32 bits here, and so does a row's offset from its token's
  const uint32_t qs = uint32_t(p.a.q_stride[1]), ks = uint32_t(p.a.k_stride[1]), vs = uint32_t(p.a.v_stride[1]);
  auto source = [&](uint64_t t, uint32_t r) {
    return r < nq ? static_cast<const TI*>(p.a.q) + t * p.a.q_stride[0] + (r * qs + d)
                  : static_cast<const TI*>(p.a.k) + t * p.a.k_stride[0] + ((r - nq) * ks + d);
  };
  auto store = [&](TC* dst, float* x, const float* scale, uint32_t h) {
    if (scale) {
      const float f = scale[h];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] /= f;
    }
    Out y;
    gather(x, y);
    *reinterpret_cast<Out*>(dst) = y;
  };
  // pieces read before the angles are there: two rows' pairs, or four rows
  constexpr int kAhead = 4;
  uint32_t buf = 0;
  Token k = token(blockIdx.x);
  for (uint64_t t = blockIdx.x; t < p.a.tokens; t += gridDim.x, buf ^= 1) {
    const bool live = k.idx >= 0 && k.seq >= 0;  // padding's rows are not read
    In a[kAhead], v;
#pragma unroll
    for (int y = 0; y < kAhead; ++y) {
      const uint32_t r = row0 + (half ? y / 2 : y) * step;
      if (live && r < rows) a[y] = *reinterpret_cast<const In*>(source(t, r) + (half && y % 2 ? half : 0));
    }
    const TI* vsrc = static_cast<const TI*>(p.a.v) + t * p.a.v_stride[0] + vd;
    if (live && vrow0 < H) v = *reinterpret_cast<const In*>(vsrc + vrow0 * vs);
    const KvPlace at = token_place(p, k.seq, k.idx);
    if (live) angles(p.a, k.pos, cs[buf], sn[buf]);
    if (t + gridDim.x < p.a.tokens) k = token(t + gridDim.x);
    __syncthreads();
    if (at.page < 0) continue;
    // halves: eight angles; pairs: four, each for two elements
    const float4* c4 = reinterpret_cast<const float4*>(&cs[buf][half ? d : d / 2]);
    const float4* s4 = reinterpret_cast<const float4*>(&sn[buf][half ? d : d / 2]);
    TC* ck = static_cast<TC*>(p.c.k) + uint64_t(at.page) * p.c.k_stride[0] + at.place * p.c.k_stride[1] + d;
    TC* cv = static_cast<TC*>(p.c.v) + uint64_t(at.page) * p.c.v_stride[0] + at.place * p.c.v_stride[1] + vd;
    TI* qo = static_cast<TI*>(p.a.q_out) + t * p.a.q_out_stride[0] + d;
    auto work = [&](uint32_t r, const In& a, const In& b) {
      float x[8], y[8];
      spread(a, x);
      if (half) {
        spread(b, y);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const float4 cv4 = c4[g], sv4 = s4[g];
          const float co[4] = {cv4.x, cv4.y, cv4.z, cv4.w}, si[4] = {sv4.x, sv4.y, sv4.z, sv4.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float u = x[4 * g + e], w = y[4 * g + e];
            x[4 * g + e] = u * co[e] - w * si[e];
            y[4 * g + e] = w * co[e] + u * si[e];
          }
        }
      } else if (turn) {
        const float4 cv4 = c4[0], sv4 = s4[0];
        const float co[4] = {cv4.x, cv4.y, cv4.z, cv4.w}, si[4] = {sv4.x, sv4.y, sv4.z, sv4.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float u = x[2 * e], w = x[2 * e + 1];
          x[2 * e] = u * co[e] - w * si[e];
          x[2 * e + 1] = w * co[e] + u * si[e];
        }
      }
      if (r < nq) {
        TI* dst = qo + r * uint32_t(p.a.q_out_stride[1]);
        In o;
        gather(x, o);
        *reinterpret_cast<In*>(dst) = o;
        if (half) {
          gather(y, o);
          *reinterpret_cast<In*>(dst + half) = o;
        }
      } else {
        TC* dst = ck + (r - nq) * uint32_t(p.c.k_stride[2]);
        store(dst, x, p.c.k_scale, r - nq);
        if (half) store(dst + half, y, p.c.k_scale, r - nq);
      }
    };
    uint32_t r = row0;
    if (half) {
#pragma unroll
      for (int y = 0; y < kAhead / 2; ++y, r += step)
        if (r < rows) work(r, a[2 * y], a[2 * y + 1]);
    } else {
#pragma unroll
      for (int y = 0; y < kAhead; ++y, r += step)
        if (r < rows) work(r, a[y], a[y]);
    }
    for (; r < rows; r += step) {
      const TI* src = source(t, r);
      a[0] = *reinterpret_cast<const In*>(src);
      if (half) a[1] = *reinterpret_cast<const In*>(src + half);
      work(r, a[0], a[1]);
    }
    for (uint32_t r = vrow0; r < H; r += vstep) {
      if (r != vrow0) v = *reinterpret_cast<const In*>(vsrc + r * vs);
      float x[8];
      spread(v, x);
      store(cv + r * uint32_t(p.c.v_stride[2]), x, p.c.v_scale, r);
    }
  }
}

// Any strides, alignment and rotation: element by element, a thread per pair.
template <class TI, class TC>
__global__ void __launch_bounds__(AT) kv_append_any_kernel(const AppendArgs p) {
  __shared__ float cs[kMaxPairs], sn[kMaxPairs];
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  const uint64_t t = blockIdx.x;
  const int32_t idx = p.a.index[t];
  const KvPlace at = token_place(p, p.a.seq ? int64_t(p.a.seq[t]) : int64_t(t), idx);
  if (at.page < 0) return;
  const uint32_t D = p.c.head_dim, half = p.a.rot_dim / 2;
  angles(p.a, p.a.positions ? p.a.positions[t] : idx, cs, sn);
  __syncthreads();
  const bool inter = p.a.flags & XKSV_KV_INTERLEAVED;
  const uint32_t items = D - half;  // pairs, then single elements
  const TI* q = static_cast<const TI*>(p.a.q) + t * p.a.q_stride[0];
  TI* qo = static_cast<TI*>(p.a.q_out) + t * p.a.q_out_stride[0];
  const TI* k = static_cast<const TI*>(p.a.k) + t * p.a.k_stride[0];
  const TI* v = static_cast<const TI*>(p.a.v) + t * p.a.v_stride[0];
  TC* ck = static_cast<TC*>(p.c.k) + uint64_t(at.page) * p.c.k_stride[0] + at.place * p.c.k_stride[1];
  TC* cv = static_cast<TC*>(p.c.v) + uint64_t(at.page) * p.c.v_stride[0] + at.place * p.c.v_stride[1];
  const uint32_t nq = p.a.q ? p.a.q_heads : 0;
  for (uint32_t w = threadIdx.x; w < (nq + p.c.kv_heads) * items; w += AT) {
    const uint32_t hh = w / items, i = w - hh * items;
    const bool is_q = hh < nq;
    const uint32_t h = is_q ? hh : hh - nq;
    const TI* src = is_q ? q + h * p.a.q_stride[1] : k + h * p.a.k_stride[1];
    const float f = !is_q && p.c.k_scale ? p.c.k_scale[h] : 1.f;
    auto put = [&](uint32_t d, float x) {
      if (is_q)
        qo[h * p.a.q_out_stride[1] + d] = from_float<TI>(x);
      else
        ck[h * p.c.k_stride[2] + d] = from_float<TC>(p.c.k_scale ? x / f : x);
    };
    if (i < half) {
      const uint32_t da = inter ? 2 * i : i, db = inter ? 2 * i + 1 : i + half;
      const float a = to_float(src[da]), b = to_float(src[db]);
      put(da, a * cs[i] - b * sn[i]);
      put(db, b * cs[i] + a * sn[i]);
    } else {
      const uint32_t d = i + half;
      put(d, to_float(src[d]));
    }
  }
  for (uint32_t w = threadIdx.x; w < p.c.kv_heads * D; w += AT) {
    const uint32_t h = w / D, d = w - h * D;
    const float x = to_float(v[h * p.a.v_stride[1] + d]);
    cv[h * p.c.v_stride[2] + d] = from_float<TC>(p.c.v_scale ? x / p.c.v_scale[h] : x);
  }
}

template <class TI, class TC>
cudaError_t append_launch(const AppendArgs& p, int sms, cudaStream_t st) {
  auto whole = [](const void* ptr, const uint64_t* stride) {  // rows of 16-byte pieces
    return (reinterpret_cast<uintptr_t>(ptr) | stride[0] * sizeof(TI) | stride[1] * sizeof(TI)) % 16 == 0;
  };
  auto near = [](uint64_t heads, uint64_t stride) { return stride < (1ull << 31) / heads; };
  const bool close = near(p.c.kv_heads, p.a.k_stride[1]) && near(p.c.kv_heads, p.a.v_stride[1]) &&
                     near(p.c.kv_heads, p.c.k_stride[2]) && near(p.c.kv_heads, p.c.v_stride[2]) &&
                     (!p.a.q || (near(p.a.q_heads, p.a.q_stride[1]) && near(p.a.q_heads, p.a.q_out_stride[1])));
  const bool pieces = close && p.a.rot_dim % (p.a.flags & XKSV_KV_INTERLEAVED ? 8 : 16) == 0 && whole(p.a.k, p.a.k_stride) &&
                      whole(p.a.v, p.a.v_stride) &&
                      (!p.a.q || (whole(p.a.q, p.a.q_stride) && whole(p.a.q_out, p.a.q_out_stride)));
  cudaLaunchConfig_t cfg = {};
  // the piecewise kernel's CTAs loop over the tokens, as many as the GPU holds
  cfg.gridDim = dim3(uint32_t(pieces ? std::min<uint64_t>(p.a.tokens, kPerSm * sms) : p.a.tokens));
  cfg.blockDim = dim3(AT);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, pieces ? kv_append_kernel<TI, TC> : kv_append_any_kernel<TI, TC>, p);
}

template <class TI>
cudaError_t append_cache(const AppendArgs& p, int sms, cudaStream_t st) {
  switch (p.c.type) {
    case XKSV_BF16: return append_launch<TI, __nv_bfloat16>(p, sms, st);
    case XKSV_FP16: return append_launch<TI, __half>(p, sms, st);
    default: return append_launch<TI, E4m3>(p, sms, st);
  }
}

// ---------------------------------------------------------- C entry checks
uint64_t elem_bytes(uint32_t type) { return type == XKSV_E4M3 ? 1 : type == XKSV_FP32 ? 4 : 2; }
bool off_align(const void* p, uintptr_t align) { return (reinterpret_cast<uintptr_t>(p) & (align - 1)) != 0; }

// The elements of a cache buffer lie inside it, on 16-byte rows, and no two
// (page, token, head) rows overlap: ordered by stride, each dimension steps
// past the whole extent of the smaller ones.
bool strides_ok(const xksv_kv_desc& d, const void* base, uint64_t bytes, const uint64_t* stride) {
  const uint64_t e = elem_bytes(d.type), total = bytes / e;
  if (!base || off_align(base, 16)) return false;
  struct Dim {
    uint64_t n, stride;
  } dim[3] = {{d.pages, stride[0]}, {d.page_size, stride[1]}, {d.kv_heads, stride[2]}};
  for (int i = 0; i < 3; ++i)
    for (int j = i + 1; j < 3; ++j)
      if (dim[j].stride < dim[i].stride) std::swap(dim[i], dim[j]);
  uint64_t extent = d.head_dim;
  if (extent > total) return false;
  for (const Dim& x : dim) {
    if (x.n == 1) continue;
    if (x.stride * e % 16 || x.stride < extent) return false;
    if (x.stride > (total - extent) / (x.n - 1)) return false;
    extent += x.stride * (x.n - 1);
  }
  return true;
}

// No two rows of an output [n, heads, dim] overlap.
bool rows_distinct(uint64_t n, uint64_t heads, uint64_t dim, const uint64_t* stride) {
  const bool token_major = stride[0] >= stride[1];
  const uint64_t n0 = token_major ? heads : n, s0 = token_major ? stride[1] : stride[0];
  const uint64_t n1 = token_major ? n : heads, s1 = token_major ? stride[0] : stride[1];
  if (n0 > 1 && s0 < dim) return false;
  const uint64_t extent = n0 > 1 ? s0 * (n0 - 1) + dim : dim;
  return n1 <= 1 || s1 >= extent;
}
bool strides_small(const uint64_t* stride) { return stride[0] < (1ull << 40) && stride[1] < (1ull << 40); }

}  // namespace

cudaError_t launch_kv_append(const AppendArgs& p, int sms, cudaStream_t st) {
  switch (p.a.type) {
    case XKSV_BF16: return append_cache<__nv_bfloat16>(p, sms, st);
    case XKSV_FP16: return append_cache<__half>(p, sms, st);
    default: return append_cache<float>(p, sms, st);
  }
}

}  // namespace xksv

using namespace xksv;

extern "C" {

int xksv_kv_create(const xksv_kv_desc* desc, xksv_kv** out) {
  if (!out) return 1;
  *out = nullptr;
  if (!desc || desc->flags || (desc->type != XKSV_BF16 && desc->type != XKSV_FP16 && desc->type != XKSV_E4M3)) return 1;
  const xksv_kv_desc& d = *desc;
  constexpr uint64_t kDim = 1ull << 31;
  if (!d.pages || !d.page_size || !d.kv_heads || !d.head_dim || d.head_dim > 256 || d.pages >= kDim ||
      d.page_size >= kDim || d.kv_heads > 65535 || d.head_dim * elem_bytes(d.type) % 16)
    return 1;
  if (d.type != XKSV_E4M3 && (d.k_scale || d.v_scale)) return 1;
  if (off_align(d.k_scale, 4) || off_align(d.v_scale, 4)) return 1;
  for (int i = 0; i < 3; ++i)
    if (d.k_stride[i] >= (1ull << 48) || d.v_stride[i] >= (1ull << 48)) return 1;
  if (!strides_ok(d, d.k, d.k_bytes, d.k_stride) || !strides_ok(d, d.v, d.v_bytes, d.v_stride)) return 1;
  auto* kv = new (std::nothrow) xksv_kv();
  if (!kv) return 1;
  kv->d = d;
  const bool ok = cudaGetDevice(&kv->device) == cudaSuccess &&
                  cudaDeviceGetAttribute(&kv->sms, cudaDevAttrMultiProcessorCount, kv->device) == cudaSuccess &&
                  cudaMalloc(&kv->d_status, sizeof(int)) == cudaSuccess &&
                  cudaMallocHost(&kv->h_status, sizeof(int)) == cudaSuccess &&
                  cudaMemset(kv->d_status, 0, sizeof(int)) == cudaSuccess && cudaStreamSynchronize(nullptr) == cudaSuccess;
  if (!ok) {
    cudaGetLastError();  // not the next launch's
    xksv_kv_destroy(kv);
    return 1;
  }
  *out = kv;
  return 0;
}

void xksv_kv_destroy(xksv_kv* kv) {
  if (!kv) return;
  if (kv->d_status) cudaFree(kv->d_status);
  if (kv->h_status) cudaFreeHost(kv->h_status);
  delete kv;
}

int xksv_kv_status(const xksv_kv* kv, void* stream) {
  if (!kv) return 1;
  DeviceGuard guard(kv->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!guard.ok || cudaMemcpyAsync(kv->h_status, kv->d_status, sizeof(int), cudaMemcpyDeviceToHost, st) != cudaSuccess ||
      cudaStreamSynchronize(st) != cudaSuccess)
    return 1;
  const int v = *kv->h_status;
  if (v && (cudaMemsetAsync(kv->d_status, 0, sizeof(int), st) != cudaSuccess || cudaStreamSynchronize(st) != cudaSuccess))
    return 1;
  return v == 0 ? 0 : 1;
}

int xksv_kv_append(const xksv_kv* kv, const xksv_kv_append_args* a, void* stream) {
  if (!kv || !a || (a->flags & ~XKSV_KV_INTERLEAVED)) return 1;
  if (a->type != XKSV_BF16 && a->type != XKSV_FP16 && a->type != XKSV_FP32) return 1;
  if (a->rot_dim % 2 || a->rot_dim > kv->d.head_dim || (a->rot_dim && !a->inv_freq) || off_align(a->inv_freq, 4)) return 1;
  if (!a->q != !a->q_out || (a->q && (!a->q_heads || a->q_heads > 65535))) return 1;
  if (!a->tokens) return 0;
  const uintptr_t e = elem_bytes(a->type);
  if (!a->k || !a->v || !a->table || !a->index || a->tokens >= (1ull << 31) || !a->table_rows || !a->table_cols ||
      (a->table_rows > 1 && a->table_stride < a->table_cols) || off_align(a->table, 4) || off_align(a->seq, 4) ||
      off_align(a->index, 4) || off_align(a->positions, 4) || off_align(a->q, e) || off_align(a->k, e) ||
      off_align(a->v, e) || off_align(a->q_out, e))
    return 1;
  if (!strides_small(a->k_stride) || !strides_small(a->v_stride) ||
      (a->q && (!strides_small(a->q_stride) || !strides_small(a->q_out_stride) ||
                !rows_distinct(a->tokens, a->q_heads, kv->d.head_dim, a->q_out_stride))))
    return 1;
  DeviceGuard guard(kv->device);
  if (!guard.ok) return 1;
  const AppendArgs p{*a, kv->d, kv->d_status};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return launch_kv_append(p, kv->sms, st) == cudaSuccess ? 0 : 1;
}

size_t xksv_kv_attend_workspace(const xksv_kv* kv, size_t seqs, size_t q_heads, size_t table_cols) {
  if (!kv || !seqs || !q_heads || q_heads % kv->d.kv_heads || q_heads > 65535 || !table_cols || table_cols >= (1ull << 31))
    return 0;
  return size_t(kv_attend_plan(kv->d, seqs, uint32_t(q_heads), table_cols, kv->sms).bytes);
}

int xksv_kv_attend(const xksv_kv* kv, const xksv_kv_attend_args* a, void* d_workspace, size_t workspace_bytes,
                   void* stream) {
  if (!kv || !a || !a->q_heads || a->q_heads % kv->d.kv_heads || a->q_heads > 65535) return 1;
  if (a->type != XKSV_BF16 && a->type != XKSV_FP16) return 1;
  if (kv->d.type != XKSV_E4M3 && kv->d.type != a->type) return 1;
  if (!(a->softcap >= 0.f) || a->seqs >= (1ull << 31)) return 1;
  if (!a->seqs) return 0;
  if (!a->q || !a->out || !a->table || !a->lens || !a->table_cols || a->table_cols >= (1ull << 31) ||
      (a->seqs > 1 && a->table_stride < a->table_cols) || off_align(a->q, 2) || off_align(a->out, 2) ||
      off_align(a->lse, 4) || off_align(a->table, 4) || off_align(a->lens, 4))
    return 1;
  if (!strides_small(a->q_stride) || !strides_small(a->out_stride) ||
      !rows_distinct(a->seqs, a->q_heads, kv->d.head_dim, a->out_stride))
    return 1;
  const AttendPlan pl = kv_attend_plan(kv->d, a->seqs, a->q_heads, a->table_cols, kv->sms);
  if (pl.bytes && (!d_workspace || workspace_bytes < pl.bytes || off_align(d_workspace, 256))) return 1;
  DeviceGuard guard(kv->device);
  if (!guard.ok) return 1;
  auto* ws = static_cast<uint8_t*>(d_workspace);
  const AttendArgs p{*a, kv->d, kv->d_status, reinterpret_cast<float*>(ws), reinterpret_cast<int4*>(ws + pl.joins_off)};
  return launch_kv_attend(p, pl, static_cast<cudaStream_t>(stream)) == cudaSuccess ? 0 : 1;
}

}  // extern "C"
