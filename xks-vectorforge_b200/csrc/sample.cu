// Sampling of the next token of each row of logits (include/xksv_cuda.h,
// part 9): temperature, top-k, top-p and min-p, drawn with a given number.
//
// Tokens are ordered by logit, equal ones by index; each of the three filters
// keeps a prefix of that order, so a row's kept tokens are those above a
// border: a logit, and among the tokens of that logit an index.  The draw goes
// through the kept tokens by index, so nothing is sorted but the few
// candidates next to the border:
//   * a cluster of CTAs takes a row and holds it in shared memory: the logits
//     are read from HBM once (a row larger than its CTAs hold is read again by
//     every pass: more than eight hold, or, of rows that do not fit an SM twice, so many that
//     fewer CTAs a row are faster all the same, as in `launch`);
//   * few kept tokens: the largest logits of groups of lanes guess a distance
//     from the largest logit that as many tokens lie within as are wanted, or a few
//     more; those are gathered, sorted and drawn from by the first CTA, up to 64
//     of them by one warp without a barrier;
//   * many, in BF16: each logit has a bin of its own, so that the bins' weights say where the
//     border lies and which CTA the draw falls in;
//   * many else: a histogram of the distances says where the border lies, a pass sums
//     the weights above it, and the tokens next to it are sorted; too many of
//     them are narrowed by quarters of their bits, and of equal logits the first by
//     index are counted off;
//   * weights exp((z - largest) / temperature) and their sums are FP64: FP32
//     sums of 10^5 weights are off by more than the smaller ones, so that the
//     border and the drawn token would depend on the order of the additions.
//     All sums have a fixed order: the same call gives the same tokens.
//   * the CTAs of a row tell each other their numbers by stores into all the
//     others' shared memory ahead of a cluster barrier, so that each has all of them after it.
// Bound: for one row the chain of passes and cluster barriers (1 us each); for
// many such chains, with two CTAs an SM to hide them, and the passes' instructions,
// 45 of them an FP64 weight.  Measured on one B200: one row of 32000 BF16 logits,
// top-k 40 and top-p, 6.4 us; one of 128256 FP32 logits with 98000 tokens in the
// nucleus 40 us; 77 rows of 32003 FP16, each with its own settings, 41 us; 256 rows of
// 128256 BF16 so 123 us (a read of the logits: 10 us).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "kernels.h"
#include "sample.h"
#include "tcgen05.cuh"

namespace xksv {
namespace {

constexpr int NT = 512;  // threads of a CTA
constexpr int NW = NT / 32;
constexpr int kMaxCluster = 8;
constexpr int kParts = kMaxCluster * NW;  // warps of a row
constexpr int kGroups = 2048;             // groups of lanes whose largest logits guess the border
constexpr int NB = 2048;                  // bins of the histogram of logits
constexpr float kPerUnit = 128.f;         // of them, a unit of distance from the largest
constexpr uint32_t kEvery = 8;            // a vector in so many is sampled
constexpr uint32_t kGuessMost = 1200;     // tokens that are looked for so, at most: of more CAP would not hold all
constexpr int kGuessBins = 256;           // bins of the groups' largest logits
constexpr float kGuessPerUnit = 8.f;
constexpr int CAP = 2048;                 // candidates that are sorted
constexpr uint32_t kSide = 2048;          // BF16 magnitudes with a bin of their own: 16 binades
constexpr uint32_t kLeast = 0x3a80;       // from 2^-10, or higher ones
constexpr double kTiny = -700.0;          // weights below exp(kTiny) count as zero

struct Shared {
  alignas(16) uint32_t hist[NB];
  uint64_t list[CAP];  // this CTA's candidates: ~key, index
  float group[kGroups];
  uint64_t all[CAP];  // of the first CTA: all of them
  double part_w[2][2][kParts];  // of the row's warps, in turn
  uint32_t part_c[2][2][kParts];
  double quarter_w[2][4][kParts];
  uint32_t quarter_c[2][4][kParts];
  uint32_t part_lo[2][kParts], part_hi[2][kParts];  // their candidates' least and largest keys
  double scan_w[NW];
  uint32_t scan_c[NW];
  float best[kParts];
  double pow[16];  // 2^(i / 16)
  double guessed;
  float spread[NW];
  uint32_t listed, low, first, found;
  uint32_t ctl[2];
};

// Order-preserving integer of a float (no NaN; -0 is +0 by then).
__device__ __forceinline__ uint32_t key_of(float z) {
  const uint32_t b = __float_as_uint(z);
  return b ^ (uint32_t(int32_t(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// The larger; NaN when one is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// A float as a double, put together from its bits: the converter's rate (a
// quarter of FP64's) would bound every pass of weights.  Zero and subnormal numbers become
// numbers of 2^-127, infinity 2^128.
__device__ __forceinline__ double widened(float z) {
  const uint32_t b = __float_as_uint(z);
  return __hiloint2double(int((b & 0x80000000u) | (((b & 0x7fffffffu) >> 3) + 0x38000000u)), int(b << 29));
}
// A float of [0, 2^22) rounded to an integer, by the adder for the same reason.
__device__ __forceinline__ uint32_t rounded(float x) { return __float_as_uint(x + 12582912.f) - 0x4b400000u; }

template <class T>
struct Elems;  // of a 16-byte vector
template <>
struct Elems<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void get(const uint4& v, float* z) {
    z[0] = __uint_as_float(v.x), z[1] = __uint_as_float(v.y), z[2] = __uint_as_float(v.z), z[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ float most(const uint4& v) {
    return max_nan(max_nan(__uint_as_float(v.x), __uint_as_float(v.y)), max_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
};
template <>
struct Elems<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& v, float* z) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) z[2 * i] = __uint_as_float(w[i] << 16), z[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  static __device__ __forceinline__ float most(const uint4& v) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return __bfloat162float(__hmax_nan(m.x, m.y));
  }
};
template <>
struct Elems<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& v, float* z) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      z[2 * i] = f.x, z[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ float most(const uint4& v) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
    const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return __half2float(__hmax_nan(m.x, m.y));
  }
};
template <class T>
__device__ __forceinline__ T lowest();  // -infinity: no weight
template <>
__device__ __forceinline__ float lowest<float>() { return -INFINITY; }
template <>
__device__ __forceinline__ __nv_bfloat16 lowest<__nv_bfloat16>() { return __ushort_as_bfloat16(0xff80); }
template <>
__device__ __forceinline__ __half lowest<__half>() { return __ushort_as_half(0xfc00); }

// Another CTA's shared memory at this address.
__device__ __forceinline__ uint32_t at_rank(const void* p, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(smem_addr(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void push(double* p, uint32_t rank, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;\n" ::"r"(at_rank(p, rank)), "d"(v) : "memory");
}
__device__ __forceinline__ void push(uint32_t* p, uint32_t rank, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;\n" ::"r"(at_rank(p, rank)), "r"(v) : "memory");
}
__device__ __forceinline__ void push(float* p, uint32_t rank, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;\n" ::"r"(at_rank(p, rank)), "f"(v) : "memory");
}
__device__ __forceinline__ uint4 pull4(const uint32_t* p, uint32_t rank) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];\n"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(at_rank(p, rank))
               : "memory");
  return v;
}
__device__ __forceinline__ uint64_t pull(const uint64_t* p, uint32_t rank) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];\n" : "=l"(v) : "r"(at_rank(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t pull(const uint32_t* p, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];\n" : "=r"(v) : "r"(at_rank(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ void min_at(uint32_t* p, uint32_t rank, uint32_t n) {
  asm volatile("red.shared::cluster.min.u32 [%0], %1;\n" ::"r"(at_rank(p, rank)), "r"(n) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
  cluster_arrive();
  cluster_wait();
}

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
  return x;
}
// Inclusive scan over the warp's lanes.
template <class X>
__device__ __forceinline__ X warp_scan(X x, uint32_t lane) {
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const X o = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += o;
  }
  return x;
}
// HELD: the row lies in the cluster's shared memory (else every pass reads HBM or L2).
template <class T, bool HELD>
__global__ void __launch_bounds__(NT, 2) sample_kernel(const SampleArgs p) {
  using E = Elems<T>;
  constexpr int EPV = E::N;
  extern __shared__ __align__(16) uint8_t dyn[];
  Shared& s = *reinterpret_cast<Shared*>(dyn);
  uint4* const held = reinterpret_cast<uint4*>(dyn + p.held_off);
  const uint32_t C = p.cluster, rank = blockIdx.x % C;
  const uint64_t row = blockIdx.x / C;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, me = rank * NW + warp;
  const uint32_t V = uint32_t(p.a.vocab), parts = C * NW;
  cluster_arrive();  // (no CTA writes to another before it has begun)
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  asm volatile("griddepcontrol.wait;\n" ::: "memory");

  // this row's settings
  const float heat = p.a.temperature ? p.a.temperature[row] : p.a.temperature_all;
  const int32_t top_k = p.a.top_k ? p.a.top_k[row] : p.a.top_k_all;
  const float top_p = p.a.top_p ? p.a.top_p[row] : p.a.top_p_all;
  const float min_p = p.a.min_p ? p.a.min_p[row] : p.a.min_p_all;
  const float u = p.a.u[row];
  const bool sane = (heat == 0.f || (heat >= kSampleColdest && heat <= kSampleHottest)) && top_p == top_p && min_p == min_p && u == u;

  // ---- the row's 16-byte vectors; its first element is element `skew` of
  // the first vector; this warp's vectors [wv0, wv1)
  const T* const src = static_cast<const T*>(p.a.logits) + row * p.a.stride;
  const uint32_t skew = uint32_t(reinterpret_cast<uintptr_t>(src) % 16 / sizeof(T));
  const uint4* const vecs = reinterpret_cast<const uint4*>(src - skew);
  const uint32_t nv = (skew + V + EPV - 1) / EPV;
  const uint32_t per = (nv + C - 1) / C, v0 = min(nv, rank * per), v1 = min(nv, v0 + per);
  const uint32_t wper = (v1 - v0 + NW - 1) / NW, wv0 = min(v1, v0 + warp * wper), wv1 = min(v1, wv0 + wper);
  // vector v from HBM; elements outside the row are -infinity
  auto at_end = [&](uint32_t v) { return v == 0 || v + 1 == nv; };
  auto read_end = [&](uint32_t v) {
    uint4 w;
    T* e = reinterpret_cast<T*>(&w);
    for (int i = 0; i < EPV; ++i) {
      const uint32_t at = v * EPV + i;
      e[i] = at >= skew && at - skew < V ? src[at - skew] : lowest<T>();
    }
    return w;
  };
  auto read = [&](uint32_t v) { return at_end(v) ? read_end(v) : __ldg(vecs + v); };
  auto fetch = [&](uint32_t v, float* z) {
    E::get(HELD ? held[v - v0] : read(v), z);
#pragma unroll
    for (int i = 0; i < EPV; ++i) z[i] += 0.f;  // -0 becomes +0
  };

  // ---- the largest logit, of the row and of the groups of lanes ----
  float mine = -INFINITY;
  if (nv < 3)  // all are ends
    for (uint32_t v = wv0 + lane; v < wv1; v += 32) {
      const uint4 w = read_end(v);
      if (HELD) held[v - v0] = w;
      mine = max_nan(mine, E::most(w));
    }
  else for (uint32_t v = wv0 + lane; v < wv1; v += 128) {
    // four loads in flight, without a branch ahead of them: an end's is
    // another vector's at first
    uint4 w[4];
    const uint32_t last = wv1 - 1;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __ldg(vecs + max(1u, min(min(v + 32 * i, last), nv - 2)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t at = v + 32 * i;
      if (at >= wv1) break;
      if (at_end(at)) w[i] = read_end(at);
      if (HELD) held[at - v0] = w[i];
      mine = max_nan(mine, E::most(w[i]));
    }
  }
  if (tid < 16) s.pow[tid] = exp2(tid / 16.0);
  if (tid == 0) s.listed = 0, s.first = ~0u;
  // groups: a lane, or two or four; every CTA gets all of them.  Twice as many for
  // a large top-k (256 rows of 128256 BF16, top-k 1000, 224 and 197 us).
  const uint32_t groups = min(C * NT, uint32_t(top_k > kGroups * 3 / 8 && top_k <= int(kGuessMost) ? kGroups : kGroups / 2)), wide = C * NT / groups;
  cluster_wait();
  {
    float g = mine;
    if (wide > 1) g = max_nan(g, __shfl_xor_sync(0xffffffffu, g, 1));
    if (wide > 2) g = max_nan(g, __shfl_xor_sync(0xffffffffu, g, 2));
    for (uint32_t r = lane % wide; r < C; r += wide) push(&s.group[(rank * NT + tid) / wide], r, g);
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) mine = max_nan(mine, __shfl_xor_sync(0xffffffffu, mine, d));
    if (lane < C) push(&s.best[me], lane, mine);
  }
  cluster_sync();
  float zmax = -INFINITY;
  for (uint32_t i = lane; i < parts; i += 32) zmax = max_nan(zmax, s.best[i]);
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) zmax = max_nan(zmax, __shfl_xor_sync(0xffffffffu, zmax, d));
  zmax += 0.f;

  auto answer = [&](int64_t token, int32_t kept, float logprob) {
    p.a.tokens[row] = token;
    if (p.a.kept) p.a.kept[row] = kept;
    if (p.a.logprob) p.a.logprob[row] = logprob;
  };
  // a largest of NaN or +-infinity has no distribution
  if (!sane || !(fabsf(zmax) < INFINITY)) {
    if (rank == 0 && tid == 0) answer(-1, 0, NAN);
    return;
  }
  if (heat == 0.f || top_k == 1 || top_p <= 0.f) {  // the first of the largest
    uint32_t first = ~0u;
    for (uint32_t v = wv0 + lane; v < wv1; v += 32) {
      float z[EPV];
      fetch(v, z);
#pragma unroll
      for (int i = 0; i < EPV; ++i)
        if (z[i] == zmax) first = min(first, v * EPV + i - skew);
    }
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0 && first != ~0u) min_at(&s.first, 0, first);
    cluster_sync();
    if (rank == 0 && tid == 0) answer(s.first, 1, 0.f);
    return;
  }
  // exp((z - zmax) / heat) = 2^((n + f) / 16) with n whole and |f| <= 1/2; the
  // series of exp(r), r = f log(2) / 16, to the 6th power (the 7th: 5e-16), in
  // short chains: a pass of weights is bound by their latency.  No branch: a
  // token that does not count enters with -infinity.
  const double zm = widened(zmax), cool = 1.0 / double(heat);
  constexpr double kLn2 = 0.69314718055994530942, kBig = 6755399441055744.0;  // 1.5 * 2^52
  const double cool16 = 16.0 / kLn2 * cool;
  auto weight = [&](float z) {
    const double y = (widened(z) - zm) * cool16;
    const double big = y + kBig;
    const int n = __double2loint(big);
    const double r = (y - (big - kBig)) * (kLn2 / 16), r2 = r * r;
    const double a = fma(r, 1.0 / 6, 0.5), b = fma(r, 1.0 / 120, 1.0 / 24);
    const double e = s.pow[n & 15] * fma(r2, fma(r2, fma(r2, 1.0 / 720, b), a), 1.0 + r);
    return y < kTiny * 16.0 / kLn2 ? 0.0 : __hiloint2double(__double2hiint(e) + (n >> 4 << 20), __double2loint(e));
  };
  // the least logit that min-p and the smallest weight leave
  const double lowest_x = min_p > 0.f ? fmax(kTiny, log(fmin(1.0, double(min_p)))) : kTiny;
  const float floor_z = __double2float_ru(double(zmax) + lowest_x * double(heat));

  const bool by_k = top_k > 0 && uint32_t(top_k) < V, by_p = top_p < 1.f;

  // Every warp's numbers to every CTA; after the barrier that follows all warps
  // hold the same sums, added in the same order.  Two sets in turn: one may
  // still be read while the next is written.
  uint32_t turn = 0;
  auto share_w = [&](int i, double w) {
    w = warp_sum(w);
    if (lane < C) push(&s.part_w[turn][i][me], lane, w);
  };
  auto share_c = [&](int i, uint32_t c) {
    c = __reduce_add_sync(0xffffffffu, c);
    if (lane < C) push(&s.part_c[turn][i][me], lane, c);
  };
  auto sum_of = [&](const double* part) {
    double t = 0.0;
    for (uint32_t i = lane; i < parts; i += 32) t += part[i];
    return warp_sum(t);
  };
  auto count_of = [&](const uint32_t* part) {
    uint32_t t = 0;
    for (uint32_t i = lane; i < parts; i += 32) t += part[i];
    return __reduce_add_sync(0xffffffffu, t);
  };
  // A token to this CTA's list.
  auto list_it = [&](float z, uint32_t at) {
    const uint32_t n = atomicAdd(&s.listed, 1);
    if (n < CAP) s.list[n] = uint64_t(~key_of(z)) << 32 | at;
  };
  // The first CTA: s.all[0, n) in rising order (bitonic), E entries a thread in
  // registers: exchanges within a thread, then a warp, the farthest through
  // shared memory, two boxes in turn (the histogram's halves; of four entries
  // s.list too, which has been read by then).
  auto sort_by = [&](uint32_t n, auto entries) {
    constexpr uint32_t E = decltype(entries)::value;
    uint32_t full = 32 * E;
    while (full < n) full *= 2;
    uint64_t x[E];
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) x[e] = tid * E + e < n ? s.all[tid * E + e] : ~0ull;
    __syncthreads();
    bool flip = false;
    for (uint32_t size = 2; size <= full; size *= 2)
      for (uint32_t far = size / 2; far; far /= 2) {
        const bool up = !(tid * E & size);  // (of sizes up to E: by the entry)
        if (far < E) {
#pragma unroll
          for (uint32_t e = 0; e < E; ++e) {
            const uint32_t o = e ^ far;
            if (o > e && o < E) {
              const bool rise = size < E ? !(e & size) : up;
              uint64_t hi = 0;
#pragma unroll
              for (uint32_t j = 0; j < E; ++j)
                if (j == o) hi = x[j];
              if ((x[e] > hi) == rise) {
#pragma unroll
                for (uint32_t j = 0; j < E; ++j)
                  if (j == o) x[j] = x[e];
                x[e] = hi;
              }
            }
          }
        } else if (far < 32 * E) {
          const bool least = !(tid * E & far) == up;
#pragma unroll
          for (uint32_t e = 0; e < E; ++e) {
            const uint64_t y = __shfl_xor_sync(0xffffffffu, x[e], far / E);
            if ((x[e] > y) == least) x[e] = y;
          }
        } else {
          uint64_t* const halves = reinterpret_cast<uint64_t*>(s.hist);
          uint64_t* box = E == 1 ? halves + flip * NT : flip ? s.all : s.list;
          flip = !flip;
#pragma unroll
          for (uint32_t e = 0; e < E; ++e) box[e * NT + tid] = x[e];
          __syncthreads();
          const bool least = !(tid * E & far) == up;
#pragma unroll
          for (uint32_t e = 0; e < E; ++e) {
            const uint64_t y = box[e * NT + (tid ^ far / E)];
            if ((x[e] > y) == least) x[e] = y;
          }
        }
      }
    __syncthreads();
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) s.all[tid * E + e] = x[e];
    __syncthreads();
  };
  auto sort_all = [&](uint32_t n) {
    static_assert(CAP == 4 * NT, "up to four entries a thread");
    if (n <= NT)
      sort_by(n, std::integral_constant<uint32_t, 1>());
    else
      sort_by(n, std::integral_constant<uint32_t, 4>());
  };
  // Where each CTA's candidates begin among all (their numbers are the parts'
  // counts `c`), and how many there are.
  auto begins_of = [&](const uint32_t* c, uint32_t* begin) {
    static_assert(NW == 16 && kParts == 128, "four lanes hold a CTA's parts");
    uint32_t mine = 0, n = 0;
    for (int i = 0; i < 4; ++i) mine += 4 * lane + i < parts ? c[4 * lane + i] : 0;
    mine += __shfl_xor_sync(0xffffffffu, mine, 1);
    mine += __shfl_xor_sync(0xffffffffu, mine, 2);
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) {
      begin[r] = n;
      n += __shfl_sync(0xffffffffu, mine, 4 * r);
    }
    return n;
  };
  auto candidate = [&](const uint32_t* begin, uint32_t i) {  // from the list of the CTA that holds it
    uint32_t from = 0, at = i;
#pragma unroll
    for (int r = 1; r < kMaxCluster; ++r)
      if (r < C && i >= begin[r]) from = r, at = i - begin[r];
    return pull(&s.list[at], from);
  };
  // The first CTA gathers the candidates of all and sorts them.
  auto gather = [&](const uint32_t* c) {
    uint32_t begin[kMaxCluster];
    const uint32_t n = begins_of(c, begin);
    for (uint32_t i = tid; i < n; i += NT) s.all[i] = candidate(begin, i);
    if (tid == 0) s.low = 0;
    cluster_sync();  // (the other CTAs wait here before they touch their lists)
    sort_all(n);
    return n;
  };
  auto weight_at = [&](uint32_t i) { return weight(value_of(~uint32_t(s.all[i] >> 32))); };
  constexpr int EACH = CAP / NT;  // entries of a thread
  // How many of the n sorted tokens are kept, each while the weight before it
  // is short of the target.
  auto kept_of = [&](uint32_t n, double above, double target) {
    double x[EACH], t = 0.0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) t += x[i] = tid * EACH + i < n ? weight_at(tid * EACH + i) : 0.0;
    const double inc = warp_scan(t, lane);
    if (lane == 31) s.scan_w[warp] = inc;
    __syncthreads();
    double before = above;
    for (uint32_t y = 0; y < warp; ++y) before += s.scan_w[y];
    before += inc - t;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      if (tid * EACH + i < n && before < target) atomicMax(&s.low, tid * EACH + i + 1);
      before += x[i];
    }
    __syncthreads();
    return s.low;
  };
  // The draw by one warp, where all kept tokens are among up to 64 candidates:
  // two a lane, sorted in registers, without a barrier (k: top-k's, or n).
  auto draw_few = [&](const uint32_t* c, uint32_t k, double whole) {
    uint32_t begin[kMaxCluster];
    const uint32_t n = begins_of(c, begin);
    uint64_t x[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) x[e] = 2 * lane + e < n ? candidate(begin, 2 * lane + e) : ~0ull;
    cluster_arrive();  // (the lists may go)
#pragma unroll
    for (uint32_t size = 2; size <= 64; size *= 2) {
      const bool up = !(2 * lane & size);
#pragma unroll
      for (uint32_t far = size / 2; far >= 2; far /= 2) {
        const bool least = !(2 * lane & far) == up;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint64_t y = __shfl_xor_sync(0xffffffffu, x[e], far / 2);
          if ((x[e] > y) == least) x[e] = y;
        }
      }
      if ((x[0] > x[1]) == up) {
        const uint64_t y = x[0];
        x[0] = x[1], x[1] = y;
      }
    }
    // kept: the first k, while the weight before is short of top-p's share, above min-p's border
    float z[2];
    double w[2];
    uint32_t at[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      at[e] = uint32_t(x[e]);
      z[e] = value_of(~uint32_t(x[e] >> 32));
      const bool in = 2 * lane + e < min(n, k);
      z[e] = in ? z[e] : -INFINITY;
      w[e] = weight(z[e]);
    }
    const double inc = warp_scan(w[0] + w[1], lane);
    if (by_k) whole = __shfl_sync(0xffffffffu, inc, 31);
    const double target = by_p ? double(top_p) * whole : INFINITY, before = inc - (w[0] + w[1]);
    const bool keep0 = z[0] >= floor_z && z[0] > -INFINITY && before < target;
    const bool keep1 = z[1] >= floor_z && z[1] > -INFINITY && before + w[0] < target;
    const uint32_t set0 = __ballot_sync(0xffffffffu, keep0), set1 = __ballot_sync(0xffffffffu, keep1);
    const uint32_t kept = __popc(set0) + __popc(set1);
    // each kept token's weights up to its own, by index
    double all = 0.0, sum[2] = {};
    for (uint32_t j = 0; j < kept; ++j) {
      const uint32_t other = __shfl_sync(0xffffffffu, j & 1 ? at[1] : at[0], j / 2);
      const double v = __shfl_sync(0xffffffffu, j & 1 ? w[1] : w[0], j / 2);
      all += v;
      if (other <= at[0]) sum[0] += v;
      if (other <= at[1]) sum[1] += v;
    }
    const double goal = fmax(double(u), 0.0) * all;
    uint32_t first = ~0u, last = 0;
    if (keep0) first = sum[0] > goal ? at[0] : ~0u, last = at[0];
    if (keep1) first = sum[1] > goal ? min(first, at[1]) : first, last = max(last, at[1]);
    first = __reduce_min_sync(0xffffffffu, first);
    last = __reduce_max_sync(0xffffffffu, last);
    const uint32_t token = first != ~0u ? first : last;
    if ((keep0 && at[0] == token) || (keep1 && at[1] == token)) {
      const float mine = keep0 && at[0] == token ? z[0] : z[1];
      answer(int64_t(token), int32_t(kept), float((widened(mine) - zm) * cool - log(all)));
    }
    cluster_wait();
  };
  // The draw, where all kept tokens are the first CTA's first n sorted ones or
  // fewer: the ones that top-p and min-p leave, ordered by index.
  auto draw_sorted = [&](uint32_t n, double whole) {
    if (by_p) {
      if (by_k) {
        double x = 0.0;
        for (uint32_t i = tid; i < n; i += NT) x += weight_at(i);
        x = warp_sum(x);
        if (lane == 0) s.scan_w[warp] = x;
        __syncthreads();
        whole = 0.0;
        for (int y = 0; y < NW; ++y) whole += s.scan_w[y];
        __syncthreads();
      }
      n = kept_of(n, 0.0, double(top_p) * whole);
    }
    // min-p leaves a prefix too
    uint32_t keep = 0;
    for (uint32_t i = tid; i < (n + NT - 1) / NT * NT; i += NT)
      keep += __syncthreads_count(i < n && value_of(~uint32_t(s.all[i < n ? i : 0] >> 32)) >= floor_z);
    n = keep;
    for (uint32_t i = tid; i < n; i += NT) s.all[i] = s.all[i] << 32 | s.all[i] >> 32;
    if (tid == 0) s.low = ~0u;
    __syncthreads();  // (of more than NT entries the sort gives a thread others than these)
    sort_all(n);
    // (sort_all's padding is no token)
    double x[EACH], t = 0.0;
    auto z_of = [&](uint32_t i) { return value_of(~uint32_t(s.all[i])); };
#pragma unroll
    for (int i = 0; i < EACH; ++i) t += x[i] = tid * EACH + i < n ? weight(z_of(tid * EACH + i)) : 0.0;
    const double inc = warp_scan(t, lane);
    if (lane == 31) s.scan_w[warp] = inc;
    __syncthreads();
    double before = inc - t, all = 0.0;
    for (uint32_t y = 0; y < NW; ++y) {
      before += y < warp ? s.scan_w[y] : 0.0;
      all += s.scan_w[y];
    }
    const double target = fmax(double(u), 0.0) * all;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      before += x[i];
      if (tid * EACH + i < n && before > target) atomicMin(&s.low, tid * EACH + i);
    }
    __syncthreads();
    if (tid == 0) {
      const uint32_t i = min(s.low, n - 1);
      answer(int64_t(s.all[i] >> 32), int32_t(n), float((widened(z_of(i)) - zm) * cool - log(all)));
    }
  };

  // the tokens that are still in: key above bkey, or bkey with an index up to
  // bidx (at first all above -infinity)
  float nearest = -1.f;  // the distance that few candidates were looked for within,
  double weight_near = 0.0;  // and their weight
  uint32_t bkey = key_of(-INFINITY);
  int32_t bidx = -1;
  bool cut = false;
  auto in = [&](uint32_t k, uint32_t i) { return k > bkey || (k == bkey && int32_t(i) <= bidx); };
  double whole = -1.0;  // all tokens' weight, when known

  // Of this warp's tokens that `has` picks, the one that is number `left` by index.
  auto nth_of = [&](uint32_t left, auto has) {
    uint32_t got = 0;
    for (uint32_t v = wv0 + lane; v - lane < wv1; v += 32) {
      float z[EPV];
      uint32_t mask = 0;
      if (v < wv1) {
        fetch(v, z);
#pragma unroll
        for (int i = 0; i < EPV; ++i) mask |= uint32_t(has(z[i], v * EPV + i - skew)) << i;
      }
      const uint32_t inc = warp_scan(uint32_t(__popc(mask)), lane), ex = inc - __popc(mask);
      const bool here = left > ex && left <= inc;
      if (here) got = v * EPV + __fns(mask, 0, int(left - ex)) - skew;
      const uint32_t who = __ballot_sync(0xffffffffu, here);
      if (who) {
        got = __shfl_sync(0xffffffffu, got, __ffs(who) - 1);
        break;
      }
      left -= __shfl_sync(0xffffffffu, inc, 31);
    }
    return got;
  };
  // The kept tokens, once the border is known; and the draw by the warp whose
  // tokens pass the target, `before` being the weight of the warps before it.
  float border = -INFINITY;
  auto kept = [&](float z, uint32_t i) { return z >= floor_z && (z > border || (z == border && int32_t(i) <= bidx)); };
  auto draw_in = [&](double before, double target, double total, uint32_t many) {
    int32_t token = -1;
    float z_token = 0.f;
    for (uint32_t v = wv0 + lane; v - lane < wv1; v += 32) {
      float z[EPV];
      double e[EPV], t = 0.0;
      if (v < wv1) fetch(v, z);
  #pragma unroll
      for (int i = 0; i < EPV; ++i) {
        e[i] = weight(v < wv1 && kept(z[i], v * EPV + i - skew) ? z[i] : -INFINITY);
        t += e[i];
      }
      const double inc = warp_scan(t, lane);
      // the first lane that passes the target, else the last that keeps any
      const uint32_t some = __ballot_sync(0xffffffffu, t > 0.0);
      const uint32_t past = __ballot_sync(0xffffffffu, t > 0.0 && before + inc > target);
      if (some) {
        const int who = past ? __ffs(past) - 1 : 31 - __clz(some);
        int32_t got = -1;
        float zg = 0.f;
        if (lane == who) {
          double c = before + (inc - t);
          bool done = false;
  #pragma unroll
          for (int i = 0; i < EPV; ++i) {
            c += e[i];
            if (e[i] > 0.0 && !done) got = int32_t(v * EPV + i - skew), zg = z[i], done = c > target;
          }
        }
        token = __shfl_sync(0xffffffffu, got, who);
        z_token = __shfl_sync(0xffffffffu, zg, who);
      }
      if (past) break;
      before += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) answer(token, int32_t(many), float((widened(z_token) - zm) * cool - log(total)));
  };

  // Every warp finds the first of the 256 bins up to which `want` lie; with
  // none, their number.
  auto bin_with = [&](const uint32_t* bins, uint32_t want) {
    uint32_t t = 0, bin = kGuessBins;
    constexpr int PER = kGuessBins / 32;
#pragma unroll
    for (int i = 0; i < PER; ++i) t += bins[lane * PER + i];
    uint32_t run = warp_scan(t, lane) - t;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      run += bins[lane * PER + i];
      if (run >= want && bin == kGuessBins) bin = lane * PER + i;
    }
    return __reduce_min_sync(0xffffffffu, bin);
  };
  // The first CTA: the bins of all CTAs' histograms, four a thread.
  auto all_bins = [&](uint32_t* h) {
    h[0] = h[1] = h[2] = h[3] = 0;
    static_assert(NB / NT == 4, "a vector of bins a thread");
#pragma unroll
    for (uint32_t r = 0; r < kMaxCluster; ++r) {
      if (r >= C) break;
      const uint4 x = pull4(&s.hist[tid * 4], r);
      h[0] += x.x, h[1] += x.y, h[2] += x.z, h[3] += x.w;
    }
  };
  // Inclusive scan over the CTA's threads.
  auto cta_scan = [&](auto x, auto* parts_of) {
    x = warp_scan(x, lane);
    if (lane == 31) parts_of[warp] = x;
    __syncthreads();
    for (uint32_t y = 0; y < warp; ++y) x += parts_of[y];
    return x;
  };
  // Counts a logit by its distance from the largest, less `start`, rounded to
  // bins: those farther than `beyond`, and none behind the last bin.
  float start = 0.f, beyond = -1.f, per_unit = kPerUnit;
  auto count_it = [&](float z) {
    const float d = zmax - z, x = fminf((d - start) * per_unit, NB - 1.f);
    atomicAdd(&s.hist[rounded(d > beyond ? x : NB - 1.f)], 1);  // (without a branch: the last bin takes what does not count)
  };

  // A distance from the largest logit that as many groups' largest lie within as are
  // wanted, or a few more; -1 with none.
  auto near_groups = [&](uint32_t want) {
    if (tid < kGuessBins) s.hist[tid] = 0;
    __syncthreads();
    for (uint32_t i = tid; i < groups; i += NT) {
      const float x = (zmax - s.group[i]) * kGuessPerUnit;
      if (x < float(kGuessBins) - 1.5f) atomicAdd(&s.hist[rounded(x)], 1);
    }
    __syncthreads();
    const uint32_t bin = bin_with(s.hist, want);
    return bin < kGuessBins ? (bin + 0.5f) / kGuessPerUnit : -1.f;  // (a distance of at most that has no later bin)
  };

  // ---- BF16, top-p without top-k: few distinct logits.  Each has a bin that counts its tokens,
  // so that a weight is formed once a bin, not once a token; tokens outside the
  // bins (magnitudes below 16 binades, or above) are weighed one by one.  The bins
  // tell the whole, the border (all tokens above its logit, and of its own the
  // first by index) and each CTA's kept weight; the CTA that the draw falls in
  // weighs its tokens.  Where the border or min-p's bound lies among the tokens
  // outside the bins, the general form below goes on.  One row of 128256, 99000 tokens
  // in the nucleus: 23 us, the general form 41; 256 such rows 197 and 448.  (Without top-p one pass
  // weighs all: 14 us, and 19 by bins.)
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    if (by_p && !by_k) {
      static_assert(sizeof(s.all) == 2 * kSide * sizeof(uint32_t), "the bins lie where candidates are gathered later");
      uint32_t* const bins = reinterpret_cast<uint32_t*>(s.all);  // [sign, magnitude]
      // magnitudes [least, least + kSide): up to 2^6, or to the power of two above the largest logit's
      const uint32_t end = (__float_as_uint(zmax) >> 16 & 0x7f80u) + 0x80u, least = max(kLeast, end - min(end, kSide));
      auto bin_z = [&](uint32_t b) { return __uint_as_float(((b / kSide << 15) | (least + b % kSide)) << 16); };
      const float middle = __uint_as_float(least << 16);  // outside: |z| < middle, and far ones
      const float weighed = __double2float_ru(double(zmax) + kTiny * double(heat)), reach = near_groups(groups / 4);
      for (uint32_t i = tid; i < 2 * kSide; i += NT) bins[i] = 0;
      __syncthreads();
      double w_mid = 0.0, w_far = 0.0, w_near = 0.0;
      uint32_t n_mid = 0, n_far = 0, n_near = 0;
      for (uint32_t v = wv0 + lane; v < wv1; v += 32) {
        const uint4 raw = HELD ? held[v - v0] : read(v);
        const uint32_t word[4] = {raw.x, raw.y, raw.z, raw.w};
        uint32_t outside = 0;
#pragma unroll
        for (int i = 0; i < EPV; ++i) {
          const uint32_t b = i & 1 ? word[i / 2] >> 16 : word[i / 2] & 0xffffu, m = (b & 0x7fffu) - least;
          if (m < kSide)
            atomicAdd(&bins[m + (b >> 15) * kSide], 1);
          else
            outside |= 1u << i;
        }
        auto z_of = [&](uint32_t i) {
          const uint32_t x = i < 4 ? (i < 2 ? raw.x : raw.y) : i < 6 ? raw.z : raw.w;
          return __uint_as_float(i & 1 ? x & 0xffff0000u : x << 16) + 0.f;
        };
        for (; outside; outside &= outside - 1) {
          const float z = z_of(__ffs(outside) - 1);
          if (z < weighed) continue;
          const double e = weight(z);
          if (fabsf(z) < middle)
            w_mid += e, ++n_mid;
          else
            w_far += e, ++n_far;
        }
        if (zmax - E::most(raw) <= reach)
          for (uint32_t i = 0; i < EPV; ++i) {
            const float z = z_of(i);
            if (zmax - z > reach) continue;
            w_near += weight(z), ++n_near;
            list_it(z, v * EPV + i - skew);
          }
      }
      auto share_q = [&](int i, double x) {
        x = warp_sum(x);
        if (lane < C) push(&s.quarter_w[turn][i][me], lane, x);
      };
      share_q(0, w_mid), share_q(1, w_far), share_q(2, w_near);
      share_c(0, n_near), share_c(1, n_far);
      cluster_sync();
      const double mid = sum_of(s.quarter_w[turn][0]), far = sum_of(s.quarter_w[turn][1]);
      const uint32_t near = count_of(s.part_c[turn][0]), fars = count_of(s.part_c[turn][1]);
      const uint32_t listed = turn;
      turn ^= 1;
      // a thread's bins, from the largest logit down: the positive ones, then
      // the negative ones; each counts in all CTAs
      const uint32_t some = 2 * kSide / (C * NT), p0 = (rank * NT + tid) * some;
      auto at = [](uint32_t p) { return p < kSide ? kSide - 1 - p : p; };
      auto all_of = [&](uint32_t b) {
        uint32_t n = 0;
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r)
          if (r < C) n += pull(&bins[b], r);
        return n;
      };
      double t = 0.0;
      for (uint32_t e = 0; e < some; ++e) {
        const uint32_t b = at(p0 + e), n = all_of(b);
        if (n) t += n * weight(bin_z(b));
      }
      share_w(0, t);
      cluster_sync();
      // every warp finds the row's warp whose bins hold the border
      constexpr int PER = kParts / 32;
      double x[PER], sum = 0.0;
#pragma unroll
      for (int i = 0; i < PER; ++i) sum += x[i] = lane * PER + i < parts ? s.part_w[turn][0][lane * PER + i] : 0.0;
      const double inc = warp_scan(sum, lane);
      whole = __shfl_sync(0xffffffffu, inc, 31) + mid + far;
      turn ^= 1;
      const double target = double(top_p) * whole;
      weight_near = sum_of(s.quarter_w[listed][2]);
      if (near && near <= CAP && weight_near >= target * (1.0 + 1e-12)) {  // all that is kept is among the nearest
        if (rank == 0 && near <= 64) {
          if (warp == 0)
            draw_few(s.part_c[listed][0], near, whole);
          else
            cluster_sync();
        } else if (rank == 0) {
          gather(s.part_c[listed][0]);
          draw_sorted(near, whole);
        } else {
          cluster_sync();
        }
        return;
      }
      // (up to the middle as the bins' sums were added: the negative ones' warps are
      // the upper half)
      uint32_t owner = ~0u;
      double run = inc - sum, before = 0.0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const uint32_t part = lane * PER + i;
        const double from = run + (part >= parts / 2 ? mid : 0.0);
        run += x[i];
        if (owner == ~0u && part < parts && x[i] > 0.0 && from + x[i] >= target) owner = part, before = from;
      }
      const uint32_t who = __ballot_sync(0xffffffffu, owner != ~0u);
      // (in vain where the border or min-p's bound lies among the tokens outside the bins)
      bool exact = who != 0 && !(min_p > 0.f && ((mid > 0.0 && fabsf(floor_z) < 2 * middle) || (fars && floor_z <= bin_z(2 * kSide - 1))));
      if (who) {
        owner = __shfl_sync(0xffffffffu, owner, __ffs(who) - 1);
        before = __shfl_sync(0xffffffffu, before, __ffs(who) - 1);
        exact = exact && before < target;
      }
      if (exact) {
        // each CTA finds the border's bin among that warp's, and how many of the
        // border's own tokens, the first by index, are kept of its own
        if (warp == 0) {
          const uint32_t q0 = (owner * 32 + lane) * some;
          t = 0.0;
          for (uint32_t e = 0; e < some; ++e) {
            const uint32_t b = at(q0 + e), n = all_of(b);
            if (n) t += n * weight(bin_z(b));
          }
          const double up = warp_scan(t, lane);
          const uint32_t first = __ballot_sync(0xffffffffu, t > 0.0 && before + up >= target);
          const uint32_t last = __ballot_sync(0xffffffffu, t > 0.0);
          // (by rounding none: the last that has any)
          if (lane == (first ? __ffs(first) - 1 : 31 - __clz(last))) {
            double c = before + (up - t), above = c;
            uint32_t got = 0, ties = 0;
            for (uint32_t e = 0; e < some; ++e) {
              const uint32_t b = at(q0 + e), n = all_of(b);
              if (!n) continue;
              got = b, ties = n, above = c;
              c += n * weight(bin_z(b));
              if (c >= target) break;
            }
            const double need = ceil((target - above) / weight(bin_z(got)));
            uint32_t m = need < 1.0 ? 1u : need > double(ties) ? ties : uint32_t(need);
            for (uint32_t r = 0; r < rank; ++r) m -= min(m, pull(&bins[got], r));
            s.found = got, s.ctl[0] = min(m, bins[got]), s.ctl[1] = bins[got];
          }
        }
        __syncthreads();
        const uint32_t border_bin = s.found, mine = s.ctl[0], ours = s.ctl[1];
        border = bin_z(border_bin);
        bidx = mine == ours ? INT32_MAX : -1;
        const float from = fmaxf(floor_z, border);
        double w = 0.0;
        uint32_t n = 0;
        static_assert(offsetof(Shared, all) == 2 * kSide * sizeof(double), "all that lies ahead of the bins is free by now");
        double* const weights = reinterpret_cast<double*>(s.hist);  // of the bins' tokens that are kept
        for (uint32_t b = tid; b < 2 * kSide; b += NT) {
          const float z = bin_z(b);
          const uint32_t c = z < from ? 0 : b == border_bin ? mine : bins[b];
          const double e = c ? weight(z) : 0.0;
          weights[b] = e;
          n += c, w += c * e;
        }
        if (border < 0.f && floor_z < 0.f) w += w_mid, n += n_mid;  // (those farther away are not kept)
        share_w(0, w);
        share_c(0, n);
        cluster_sync();
        const uint32_t many = count_of(s.part_c[turn][0]);
        // the CTA whose weights pass the draw's target, else the last that keeps any
        double x = 0.0;
        if (lane < C)
          for (int y = 0; y < NW; ++y) x += s.part_w[turn][0][lane * NW + y];
        const double inc = warp_scan(x, lane), total = __shfl_sync(0xffffffffu, inc, 31), goal = fmax(double(u), 0.0) * total;
        const uint32_t past = __ballot_sync(0xffffffffu, x > 0.0 && inc > goal), any = __ballot_sync(0xffffffffu, x > 0.0);
        const uint32_t cta = past ? __ffs(past) - 1 : 31 - __clz(any);
        if (rank != cta) return;
        double before = __shfl_sync(0xffffffffu, inc - x, cta);
        if (mine != ours && mine) {  // the index of the last of the border's
          uint32_t c = 0;
          for (uint32_t v = wv0 + lane; v < wv1; v += 32) {
            float z[EPV];
            fetch(v, z);
#pragma unroll
            for (int i = 0; i < EPV; ++i) c += z[i] == border;
          }
          c = __reduce_add_sync(0xffffffffu, c);
          if (lane == 0) s.scan_c[warp] = c;
          __syncthreads();
          uint32_t run = 0;
          for (uint32_t y = 0; y < warp; ++y) run += s.scan_c[y];
          if (mine > run && mine - run <= c) {
            const uint32_t i = nth_of(mine - run, [&](float z, uint32_t) { return z == border; });
            if (lane == 0) s.found = i;
          }
          __syncthreads();
          bidx = int32_t(s.found);
        }
        w = 0.0;
        for (uint32_t v = wv0 + lane; v < wv1; v += 32) {
          float z[EPV];
          fetch(v, z);
#pragma unroll
          for (int i = 0; i < EPV; ++i) {
            const uint32_t b = __float_as_uint(z[i]) >> 16, m = (b & 0x7fffu) - least;
            if (m < kSide) {
              if (z[i] != border || int32_t(v * EPV + i - skew) <= bidx) w += weights[m + (b >> 15) * kSide];
            } else if (kept(z[i], 0)) {
              w += weight(z[i]);
            }
          }
        }
        w = warp_sum(w);
        if (lane == 0) s.scan_w[warp] = w;
        __syncthreads();
        const double part = lane < NW ? s.scan_w[lane] : 0.0, to = before + warp_scan(part, lane);
        const uint32_t over = __ballot_sync(0xffffffffu, part > 0.0 && to > goal), some = __ballot_sync(0xffffffffu, part > 0.0);
        const uint32_t owner = over ? __ffs(over) - 1 : 31 - __clz(some);
        before = over ? __shfl_sync(0xffffffffu, to - part, owner) : -INFINITY;  // (no token passes: the last one)
        if (warp == owner) draw_in(before, goal, total, many);
        return;
      }
      border = -INFINITY, bidx = -1;
      if (tid == 0) s.listed = 0;
    }

  // ---- few candidates: all tokens within `reach` of the largest logit, guessed so
  // that they are as many as are kept or a few more.  Up to three quarters of
  // the groups, and 1200: `want` groups have a token as near as the farthest of
  // their largest ones.  Above that, from a sample.
  if (by_k ? uint32_t(top_k) <= CAP * 3 / 4 : by_p) {
    float reach = -1.f;
    const uint32_t want = by_k ? uint32_t(top_k) : groups / 4;
    if (want <= min(3 * groups / 4, kGuessMost)) {
      reach = near_groups(want);
    } else {
      for (uint32_t i = tid; i < NB; i += NT) s.hist[i] = 0;
      __syncthreads();
      for (uint32_t v = wv0 + lane, it = lane; v < wv1; v += 32, ++it) {
        if (it % kEvery) continue;
        float z[EPV];
        fetch(v, z);
#pragma unroll
        for (int i = 0; i < EPV; ++i) count_it(z[i]);
      }
      cluster_sync();
      if (rank == 0) {
        uint32_t h[4];
        all_bins(h);
        // four standard deviations more than wanted
        const uint32_t some = uint32_t(ceilf(want / float(kEvery) + 4.f * sqrtf(want / float(kEvery))));
        if (tid == 0) s.low = NB;
        const uint32_t c = h[0] + h[1] + h[2] + h[3];
        uint32_t run = cta_scan(c, s.scan_c) - c;
        for (int i = 0; i < 4; ++i) {
          run += h[i];
          if (run >= some) atomicMin(&s.low, tid * 4 + i);
        }
        __syncthreads();
        if (tid < C) push(&s.ctl[0], tid, s.low);
      }
      cluster_sync();
      if (s.ctl[0] < NB) reach = (s.ctl[0] + 0.5f) / kPerUnit;
    }
    if (reach >= 0.f) {
      double w = 0.0, wl = 0.0;
      uint32_t n = 0;
      for (uint32_t v = wv0 + lane; v < wv1; v += 32) {
        const uint4 raw = HELD ? held[v - v0] : read(v);
        const bool any = zmax - E::most(raw) <= reach;
        if (by_k && !any) continue;
        float z[EPV];
        E::get(raw, z);
        if (!by_k) {
          double e[EPV];
#pragma unroll
          for (int i = 0; i < EPV; ++i) e[i] = weight(z[i]);
#pragma unroll
          for (int i = 0; i < EPV; ++i) {
            w += e[i];
            if (zmax - z[i] <= reach) wl += e[i];
          }
        }
        if (!any) continue;
#pragma unroll
        for (int i = 0; i < EPV; ++i) {
          z[i] += 0.f;
          if (zmax - z[i] <= reach) {
            ++n;
            list_it(z[i], v * EPV + i - skew);
          }
        }
      }
      share_c(0, n);
      if (!by_k) share_w(0, w), share_w(1, wl);
      cluster_sync();
      n = count_of(s.part_c[turn][0]);
      bool enough = n <= CAP && (!by_k || n >= want);
      if (!by_k) {
        whole = sum_of(s.part_w[turn][0]);
        nearest = reach, weight_near = sum_of(s.part_w[turn][1]);
        enough = enough && weight_near >= double(top_p) * whole * (1.0 + 1e-12);
      }
      if (enough) {  // all that is kept is among them
        if (rank == 0 && n <= 64) {
          if (warp == 0)
            draw_few(s.part_c[turn][0], by_k ? want : n, whole);
          else
            cluster_sync();
        } else if (rank == 0) {
          gather(s.part_c[turn][0]);
          draw_sorted(by_k ? want : n, whole);
        } else {
          cluster_sync();
        }
        return;
      }
      turn ^= 1;
      if (tid == 0) s.listed = 0;
    }
  }

  // The border of a prefix: by weight, the shortest whose weight reaches top_p
  // of the whole; else the first top_k tokens.  A histogram says where it lies,
  // exactly for counts and nearly for weights; the tokens there are the
  // candidates, and the weight above them is summed.  `passed`: this lane's weights above
  // the candidates' keys [klo, khi].
  double passed = 0.0;
  uint32_t klo = 0, khi = 0, passed_n = 0;
  bool whole_list = false;  // this CTA's list still holds its candidates
  bool all_in = false;      // `passed` has all that is kept: what lies in [klo, khi] too
  auto select = [&](bool by_weight) {
    const uint32_t k = uint32_t(top_k);
    // Where the guess above was tried the weight of the tokens nearer than `start` is
    // known, and falls short unless they were only too many; behind `end` all V
    // tokens weigh less than the whole leaves.
    const bool tried = by_weight && !cut && whole >= 0.0 && nearest >= 0.f && weight_near < double(top_p) * whole;
    start = 0.f, beyond = -1.f, per_unit = kPerUnit;
    if (tried) {
      const float end = float(log(V / ((1.0 - double(top_p)) * whole)) * double(heat));
      start = beyond = nearest;
      per_unit = fminf(fmaxf((NB - 2) / fmaxf(end - start, 1e-3f), kPerUnit), 4096.f);
    }
    const double known = tried ? weight_near : 0.0;
    for (uint32_t i = tid; i < NB; i += NT) s.hist[i] = 0;
    if (tid == 0) s.listed = 0;
    __syncthreads();
    const bool weigh = by_weight && (cut || whole < 0.0);
    double w = 0.0;
    for (uint32_t v = wv0 + lane; v < wv1; v += 32) {
      float z[EPV];
      fetch(v, z);
#pragma unroll
      for (int i = 0; i < EPV; ++i)
        if (cut && !in(key_of(z[i]), v * EPV + i - skew)) z[i] = -INFINITY;
      if (weigh) {
#pragma unroll
        for (int i = 0; i < EPV; ++i) w += weight(z[i]);
      }
#pragma unroll
      for (int i = 0; i < EPV; ++i) count_it(z[i]);
    }
    if (weigh) share_w(0, w);
    cluster_sync();
    if (weigh) whole = sum_of(s.part_w[turn][0]);
    turn ^= 1;
    const double target = double(top_p) * whole;
    bool have_list = false;  // the list holds the keys [klo, khi]
    uint32_t inside = 0, ahead = 0, listed = 0;  // candidates, tokens above them, the set of their counts
    double above = 0.0, astray = 0.0;            // weight of all keys above khi
    bool hit = false;
    for (int tries = 0; tries < 3; ++tries) {
      if (rank == 0) {
        // bins before which the border cannot lie (counts) or should not (weights:
        // a bin's are taken as those of its middle), and the last it may
        uint32_t h[4];
        all_bins(h);
        if (tid == 0) s.low = NB, s.found = NB;
        if (by_weight) {
          double x[4], t = 0.0;
#pragma unroll
          for (int i = 0; i < 4; ++i) t += x[i] = h[i] ? h[i] * weight(zmax - start - (tid * 4 + i) / per_unit) : 0.0;
          double run = known + (cta_scan(t, s.scan_w) - t);
          // four standard deviations, were the bins' weights off by even chances
          // of up to half a bin
          const float squares = warp_sum(x[0] * x[0] + x[1] * x[1] + x[2] * x[2] + x[3] * x[3]);
          if (lane == 0) s.spread[warp] = squares;
          __syncthreads();
          float spread = 0.f;
          for (int y = 0; y < NW; ++y) spread += s.spread[y];
          const double slack = 4 * 0.2887 * cool / per_unit * sqrtf(spread) + 1e-7 * target, goal = target + astray;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            run += x[i];
            if (run >= goal - slack) atomicMin(&s.low, tid * 4 + i);
            if (run >= goal + slack) atomicMin(&s.found, tid * 4 + i);
          }
          __syncthreads();
          run -= x[0] + x[1] + x[2] + x[3];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (s.low == tid * 4 + i) s.guessed = run;
            run += x[i];
          }
        } else {
          const uint32_t c = h[0] + h[1] + h[2] + h[3];
          uint32_t run = cta_scan(c, s.scan_c) - c;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            run += h[i];
            if (run >= k) atomicMin(&s.low, tid * 4 + i);
            if (run >= k) atomicMin(&s.found, tid * 4 + i);
          }
        }
        __syncthreads();
        if (tid < C) push(&s.ctl[0], tid, s.low), push(&s.ctl[1], tid, s.found);
      }
      cluster_sync();
      // The candidates' distances; with no border among the bins, all there are
      const bool some = s.ctl[0] < NB;
      const float near = some ? start + (s.ctl[0] - 0.5f) / per_unit : -1.f;
      const float far = s.ctl[1] < NB ? start + (s.ctl[1] + 0.5f) / per_unit : INFINITY;
      uint32_t n = 0, lo = ~0u, hi = 0, over = 0;
      double wl = 0.0;
      w = 0.0;
      if (some)
        for (uint32_t v = wv0 + lane; v < wv1; v += 32) {
          const uint4 raw = HELD ? held[v - v0] : read(v);
          if (zmax - E::most(raw) > far) continue;
          float z[EPV];
          E::get(raw, z);
          bool any = false;
          double e[EPV];
#pragma unroll
          for (int i = 0; i < EPV; ++i) {
            z[i] += 0.f;
            if (cut && !in(key_of(z[i]), v * EPV + i - skew)) z[i] = -INFINITY;
            const float d = zmax - z[i];
            any |= d >= near && d <= far;
            over += d < near;
            if (by_weight) e[i] = weight(d < near ? z[i] : -INFINITY);
          }
          if (by_weight) {
#pragma unroll
            for (int i = 0; i < EPV; ++i) w += e[i];
          }
          if (!any) continue;
#pragma unroll
          for (int i = 0; i < EPV; ++i)
            if (zmax - z[i] >= near && zmax - z[i] <= far && z[i] > -INFINITY) {
              const uint32_t kz = key_of(z[i]);
              ++n, lo = min(lo, kz), hi = max(hi, kz);
              if (by_weight) wl += weight(z[i]);
              list_it(z[i], v * EPV + i - skew);
            }
        }
      share_c(0, n);
      share_c(1, over);
      lo = __reduce_min_sync(0xffffffffu, lo), hi = __reduce_max_sync(0xffffffffu, hi);
      if (lane < C) push(&s.part_lo[turn][me], lane, lo), push(&s.part_hi[turn][me], lane, hi);
      if (by_weight) share_w(0, w), share_w(1, wl);
      cluster_sync();
      inside = count_of(s.part_c[turn][0]), ahead = count_of(s.part_c[turn][1]);
      klo = ~0u, khi = 0;
      for (uint32_t i = lane; i < parts; i += 32) klo = min(klo, s.part_lo[turn][i]), khi = max(khi, s.part_hi[turn][i]);
      klo = __reduce_min_sync(0xffffffffu, klo), khi = __reduce_max_sync(0xffffffffu, khi);
      above = by_weight ? sum_of(s.part_w[turn][0]) : 0.0;  // weight of all keys above khi
      hit = inside && (by_weight ? above < target && above + sum_of(s.part_w[turn][1]) >= target : ahead < k && ahead + inside >= k);
      listed = turn;
      turn ^= 1;
      if (hit) {
        passed += w, passed_n += over;
        break;
      }
      // the weight above the candidates is known now, and so how far the bins'
      // sums are out there
      if (!some || !by_weight) break;
      astray = s.guessed - above;  // (of the first CTA)
      if (tid == 0) s.listed = 0;
      __syncthreads();
    }
    bool listing = hit && inside <= CAP && klo != khi, counted = hit && klo == khi;
    if (!hit) {  // the border lies elsewhere: in the whole range
      klo = key_of(-INFINITY) + 1, khi = key_of(zmax), inside = ~0u, ahead = 0, above = 0.0;
      passed = 0.0, passed_n = 0;
    }
    // Few enough candidates are sorted; else a quarter of the keys' range is
    // kept a round (at most 16), down to a single key, of which the first by
    // index are counted off.
    for (;;) {
      uint32_t key = klo;
      int32_t index = INT32_MAX;
      bool found = true;
      if (listing) {
        if (rank == 0) {
          gather(s.part_c[listed][0]);
          const uint32_t keep = by_weight ? kept_of(inside, above, target) : min(k - ahead, inside);
          if (tid < C) {
            // (no candidate, by rounding: all that lies above)
            const uint64_t end = keep ? s.all[keep - 1] : 0;
            push(&s.ctl[0], tid, keep ? ~uint32_t(end >> 32) : khi);
            push(&s.ctl[1], tid, keep ? uint32_t(end) : ~0u);
          }
        } else {
          cluster_sync();
        }
        cluster_sync();
        key = s.ctl[0];
        index = int32_t(s.ctl[1]);
      } else {
        const bool single = klo == khi, have = counted;
        have_list = counted;
        counted = false;
        const int shift = max(0, 32 - __clz(khi - klo) - 2);
        double wq[4] = {};
        uint32_t cq[4] = {};
        listing = inside <= CAP && !single;
        if (!have && tid == 0) s.listed = 0;
        __syncthreads();
        for (uint32_t v = have ? wv1 : wv0 + lane; v < wv1; v += 32) {
          float z[EPV];
          fetch(v, z);
#pragma unroll
          for (int i = 0; i < EPV; ++i) {
            const uint32_t kz = key_of(z[i]), at = v * EPV + i - skew;
            if (kz < klo || kz > khi || (cut && !in(kz, at))) continue;
            if (listing) {
              list_it(z[i], at), ++cq[0];
            } else {
              const uint32_t q = (khi - kz) >> shift;
              const double x = by_weight && !single ? weight(z[i]) : 0.0;
#pragma unroll
              for (uint32_t j = 0; j < 4; ++j)
                if (q == j) ++cq[j], wq[j] += x;
            }
          }
        }
        if (have) {
        } else if (listing || single) {
          share_c(0, cq[0]);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const double x = warp_sum(wq[j]);
            const uint32_t c = __reduce_add_sync(0xffffffffu, cq[j]);
            if (lane < C) push(&s.quarter_w[turn][j][me], lane, x), push(&s.quarter_c[turn][j][me], lane, c);
          }
        }
        if (!have) cluster_sync();
        const uint32_t now = have ? listed : turn;
        if (!have) turn ^= 1;
        if (listing) {
          listed = now;
          continue;
        }
        if (single) {
          // the first `m` by index of the tokens of one key
          uint32_t m = k - ahead;
          if (by_weight) {
            const double need = ceil((target - above) / weight(value_of(khi)));
            m = need < 1.0 ? 1u : need > 4e9 ? ~0u : uint32_t(need);
          }
          // every warp finds the row's warp that holds the m-th
          constexpr int PER = kParts / 32;
          uint32_t c[PER], t = 0, owner = ~0u, before = 0;
#pragma unroll
          for (int i = 0; i < PER; ++i) t += c[i] = lane * PER + i < parts ? s.part_c[now][0][lane * PER + i] : 0;
          uint32_t run = warp_scan(t, lane) - t, mine = 0;
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            if (m > run && m - run <= c[i]) owner = lane * PER + i, before = run;
            if (lane * PER + i == me) mine = m > run ? min(c[i], m - run) : 0;  // of this warp's, that are kept
            run += c[i];
          }
          if (by_weight && mine) passed += mine * weight(value_of(khi)), passed_n += mine;
          all_in = by_weight;
          const uint32_t who = __ballot_sync(0xffffffffu, owner != ~0u);
          if (who) {
            owner = __shfl_sync(0xffffffffu, owner, __ffs(who) - 1);
            before = __shfl_sync(0xffffffffu, before, __ffs(who) - 1);
            if (me == owner) {
              const uint32_t at = nth_of(m - before, [&](float z, uint32_t i) { return key_of(z) == khi && in(khi, i); });
              if (lane < C) push(&s.found, lane, at);
            }
          }
          cluster_sync();
          if (who) index = int32_t(s.found);
        } else {
          double run = above;
          uint32_t count = ahead;
          // (should the quarters together fall short, by the order of their sums: all
          // of them, and `passed` takes them all)
          for (uint32_t j = 0; j < 4; ++j) {
            const uint32_t c = count_of(s.quarter_c[now][j]);
            const double t = sum_of(s.quarter_w[now][j]);
            if (c && (by_weight ? run + t >= target : count + c >= k)) {
              const uint32_t top = khi - (j << shift), step = 1u << shift;
              klo = top - klo >= step ? top - step + 1 : klo;
              khi = top;
              inside = c, ahead = count, above = run;
              found = false;
              break;
            }
            run += t, count += c;
            passed += j == 0 ? wq[0] : j == 1 ? wq[1] : j == 2 ? wq[2] : wq[3];
            passed_n += j == 0 ? cq[0] : j == 1 ? cq[1] : j == 2 ? cq[2] : cq[3];
          }
          all_in = by_weight && found;
        }
      }
      if (found) {
        // (a border that keeps all of a key leaves an earlier one as it is)
        if (key > bkey || (key == bkey && index < bidx)) bkey = key, bidx = index;
        cut = true;
        whole_list = hit && (listing ? inside <= NT : have_list && inside <= CAP);
        return;
      }
    }
  };
  if (by_k) select(false);
  if (by_p) {
    passed = 0.0, passed_n = 0;
    select(true);
  }

  // ---- the kept tokens' weights, and the draw by index.  Where top-p was the
  // last cut and min-p leaves all of them, the weights above its candidates
  // have been summed already.
  border = value_of(bkey);
  const bool summed = by_p && floor_z <= value_of(klo);
  const float upto = summed ? value_of(khi) : INFINITY, from = fmaxf(floor_z, border);
  double w = summed ? passed : 0.0;
  uint32_t n = summed ? passed_n : 0;
  if (summed && all_in) {
  } else if (summed && whole_list) {
    // each warp takes its own of them; their order is not fixed, so they are
    // added as integers
    uint64_t fixed = 0;
    const uint32_t many = s.listed;
    for (uint32_t i = lane; i < many; i += 32) {
      const uint32_t at = uint32_t(s.list[i]), v = (at + skew) / EPV;
      const float z = value_of(~uint32_t(s.list[i] >> 32));
      if (v >= wv0 && v < wv1 && kept(z, at)) fixed += uint64_t(weight(z) * 0x1p52 + 0.5), ++n;
    }
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) fixed += __shfl_xor_sync(0xffffffffu, fixed, d);
    if (lane == 0) w += double(fixed) * 0x1p-52;
  } else for (uint32_t v = wv0 + lane; v < wv1; v += 32) {
    const uint4 raw = HELD ? held[v - v0] : read(v);
    if (E::most(raw) < from) continue;
    float z[EPV];
    E::get(raw, z);
    bool any = false;
#pragma unroll
    for (int i = 0; i < EPV; ++i) {
      z[i] += 0.f;
      const bool now = z[i] <= upto && kept(z[i], v * EPV + i - skew);
      z[i] = now ? z[i] : -INFINITY;
      n += now;
      any |= now;
    }
    if (!any) continue;
    double e[EPV];
#pragma unroll
    for (int i = 0; i < EPV; ++i) e[i] = weight(z[i]);
#pragma unroll
    for (int i = 0; i < EPV; ++i) w += e[i];
  }
  share_w(0, w);
  share_c(0, n);
  cluster_sync();
  const uint32_t many = count_of(s.part_c[turn][0]);
  // every warp finds the row's warp whose weights pass the target; else the
  // last one that keeps any
  constexpr int PER = kParts / 32;
  double x[PER], t = 0.0;
#pragma unroll
  for (int i = 0; i < PER; ++i) t += x[i] = lane * PER + i < parts ? s.part_w[turn][0][lane * PER + i] : 0.0;
  const double inc = warp_scan(t, lane), total = __shfl_sync(0xffffffffu, inc, 31);
  const double target = fmax(double(u), 0.0) * total;
  uint32_t owner = ~0u, last = 0;
  double run = inc - t, before = 0.0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (x[i] > 0.0) {
      last = lane * PER + i + 1;
      if (owner == ~0u && run + x[i] > target) owner = last - 1, before = run;
    }
    run += x[i];
  }
  const uint32_t who = __ballot_sync(0xffffffffu, owner != ~0u);
  last = __reduce_max_sync(0xffffffffu, last) - 1;
  if (who) {
    owner = __shfl_sync(0xffffffffu, owner, __ffs(who) - 1);
    before = __shfl_sync(0xffffffffu, before, __ffs(who) - 1);
  } else {
    owner = last;
    before = -INFINITY;  // (no token of it passes: its last one)
  }
  if (me != owner) return;
  draw_in(before, target, total, many);
}

template <class T>
cudaError_t launch(const SampleArgs& given, int sms, cudaStream_t st) {
  SampleArgs p = given;
  constexpr uint64_t kOver = (sizeof(Shared) + 15) / 16 * 16, kMost = 227 * 1024;
  const uint64_t row = (p.a.vocab + 16 / sizeof(T)) * sizeof(T);  // and its skew
  auto bytes = [&](uint32_t c) { return kOver + (row / 16 / c + 2) * 16; };
  // Where a row, in eight pieces or fewer, leaves an SM room for two CTAs, no
  // fewer pieces than that and up to four CTAs an SM; else two or more, up to eight CTAs an
  // SM, held or not.  Clusters of
  // 1, 2, 4 and 8 CTAs, rows with settings of their own, us: of 32003 BF16 40 rows 60,
  // 42, 37 and 37; 77 59, 42, 42 and 52; 150 70, 58, 63 and 79; 500 99, 92, 118 and
  // 185; of 128256 BF16 77 rows 269, 126, 80 and 72; 300 718, 404, 316 and 259; of
  // 128256 FP32, which do not fit twice, 77 rows 325, 192, 83 and 79; 150 216, 129, 117
  // and 147; 500 311, 220, 303 and 438; 1000 656, 446, 572 and 808; 2000 1011, 771,
  // 1122 and 1621; of 256000 BF16 600 1239, 716, 617 and 767; 2000 1935, 1342, 1760 and 2335.
  const bool twice = bytes(kMaxCluster) <= kMost / 2;
  const uint64_t most = uint64_t(sms) * (twice ? 4 : 8);
  uint32_t c = twice ? 1 : 2;
  while (c < kMaxCluster && (p.a.rows * c * 2 <= most || (twice && bytes(c) > kMost / 2))) c *= 2;
  p.cluster = c;
  const bool holds = bytes(c) <= kMost;
  p.held_off = uint32_t(kOver);
  const uint64_t smem = holds ? bytes(c) : kOver;
  auto kernel = holds ? sample_kernel<T, true> : sample_kernel<T, false>;
  static std::atomic<uint64_t> done[2] = {};
  const cudaError_t e = opt_in_smem(kernel, kMost, done[holds]);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(uint32_t(p.a.rows * c));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = c;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

}  // namespace

cudaError_t launch_sample(const SampleArgs& p, int sms, cudaStream_t st) {
  switch (p.a.type) {
    case XKSV_BF16: return launch<__nv_bfloat16>(p, sms, st);
    case XKSV_FP16: return launch<__half>(p, sms, st);
    default: return launch<float>(p, sms, st);
  }
}

}  // namespace xksv

using namespace xksv;

extern "C" {

int xksv_sample(const xksv_sample_args* a, void* stream) {
  if (!a || a->flags || (a->type != XKSV_BF16 && a->type != XKSV_FP16 && a->type != XKSV_FP32)) return 1;
  const float t = a->temperature_all;
  if (!a->temperature && !(t == 0.f || (t >= kSampleColdest && t <= kSampleHottest))) return 1;
  if ((!a->top_p && a->top_p_all != a->top_p_all) || (!a->min_p && a->min_p_all != a->min_p_all)) return 1;
  if (!a->rows) return 0;
  const uintptr_t e = a->type == XKSV_FP32 ? 4 : 2;
  auto off = [](const void* p, uintptr_t align) { return (reinterpret_cast<uintptr_t>(p) & (align - 1)) != 0; };
  if (!a->logits || !a->u || !a->tokens || !a->vocab || a->vocab > XKSV_SAMPLE_MAX_VOCAB || a->rows > (1u << 24) ||
      a->stride >= (1ull << 40) || off(a->logits, e) || off(a->u, 4) ||
      off(a->tokens, 8) || off(a->kept, 4) || off(a->logprob, 4) || off(a->temperature, 4) || off(a->top_k, 4) ||
      off(a->top_p, 4) || off(a->min_p, 4))
    return 1;
  DeviceGuard guard(int(a->device));
  int sms = 0;
  if (!guard.ok || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, int(a->device)) != cudaSuccess) {
    cudaGetLastError();  // not the next launch's
    return 1;
  }
  return launch_sample(SampleArgs{*a, 0, 0}, sms, static_cast<cudaStream_t>(stream)) == cudaSuccess ? 0 : 1;
}

}  // extern "C"
