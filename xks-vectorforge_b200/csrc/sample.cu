// Sampling of the next token of each row of logits (include/xksv_cuda.h,
// part 9): temperature, top-k, top-p and min-p, drawn with a given number.
//
// Tokens are ordered by logit, equal ones by index; each of the three filters
// keeps a prefix of that order, so a row's kept tokens are those above a
// border: a logit, and among the tokens of that logit an index.  The draw goes
// through the kept tokens by index, so nothing is sorted but the few
// candidates next to the border:
//   * a cluster of CTAs takes a row and holds it in shared memory: the logits
//     are read from HBM once;
//   * a histogram of the distances from the largest logit bounds the border
//     (counts are exact; a bin's weights are known within its width), further
//     histograms over the bits of the border's bins narrow it until the
//     candidates fit a list, which one CTA sorts;
//   * weights exp((z - largest) / temperature) and their sums are FP64: FP32
//     sums of 10^5 weights are off by more than the smaller ones, so that the
//     border and the drawn token would depend on the order of the additions.
//     All sums have a fixed order: the same call gives the same tokens.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "kernels.h"
#include "sample.h"
#include "tcgen05.cuh"

namespace xksv {
namespace {

constexpr int NT = 512;         // threads of a CTA
constexpr int NW = NT / 32;
constexpr int NB = 2048;        // bins of a histogram
constexpr int kBinsPerUnit = 64;  // of the first one: bins per unit of distance (top-k) or exponent (top-p)
constexpr int CAP = 1024;       // candidates that are sorted
constexpr int kMaxCluster = 8;
constexpr double kTiny = -700.0;  // weights below exp(kTiny) count as zero

// What the first CTA tells the others: the border lies among the keys [klo,
// khi], `inside` tokens with `ahead` above them; or it is key klo, index khi.
struct Ctl {
  uint32_t klo, khi, inside, ahead;
};

struct Shared {
  uint32_t hist[NB];
  uint64_t list[CAP], all[CAP], sorted[CAP];
  double sum[NW + 1];      // the warps' weights, and the CTA's
  uint64_t best[NW + 1];   // their largest logits
  double part_w[4][NW + 1], scan_l[NW], scan_u[NW];
  uint32_t part_c[4][NW + 1], scan_c[NW];
  uint32_t count[NW + 1];  // their tokens
  uint32_t listed, low, high, ahead, inside, found;
  Ctl ctl;
};

// Order-preserving integer of a float (no NaN; -0 is +0 by then).
__device__ __forceinline__ uint32_t key_of(float z) {
  const uint32_t b = __float_as_uint(z);
  return b ^ (uint32_t(int32_t(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

template <class T>
struct Elems;  // of a 16-byte vector
template <>
struct Elems<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void get(const uint4& v, float* z) {
    z[0] = __uint_as_float(v.x), z[1] = __uint_as_float(v.y), z[2] = __uint_as_float(v.z), z[3] = __uint_as_float(v.w);
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
};
template <class T>
__device__ __forceinline__ T lowest();  // -infinity: no weight
template <>
__device__ __forceinline__ float lowest<float>() { return -INFINITY; }
template <>
__device__ __forceinline__ __nv_bfloat16 lowest<__nv_bfloat16>() { return __ushort_as_bfloat16(0xff80); }
template <>
__device__ __forceinline__ __half lowest<__half>() { return __ushort_as_half(0xfc00); }

// Reads of another CTA's shared memory at this address.
__device__ __forceinline__ uint32_t at_rank(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(smem_addr(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ uint32_t remote(const uint32_t* p, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];\n" : "=r"(v) : "r"(at_rank(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ uint64_t remote(const uint64_t* p, uint32_t rank) {
  uint64_t v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];\n" : "=l"(v) : "r"(at_rank(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ double remote(const double* p, uint32_t rank) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];\n" : "=d"(v) : "r"(at_rank(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
  return x;
}

template <class T>
__global__ void __launch_bounds__(NT, 2) sample_kernel(const SampleArgs p) {
  using E = Elems<T>;
  constexpr int EPV = E::N;
  extern __shared__ __align__(16) uint8_t dyn[];
  Shared& s = *reinterpret_cast<Shared*>(dyn);
  uint4* const held = reinterpret_cast<uint4*>(dyn + p.held_off);
  const uint32_t C = p.cluster, rank = blockIdx.x % C;
  const uint64_t row = blockIdx.x / C;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t V = uint32_t(p.a.vocab);

  // this row's settings
  float heat = p.a.temperature ? p.a.temperature[row] : p.a.temperature_all;
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
  auto read = [&](uint32_t v) {
    if (v != 0 && v + 1 != nv) return __ldg(vecs + v);
    uint4 w;
    T* e = reinterpret_cast<T*>(&w);
    for (int i = 0; i < EPV; ++i) {
      const uint32_t at = v * EPV + i;
      e[i] = at >= skew && at - skew < V ? src[at - skew] : lowest<T>();
    }
    return w;
  };
  const bool resident = p.resident;
  auto fetch = [&](uint32_t v, float* z) {
    E::get(resident ? held[v - v0] : read(v), z);
#pragma unroll
    for (int i = 0; i < EPV; ++i) z[i] += 0.f;  // -0 becomes +0
  };

  // ---- the largest logit and its first index; NaN among them ----
  uint64_t best = 0;
  bool nan = false;
  for (uint32_t v = wv0 + lane; v < wv1; v += 32) {
    const uint4 w = read(v);
    if (resident) held[v - v0] = w;
    float z[EPV];
    E::get(w, z);
#pragma unroll
    for (int i = 0; i < EPV; ++i) {
      z[i] += 0.f;
      nan |= z[i] != z[i];
      const uint64_t me = uint64_t(key_of(z[i])) << 32 | ~(v * EPV + i - skew);
      best = me > best ? me : best;
    }
  }
  if (nan) best = ~0ull;
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) {
    const uint64_t o = __shfl_xor_sync(0xffffffffu, best, d);
    best = o > best ? o : best;
  }
  if (lane == 0) s.best[warp] = best;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < NW; ++w) best = s.best[w] > best ? s.best[w] : best;
    s.best[NW] = best;
  }
  cluster_sync();
  best = 0;
  for (uint32_t r = 0; r < C; ++r) {
    const uint64_t o = remote(&s.best[NW], r);
    best = o > best ? o : best;
  }
  const float zmax = value_of(uint32_t(best >> 32));
  const uint32_t first = ~uint32_t(best);

  auto answer = [&](int64_t token, int32_t kept, float logprob) {
    p.a.tokens[row] = token;
    if (p.a.kept) p.a.kept[row] = kept;
    if (p.a.logprob) p.a.logprob[row] = logprob;
  };
  // NaN's key is above infinity's; a largest of +-infinity has no distribution
  const bool bad = !sane || !(fabsf(zmax) < INFINITY);
  if (bad || heat == 0.f || top_k == 1 || top_p <= 0.f) {
    if (rank == 0 && tid == 0) answer(bad ? -1 : int64_t(first), bad ? 0 : 1, bad ? NAN : 0.f);
    cluster_sync();  // nobody's shared memory ends while it is read
    return;
  }
  const double zm = zmax, cool = 1.0 / double(heat);
  auto weight = [&](float z) { return exp((double(z) - zm) * cool); };
  // the least logit that min-p and the smallest weight leave
  const double lowest_x = min_p > 0.f ? fmax(kTiny, log(fmin(1.0, double(min_p)))) : kTiny;
  const float floor_z = __double2float_ru(zm + lowest_x * double(heat));

  // the tokens that are still in: key above bkey, or bkey with an index up to
  // bidx (at first all above -infinity)
  uint32_t bkey = key_of(-INFINITY);
  int32_t bidx = -1;
  auto in = [&](uint32_t k, uint32_t i) { return k > bkey || (k == bkey && int32_t(i) <= bidx); };

  // The lanes' weights and counts summed into s.sum[NW] and s.count[NW].
  auto cta_sums = [&](double w, uint32_t c) {
    w = warp_sum(w);
    c = __reduce_add_sync(0xffffffffu, c);
    if (lane == 0) s.sum[warp] = w, s.count[warp] = c;
    __syncthreads();
    if (tid == 0) {
      double t = 0.0;
      uint32_t n = 0;
      for (int i = 0; i < NW; ++i) t += s.sum[i], n += s.count[i];
      s.sum[NW] = t, s.count[NW] = n;
    }
  };
  auto cluster_weight = [&]() {
    double t = 0.0;
    for (uint32_t r = 0; r < C; ++r) t += remote(&s.sum[NW], r);
    return t;
  };

  // The border of a prefix: by_weight, the shortest whose weight reaches share
  // of the whole; else the first `k` tokens.
  auto select = [&](bool by_weight, uint32_t k, double share) {
    const float bins = by_weight ? float(kBinsPerUnit * cool) : float(kBinsPerUnit);
    // rounded distance in bins; the last bin is for all beyond and not counted
    auto bin_of = [&](float z) {
      const float x = (zmax - z) * bins;
      return x < float(NB - 1) ? __float2uint_rn(x) : uint32_t(NB - 1);
    };
    for (uint32_t i = tid; i < NB; i += NT) s.hist[i] = 0;
    if (tid == 0) s.listed = 0;
    __syncthreads();
    double w = 0.0;
    for (uint32_t v = wv0 + lane; v < wv1; v += 32) {
      float z[EPV];
      fetch(v, z);
#pragma unroll
      for (int i = 0; i < EPV; ++i) {
        if (!in(key_of(z[i]), v * EPV + i - skew)) continue;
        const uint32_t b = bin_of(z[i]);
        if (b < NB - 1) atomicAdd(&s.hist[b], 1);
        if (by_weight) w += weight(z[i]);
      }
    }
    cta_sums(w, 0);
    cluster_sync();
    const double whole = by_weight ? cluster_weight() : 0.0, target = share * whole;
    if (rank == 0) {
      // The bins of all CTAs, four a thread.  The border's bin: counts are
      // exact; a bin's weights lie between those of its edges (and the FP32
      // distance's slack), so that the border lies between the first bin up to
      // whose end they may reach the target and the first where they must.
      constexpr int PER = NB / NT;
      uint32_t h[PER], c = 0;
      double wl[PER], wu[PER], tl = 0.0, tu = 0.0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const uint32_t b = tid * PER + i;
        h[i] = 0;
        for (uint32_t r = 0; r < C; ++r) h[i] += remote(&s.hist[b], r);
        wl[i] = by_weight && h[i] ? h[i] * exp(-(b + 0.5) / kBinsPerUnit) * (1.0 - 1e-4) : 0.0;
        wu[i] = by_weight && h[i] ? h[i] * exp(-(b - 0.5) / kBinsPerUnit) * (1.0 + 1e-4) : 0.0;
        c += h[i], tl += wl[i], tu += wu[i];
      }
      uint32_t ic = c;
      double il = tl, iu = tu;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const uint32_t oc = __shfl_up_sync(0xffffffffu, ic, d);
        const double ol = __shfl_up_sync(0xffffffffu, il, d), ou = __shfl_up_sync(0xffffffffu, iu, d);
        if (lane >= d) ic += oc, il += ol, iu += ou;
      }
      if (tid == 0) s.low = s.high = NB - 1, s.ahead = s.inside = 0;
      if (lane == 31) s.scan_c[warp] = ic, s.scan_l[warp] = il, s.scan_u[warp] = iu;
      __syncthreads();
      ic -= c, il -= tl, iu -= tu;
      for (uint32_t x = 0; x < warp; ++x) ic += s.scan_c[x], il += s.scan_l[x], iu += s.scan_u[x];
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const uint32_t b = tid * PER + i;
        ic += h[i], il += wl[i], iu += wu[i];
        if (b < NB - 1 && (by_weight ? iu >= target : ic >= k)) atomicMin(&s.low, b);
        if (b < NB - 1 && (by_weight ? il >= target : ic >= k)) atomicMin(&s.high, b);
      }
      __syncthreads();
      const uint32_t lo = s.low, hi = s.high;
      uint32_t before = 0, within = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const uint32_t b = tid * PER + i;
        before += b < lo ? h[i] : 0;
        within += b >= lo && b <= hi ? h[i] : 0;
      }
      before = __reduce_add_sync(0xffffffffu, before);
      within = __reduce_add_sync(0xffffffffu, within);
      if (lane == 0) atomicAdd(&s.ahead, before), atomicAdd(&s.inside, within);
      __syncthreads();
      if (warp == 0) {
        // the bins' keys.  Bins fall as keys rise: the largest key whose bin is
        // at least b, five bits of it a step
        auto last_of = [&](uint32_t b) {
          uint32_t at = 0;
          for (int sh = 27; sh >= -3; sh -= 5) {
            const uint32_t c = at + (sh >= 0 ? lane << sh : lane >> -sh);
            const bool ok = c <= key_of(-INFINITY) || (c <= key_of(zmax) && bin_of(value_of(c)) >= b);
            at = __shfl_sync(0xffffffffu, c, 31 - __clz(__ballot_sync(0xffffffffu, ok)));
          }
          return at;
        };
        const uint32_t top = lo == 0 ? key_of(zmax) : last_of(lo);
        const uint32_t end = hi >= NB - 1 ? key_of(-INFINITY) : last_of(hi + 1);
        if (lane == 0) {
          // (the last bin's tokens have not been counted)
          s.ctl = Ctl{end + 1, top, hi >= NB - 1 ? ~0u : s.inside, s.ahead};
        }
      }
    }
    cluster_sync();
    uint32_t klo = remote(&s.ctl.klo, 0), khi = remote(&s.ctl.khi, 0);
    uint32_t inside = remote(&s.ctl.inside, 0), ahead = remote(&s.ctl.ahead, 0);
    uint32_t prev = ~0u;  // keys above it are in `above`
    double above = 0.0;
    // The candidates, keys [klo, khi]: few enough are sorted; else a quarter of
    // the keys' range is kept a round (at most 16), down to a single key, of
    // which the first by index are counted off.
    for (;;) {
      const bool listing = inside <= CAP, single = !listing && klo == khi;
      const int shift = max(0, 32 - __clz(khi - klo) - 2);
      if (tid == 0) s.listed = 0;
      __syncthreads();
      double w = 0.0, wq[4] = {};
      uint32_t cq[4] = {};
      for (uint32_t v = wv0 + lane; v < wv1; v += 32) {
        float z[EPV];
        fetch(v, z);
#pragma unroll
        for (int i = 0; i < EPV; ++i) {
          const uint32_t kz = key_of(z[i]), at = v * EPV + i - skew;
          if (kz < klo || !in(kz, at)) continue;
          if (kz > khi) {
            if (by_weight && kz <= prev) w += weight(z[i]);
          } else if (listing) {
            const uint32_t n = atomicAdd(&s.listed, 1);
            if (n < CAP) s.list[n] = uint64_t(~kz) << 32 | at;
          } else {
            const uint32_t q = (khi - kz) >> shift;
            const double x = by_weight && !single ? weight(z[i]) : 0.0;
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j)
              if (q == j) ++cq[j], wq[j] += x;
          }
        }
      }
      if (!listing && !single) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          wq[j] = warp_sum(wq[j]);
          cq[j] = __reduce_add_sync(0xffffffffu, cq[j]);
          if (lane == 0) s.part_w[j][warp] = wq[j], s.part_c[j][warp] = cq[j];
        }
      }
      cta_sums(w, cq[0]);
      if (!listing && !single && tid < 4) {
        double t = 0.0;
        uint32_t n = 0;
        for (int i = 0; i < NW; ++i) t += s.part_w[tid][i], n += s.part_c[tid][i];
        s.part_w[tid][NW] = t, s.part_c[tid][NW] = n;
      }
      cluster_sync();
      if (by_weight) above += cluster_weight();
      prev = khi;
      uint32_t key = klo;
      int32_t index = INT32_MAX;
      bool found = true;
      if (listing) {
        if (rank == 0) {
          // the candidates of all CTAs, in order
          uint32_t n = 0;
          for (uint32_t r = 0; r < C; ++r) {
            const uint32_t m = min(remote(&s.listed, r), CAP - n);
            for (uint32_t i = tid; i < m; i += NT) s.all[n + i] = remote(&s.list[i], r);
            n += m;
          }
          __syncthreads();
          for (uint32_t i = tid; i < n; i += NT) {
            const uint64_t me = s.all[i];
            uint32_t below = 0;
            for (uint32_t j = 0; j < n; ++j) below += s.all[j] < me;
            s.sorted[below] = me;
          }
          if (tid == 0) s.low = by_weight ? 0 : k - ahead;
          __syncthreads();
          if (by_weight) {  // kept while the weight before is short of the target
            constexpr int PER = CAP / NT;
            double x[PER], t = 0.0;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
              const uint32_t j = tid * PER + i;
              x[i] = j < n ? weight(value_of(~uint32_t(s.sorted[j] >> 32))) : 0.0;
              t += x[i];
            }
            double inc = t;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
              const double o = __shfl_up_sync(0xffffffffu, inc, d);
              if (lane >= d) inc += o;
            }
            if (lane == 31) s.scan_l[warp] = inc;
            __syncthreads();
            double before = above + (inc - t);
            for (uint32_t y = 0; y < warp; ++y) before += s.scan_l[y];
#pragma unroll
            for (int i = 0; i < PER; ++i) {
              if (tid * PER + i < n && before < target) atomicMax(&s.low, tid * PER + i + 1);
              before += x[i];
            }
            __syncthreads();
          }
          if (tid == 0) {
            // (no candidate, by rounding: all that lies above)
            const uint32_t keep = min(s.low, n);
            const uint64_t end = keep ? s.sorted[keep - 1] : 0;
            s.ctl = Ctl{keep ? ~uint32_t(end >> 32) : khi, keep ? uint32_t(end) : ~0u, 0, 0};
          }
        }
        cluster_sync();
        key = remote(&s.ctl.klo, 0);
        index = int32_t(remote(&s.ctl.khi, 0));
      } else if (single) {
        // the first `m` by index of the tokens of one key
        uint32_t m = k - ahead, before = 0, owner = 0, n;
        if (by_weight) {
          const double need = ceil((target - above) / weight(value_of(khi)));
          m = need < 1.0 ? 1u : need > 4e9 ? ~0u : uint32_t(need);
        }
        while (owner < C && m > before + (n = remote(&s.count[NW], owner))) before += n, ++owner;
        if (rank == owner) {
          uint32_t left = m - before, x = 0;
          while (left > s.count[x]) left -= s.count[x++];
          if (warp == x) {
            for (uint32_t v = wv0 + lane; v - lane < wv1; v += 32) {
              float z[EPV];
              uint32_t mine = 0;
              if (v < wv1) {
                fetch(v, z);
#pragma unroll
                for (int i = 0; i < EPV; ++i)
                  mine |= uint32_t(key_of(z[i]) == khi && in(khi, v * EPV + i - skew)) << i;
              }
              uint32_t inc = __popc(mine);
#pragma unroll
              for (int d = 1; d < 32; d <<= 1) {
                const uint32_t o = __shfl_up_sync(0xffffffffu, inc, d);
                if (lane >= d) inc += o;
              }
              const uint32_t ex = inc - __popc(mine);
              if (left > ex && left <= inc) s.found = v * EPV + __fns(mine, 0, int(left - ex)) - skew;
              const uint32_t got = __shfl_sync(0xffffffffu, inc, 31);
              if (left <= got) break;
              left -= got;
            }
          }
        }
        cluster_sync();
        if (owner < C) index = int32_t(remote(&s.found, owner));
      } else {
        double run = above;
        uint32_t count = ahead;
        found = true;  // the quarters together fall short: all of them
        for (uint32_t j = 0; j < 4; ++j) {
          uint32_t n = 0;
          double t = 0.0;
          for (uint32_t r = 0; r < C; ++r) n += remote(&s.part_c[j][NW], r), t += remote(&s.part_w[j][NW], r);
          if (n && (by_weight ? run + t >= target : count + n >= k)) {
            const uint32_t top = khi - (j << shift), step = 1u << shift;
            klo = top - klo >= step ? top - step + 1 : klo;
            khi = prev = top;
            inside = n, ahead = count, above = run;
            found = false;
            break;
          }
          run += t, count += n;
        }
      }
      // the next round's writes wait for these reads
      cluster_sync();
      if (found) {
        // (a border that keeps all of a key leaves an earlier one as it is)
        if (key > bkey || (key == bkey && index < bidx)) bkey = key, bidx = index;
        return;
      }
    }
  };
  if (top_k > 0 && uint32_t(top_k) < V) select(false, uint32_t(top_k), 0.0);
  if (top_p < 1.f) select(true, 0, double(top_p));

  // ---- the kept tokens' weights, and the draw by index ----
  const float border = value_of(bkey);
  auto kept = [&](float z, uint32_t i) { return z >= floor_z && (z > border || (z == border && int32_t(i) <= bidx)); };
  double w = 0.0;
  uint32_t n = 0;
  for (uint32_t v = wv0 + lane; v < wv1; v += 32) {
    float z[EPV];
    fetch(v, z);
#pragma unroll
    for (int i = 0; i < EPV; ++i)
      if (kept(z[i], v * EPV + i - skew)) w += weight(z[i]), ++n;
  }
  cta_sums(w, n);
  cluster_sync();
  double total = 0.0, before = 0.0;
  uint32_t many = 0, last = 0;
  for (uint32_t r = 0; r < C; ++r) {
    const uint32_t c = remote(&s.count[NW], r);
    many += c;
    if (c) last = r;
    total += remote(&s.sum[NW], r);
  }
  const double target = fmax(double(u), 0.0) * total;
  // the CTA whose weights pass the target; else the last one that keeps any
  uint32_t owner = last;
  double run = 0.0;
  for (uint32_t r = 0; r < C; ++r) {
    const double next = run + remote(&s.sum[NW], r);
    if (next > target) {
      owner = r;
      break;
    }
    if (r < last) run = next;
  }
  before = run;
  if (rank == owner) {
    uint32_t x = 0, last_warp = 0;
    for (int i = 0; i < NW; ++i)
      if (s.count[i]) last_warp = i;
    while (x < last_warp && !(before + s.sum[x] > target)) before += s.sum[x++];
    if (warp == x) {
      int32_t token = -1;
      float z_token = 0.f;
      for (uint32_t v = wv0 + lane; v - lane < wv1 ; v += 32) {
        float z[EPV];
        double e[EPV], t = 0.0;
        if (v < wv1) fetch(v, z);
#pragma unroll
        for (int i = 0; i < EPV; ++i) {
          e[i] = v < wv1 && kept(z[i], v * EPV + i - skew) ? weight(z[i]) : 0.0;
          t += e[i];
        }
        double inc = t;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const double o = __shfl_up_sync(0xffffffffu, inc, d);
          if (lane >= d) inc += o;
        }
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
      if (lane == 0) answer(token, int32_t(many), float((double(z_token) - zm) * cool - log(total)));
    }
  }
  cluster_sync();
}

template <class T>
cudaError_t launch(const SampleArgs& given, int sms, cudaStream_t st) {
  SampleArgs p = given;
  constexpr uint64_t kOver = (sizeof(Shared) + 15) / 16 * 16, kMost = 227 * 1024;
  const uint64_t row = (p.a.vocab + 16 / sizeof(T)) * sizeof(T);  // and its skew
  auto bytes = [&](uint32_t c) { return kOver + (row / 16 / c + 2) * 16; };
  // few rows: as many CTAs a row as the GPU has; many rows: as many as let two
  // CTAs share an SM
  uint32_t c = 1;
  while (c < kMaxCluster && (p.a.rows * c * 2 <= uint64_t(sms) || bytes(c) > kMost / 2)) c *= 2;
  p.cluster = c;
  p.resident = bytes(c) <= kMost;
  p.held_off = uint32_t(kOver);
  const uint64_t smem = p.resident ? bytes(c) : kOver;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = opt_in_smem(sample_kernel<T>, kMost, done);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(uint32_t(p.a.rows * c));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = c;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sample_kernel<T>, p);
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
  return launch_sample(SampleArgs{*a, 0, 0, 0}, sms, static_cast<cudaStream_t>(stream)) == cudaSuccess ? 0 : 1;
}

}  // extern "C"
