// Append to a paged cache of 8-bit elements with a scale for each block of
// tokens and head (include/xksv_cuda.h, part 8).
//
// A run is what one call adds to one block: tokens of a sequence that stand
// next to each other.  A CTA takes whole runs (and a share of the heads, where
// there are few): it needs a head's largest element of the run before it can
// store the first, so it goes over the run's keys and values twice, the second time
// from L1.  Scales are powers of two: a raised scale costs an earlier
// element at most the bits that fall below its new least one, and an E4M3
// element none but near zero.
#include <algorithm>

#include "kernels.h"
#include "kv_cache.h"
#include "kv_elements.cuh"
#include "kv_index.h"
#include "xksv_types.h"

namespace xksv {
namespace {

constexpr int BTH = 128;        // threads of a CTA
constexpr uint32_t kTile = 16;  // tokens whose angles lie in shared memory at a time
constexpr uint32_t kHeads = 64; // KV heads of a CTA at most

struct I8 {
  int8_t b;
};
__device__ __forceinline__ uint32_t pack4(const float* x) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // rounded by the adder, to even (NaN: zero)
    const float y = x[i] == x[i] ? fminf(fmaxf(x[i], -127.f), 127.f) : 0.f;
    w |= (__float_as_uint(y + 12582912.f) & 0xffu) << (8 * i);
  }
  return w;
}
__device__ __forceinline__ void gather(const float* x, Eight<I8>& a) {
  a.w[0] = pack4(x);
  a.w[1] = pack4(x + 4);
}
__device__ __forceinline__ void spread(const Eight<I8>& a, float* x) {
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = float(int8_t(a.w[i / 4] >> (8 * (i % 4))));
}
__device__ __forceinline__ void spread(const Eight<E4m3>& a, float* x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(a.w[i / 2] >> (16 * (i % 2))), __NV_E4M3);
    const float2 f = __half22float2(__half2(h));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <class TC>
struct Top;
template <>
struct Top<E4m3> {
  static constexpr bool kInt = false;
};
template <>
struct Top<I8> {
  static constexpr bool kInt = true;
};

// PIECES: rows of 16-byte pieces, rotated pairs that fill them; else any strides,
// alignment and rotation, element by element.
template <class TI, class TC, bool PIECES>
__global__ void __launch_bounds__(BTH, 8) kv_append_blocks_kernel(const AppendBlocksArgs p) {
  extern __shared__ float trig[];  // cos [kTile][pairs], then sin
  __shared__ uint32_t need[2][kHeads];
  __shared__ float scale[2][kHeads], ratio[2][kHeads];
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  const xksv_kv_append_args& a = p.a;
  const uint32_t tid = threadIdx.x, lane = tid & 31;
  const uint32_t D = p.c.head_dim, rot = a.rot_dim, pairs = rot / 2, B = uint32_t(p.b.block), P = uint32_t(p.c.page_size);
  const bool inter = a.flags & XKSV_KV_INTERLEAVED;
  const uint32_t nq = a.q ? a.q_heads : 0;
  // this CTA's heads and query rows
  const uint32_t y = blockIdx.y, ys = gridDim.y;
  const uint32_t h0 = uint32_t(uint64_t(p.c.kv_heads) * y / ys), hn = uint32_t(uint64_t(p.c.kv_heads) * (y + 1) / ys) - h0;
  const uint32_t q0 = uint32_t(uint64_t(nq) * y / ys), qn = uint32_t(uint64_t(nq) * (y + 1) / ys) - q0;
  // a thread's piece of a row and its first row
  const uint32_t vper = D / 8, step = BTH / vper, d0 = 8 * (tid % vper), row0 = tid / vper < step ? tid / vper : ~0u;
  float *const cs = trig, *const sn = trig + kTile * pairs;

  auto seq_of = [&](uint64_t t) { return a.seq ? int64_t(a.seq[t]) : int64_t(t); };
  const uint64_t t0 = uint64_t(blockIdx.x) * p.chunk, t1 = min(a.tokens, t0 + p.chunk);
  // the runs that begin among this CTA's tokens
  bool begins = false;
  if (t0 + lane < t1) {
    const uint64_t t = t0 + lane;
    begins = seq_of(t) >= 0 && a.index[t] >= 0 && !kv_follows(a.seq, a.index, t, B);
  }
  for (uint32_t starts = __ballot_sync(0xffffffffu, begins); starts; starts &= starts - 1) {
    const uint64_t t = t0 + __ffs(starts) - 1;
    const int64_t seq = seq_of(t);
    const int32_t index = a.index[t];
    const uint32_t in = uint32_t(index) % B;  // first new place of the block
    uint32_t len = 1;
    for (uint32_t more = ~0u; a.seq && more == ~0u; len += more == ~0u ? 32 : __ffs(~more) - 1) {
      const uint64_t o = t + len + lane;
      more = __ballot_sync(0xffffffffu, o < a.tokens && kv_follows(a.seq, a.index, o, B));
    }
    const KvPlace at = kv_place(a.table, a.table_rows, a.table_cols, a.table_stride, p.c.pages, P, seq, index);
    if (y == 0) {
      bool wrong = at.page < 0 && tid == 0;
      if (a.seq && t > 0) {
        // a sequence's tokens stand together and rise by one
        if (int64_t(a.seq[t - 1]) == seq) {
          wrong |= int64_t(a.index[t - 1]) + 1 != index;
        } else {
          for (uint64_t o = tid; o + 1 < t; o += BTH) wrong |= int64_t(a.seq[o]) == seq;
        }
      }
      if (wrong) atomicOr(p.status, kStatusHeader);
    }
    if (at.page < 0) continue;

    auto tile_angles = [&](uint32_t i0, uint32_t n) {
      for (uint32_t i = tid; i < n * pairs; i += BTH) {
        const uint32_t k = i / pairs, f = i - k * pairs;
        const uint64_t o = t + i0 + k;
        angle_of(a.positions ? a.positions[o] : index + int32_t(i0 + k), a.inv_freq[f], a.rot_scale, &cs[i], &sn[i]);
      }
    };
    // eight elements of a row, rotated by the angles of the tile's token k
    auto rotated = [&](const TI* row, uint32_t k, float* x) {
      const float *c = cs + k * pairs, *s = sn + k * pairs;
      if (PIECES) {
        spread(*reinterpret_cast<const Eight<TI>*>(row + d0), x);
        if (d0 >= rot) return;
        if (inter) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float u = x[2 * e], w = x[2 * e + 1], co = c[d0 / 2 + e], si = s[d0 / 2 + e];
            x[2 * e] = u * co - w * si;
            x[2 * e + 1] = w * co + u * si;
          }
        } else {
          const bool low = d0 < pairs;
          const uint32_t f = low ? d0 : d0 - pairs;
          float o[8];
          spread(*reinterpret_cast<const Eight<TI>*>(row + (low ? d0 + pairs : f)), o);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float co = c[f + e], si = low ? -s[f + e] : s[f + e];
            x[e] = x[e] * co + o[e] * si;
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t d = d0 + e;
          x[e] = to_float(row[d]);
          if (d >= rot) continue;
          const uint32_t f = inter ? d / 2 : d % pairs;
          const bool low = inter ? !(d & 1) : d < pairs;
          const float o = to_float(row[inter ? d ^ 1 : low ? d + pairs : f]);
          x[e] = x[e] * c[f] + o * (low ? -s[f] : s[f]);
        }
      }
    };
    auto plain = [&](const TI* row, float* x) {
      if (PIECES) {
        spread(*reinterpret_cast<const Eight<TI>*>(row + d0), x);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = to_float(row[d0 + e]);
      }
    };
    auto key_row = [&](uint32_t i, uint32_t h) { return static_cast<const TI*>(a.k) + (t + i) * a.k_stride[0] + h * a.k_stride[1]; };
    auto value_row = [&](uint32_t i, uint32_t h) { return static_cast<const TI*>(a.v) + (t + i) * a.v_stride[0] + h * a.v_stride[1]; };

    // ---- the heads' largest elements ----
    __syncthreads();  // (the former run's)
    for (uint32_t i = tid; i < 2 * hn; i += BTH) need[i / hn][i % hn] = 0;
    for (uint32_t i0 = 0; i0 < len; i0 += kTile) {
      const uint32_t n = min(kTile, len - i0);
      __syncthreads();
      tile_angles(i0, n);
      __syncthreads();
      for (uint32_t r = row0; r < 2 * hn; r += step) {
        const bool key = r < hn;
        const uint32_t h = key ? r : r - hn;
        float high = 0.f;
        bool nan = false;
        for (uint32_t i = 0; i < n; ++i) {
          float x[8];
          if (key)
            rotated(key_row(i0 + i, h0 + h), i, x);
          else
            plain(value_row(i0 + i, h0 + h), x);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float m = fabsf(x[e]);
            nan |= m != m;
            high = m < INFINITY ? fmaxf(high, m) : high;  // an infinite one saturates
          }
        }
        atomicMax(&need[!key][h], __float_as_uint(high));
        if (Top<TC>::kInt && nan) atomicOr(p.status, kStatusHeader);  // (an integer holds none)
      }
    }
    __syncthreads();
    // ---- the scales ----
    const uint32_t block = at.place / B;
    for (uint32_t i = tid; i < 2 * hn; i += BTH) {
      const bool key = i < hn;
      const uint32_t h = key ? i : i - hn;
      const uint64_t* st = key ? p.b.k_stride : p.b.v_stride;
      float* where = (key ? p.b.k_scale : p.b.v_scale) + uint64_t(at.page) * st[0] + block * st[1] + (h0 + h) * st[2];
      float now = __int_as_float((kv_scale_exponent(need[!key][h], Top<TC>::kInt) + 127) << 23), less = 1.f;
      if (in) {
        const float had = *where;
        if (had < now)
          less = had / now;
        else if (had >= now)  // (not NaN)
          now = had;
      }
      *where = now;
      scale[!key][h] = now;
      ratio[!key][h] = less;
    }
    __syncthreads();
    auto slot = [&](bool key, uint32_t place, uint32_t h) {
      const uint64_t* st = key ? p.c.k_stride : p.c.v_stride;
      return static_cast<TC*>(key ? p.c.k : p.c.v) + uint64_t(at.page) * st[0] + place * st[1] + (h0 + h) * st[2] + d0;
    };
    // ---- the block's earlier elements, where its scale has risen ----
    if (in)
      for (uint32_t r = row0; r < 2 * hn; r += step) {
        const bool key = r < hn;
        const uint32_t h = key ? r : r - hn;
        const float less = ratio[!key][h];
        if (less == 1.f) continue;
        for (uint32_t i = 0; i < in; ++i) {
          Eight<TC>* const dst = reinterpret_cast<Eight<TC>*>(slot(key, at.place - in + i, h));
          Eight<TC> e = *dst;
          float x[8];
          spread(e, x);
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] *= less;
          gather(x, e);
          *dst = e;
        }
      }
    // ---- the new elements, and the queries ----
    for (uint32_t i0 = 0; i0 < len; i0 += kTile) {
      const uint32_t n = min(kTile, len - i0);
      if (len > kTile) {
        __syncthreads();
        tile_angles(i0, n);
        __syncthreads();
      }
      for (uint32_t r = row0; r < 2 * hn; r += step) {
        const bool key = r < hn;
        const uint32_t h = key ? r : r - hn;
        const float now = scale[!key][h];
        // by its inverse, exact for a power of two
        const bool exact = (__float_as_uint(now) & 0x7fffffu) == 0;
        const float inverse = 1.f / now;
        for (uint32_t i = 0; i < n; ++i) {
          float x[8];
          if (key)
            rotated(key_row(i0 + i, h0 + h), i, x);
          else
            plain(value_row(i0 + i, h0 + h), x);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = exact ? x[e] * inverse : x[e] / now;
          Eight<TC> e;
          gather(x, e);
          *reinterpret_cast<Eight<TC>*>(slot(key, at.place + i0 + i, h)) = e;
        }
      }
      // a thread takes both elements of a pair: the queries may be in place
      auto query = [&](uint32_t i, uint32_t h) { return static_cast<const TI*>(a.q) + (t + i0 + i) * a.q_stride[0] + (q0 + h) * a.q_stride[1]; };
      auto query_out = [&](uint32_t i, uint32_t h) {
        return static_cast<TI*>(a.q_out) + (t + i0 + i) * a.q_out_stride[0] + (q0 + h) * a.q_out_stride[1];
      };
      if (PIECES) {
        const uint32_t both = inter ? 0 : rot / 16, per = vper - both, qstep = BTH / per, c = tid % per;
        const uint32_t d = c < both ? 8 * c : 8 * (c + both);
        for (uint32_t r = tid / per < qstep ? tid / per : ~0u; r < qn; r += qstep)
          for (uint32_t i = 0; i < n; ++i) {
            const TI* row = query(i, r) + d;
            TI* out = query_out(i, r) + d;
            const float *co = cs + i * pairs, *si = sn + i * pairs;
            Eight<TI> e;
            float x[8], o[8];
            spread(*reinterpret_cast<const Eight<TI>*>(row), x);
            if (c < both) {
              spread(*reinterpret_cast<const Eight<TI>*>(row + pairs), o);
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const float u = x[j], w = o[j];
                x[j] = u * co[d + j] - w * si[d + j];
                o[j] = w * co[d + j] + u * si[d + j];
              }
              gather(o, e);
              *reinterpret_cast<Eight<TI>*>(out + pairs) = e;
            } else if (inter && d < rot) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float u = x[2 * j], w = x[2 * j + 1];
                x[2 * j] = u * co[d / 2 + j] - w * si[d / 2 + j];
                x[2 * j + 1] = w * co[d / 2 + j] + u * si[d / 2 + j];
              }
            }
            gather(x, e);
            *reinterpret_cast<Eight<TI>*>(out) = e;
          }
      } else {
        const uint32_t items = D - pairs;  // pairs, then single elements
        for (uint32_t w = tid; w < n * qn * items; w += BTH) {
          const uint32_t j = w % items, r = w / items % qn, i = w / items / qn;
          const TI* row = query(i, r);
          TI* out = query_out(i, r);
          if (j < pairs) {
            const uint32_t da = inter ? 2 * j : j, db = inter ? 2 * j + 1 : j + pairs;
            const float u = to_float(row[da]), v = to_float(row[db]), co = cs[i * pairs + j], si = sn[i * pairs + j];
            out[da] = from_float<TI>(u * co - v * si);
            out[db] = from_float<TI>(v * co + u * si);
          } else {
            out[j + pairs] = row[j + pairs];
          }
        }
      }
    }
  }
}

template <class TI, class TC>
cudaError_t append_launch(const AppendBlocksArgs& given, int sms, cudaStream_t st) {
  AppendBlocksArgs p = given;
  auto whole = [](const void* ptr, const uint64_t* stride) {  // rows of 16-byte pieces
    return (reinterpret_cast<uintptr_t>(ptr) | stride[0] * sizeof(TI) | stride[1] * sizeof(TI)) % 16 == 0;
  };
  const bool pieces = p.a.rot_dim % (p.a.flags & XKSV_KV_INTERLEAVED ? 8 : 16) == 0 && whole(p.a.k, p.a.k_stride) &&
                      whole(p.a.v, p.a.v_stride) &&
                      (!p.a.q || (whole(p.a.q, p.a.q_stride) && whole(p.a.q_out, p.a.q_out_stride)));
  // few tokens: each its own CTA (a run's first one works); else as many as a
  // block has, up to a tile.  The heads are split where there are fewer runs
  // than the GPU holds CTAs.
  p.chunk = p.a.tokens <= 512 ? 1 : uint32_t(std::min<uint64_t>(kTile, p.b.block));
  const uint64_t runs = (p.a.tokens + p.b.block - 1) / p.b.block, room = 6 * uint64_t(sms);
  uint64_t splits = std::max<uint64_t>((p.c.kv_heads + kHeads - 1) / kHeads, std::min<uint64_t>(p.c.kv_heads, room / runs));
  splits = std::max<uint64_t>(1, std::min<uint64_t>(splits, 65535));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(uint32_t((p.a.tokens + p.chunk - 1) / p.chunk), uint32_t(splits));
  cfg.blockDim = dim3(BTH);
  cfg.dynamicSmemBytes = kTile * p.a.rot_dim * sizeof(float);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, pieces ? kv_append_blocks_kernel<TI, TC, true> : kv_append_blocks_kernel<TI, TC, false>, p);
}

template <class TI>
cudaError_t append_cache(const AppendBlocksArgs& p, int sms, cudaStream_t st) {
  return p.c.type == XKSV_INT8 ? append_launch<TI, I8>(p, sms, st) : append_launch<TI, E4m3>(p, sms, st);
}

}  // namespace

cudaError_t launch_kv_append_blocks(const AppendBlocksArgs& p, int sms, cudaStream_t st) {
  switch (p.a.type) {
    case XKSV_BF16: return append_cache<__nv_bfloat16>(p, sms, st);
    case XKSV_FP16: return append_cache<__half>(p, sms, st);
    default: return append_cache<float>(p, sms, st);
  }
}

}  // namespace xksv
