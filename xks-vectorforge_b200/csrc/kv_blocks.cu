// Append to a paged cache of 8-bit elements with a scale for each block of
// tokens and head (include/xksv_cuda.h, part 8).
//
// A run is what one call adds to one block: tokens of a sequence that stand
// next to each other.  A head's elements of a run can only be stored once the
// largest of them is known.  Scales are powers of two: a raised scale costs an
// earlier element at most the bits that fall below its new least one, and an
// E4M3 element none but near zero.
//   * Runs of a token or few, and any strides and alignment: a CTA takes runs, whole
//     (and a share of the heads, where there are few runs), and goes over their
//     keys and values twice, the second time from L1.  Bound by the chain of
//     loads: place, page, rows, scale.
//   * Prompts (the rule stands in `append_launch`): the queries go through the 16-bit caches' append kernel, keys and
//     values by runs, a warp a head, which holds its rows in registers between
//     the two passes.  Bound by instructions (1.8 a cycle, 24 warps an SM), about twice those
//     of the 16-bit append's keys and values.
// Measured on one B200 (a graph of calls): one token of 32 + 8 heads of 128 6.0 us, 200
// tokens of 28 + 4 heads 8.1, 3001 of 20 + 20 heads of 80 41, 16384 of 32 + 8
// heads 112 (3290 GB/s; the 16-bit append 71).  All by the first kernel: 16384
// tokens 159 us; the second with four heads' keys and values a CTA 126, which computes the
// angles twice; queries in it too 146 (registers spill).  Longer blocks, of which a CTA
// takes those that begin among its 16 tokens, leave others idle and are read tile by
// tile, twice: of 16, 64, 128 and 256 tokens, a prompt of 1000 17, 44, 75 and 135 us, 16384
// 108, 118, 155 and 238.  Inputs off 16-byte pieces, or rotated halves that fill none, go
// element by element through the first kernel: 1000 tokens 83 us, 3001 101, 16384 307
// (17, 24 and 112 by pieces; the 16-bit append so 25, 40 and 227).
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
constexpr bool kInteger = false;
template <>
constexpr bool kInteger<I8> = true;

// Whether token o, a run's first, breaks the order that a call's tokens have to
// keep, next to the one before: a sequence's tokens stand together and rise by
// one.  `begins`: it is its sequence's first (behind another's or padding), which
// must not have come before.
__device__ __forceinline__ bool out_of_order(const xksv_kv_append_args& a, uint64_t o, bool& begins) {
  begins = false;
  if (!a.seq || !o) return false;
  begins = a.seq[o - 1] != a.seq[o] || a.index[o - 1] < 0;
  return !begins && int64_t(a.index[o - 1]) + 1 != a.index[o];
}
// Whether token o's sequence has come before: this thread's share of all tokens before
// (many loads at a time: a loop of single ones took longer than all the rest of a
// prompt's append).
__device__ __forceinline__ bool came_before(const xksv_kv_append_args& a, uint64_t o) {
  const int32_t seq = a.seq[o];
  bool wrong = false;
  constexpr int kAtOnce = 16;
  for (uint64_t e = threadIdx.x; e + 1 < o; e += kAtOnce * blockDim.x) {
    int32_t other[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) other[i] = e + i * blockDim.x + 1 < o ? a.seq[e + i * blockDim.x] : ~seq;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) wrong |= other[i] == seq && a.index[e + i * blockDim.x] >= 0;
  }
  return wrong;
}

// The same for the tokens t + i of the bits i of `begin` (of 32), read once for all of
// them: reads for each token by itself took 16384 one-token sequences 322 us, 120 without `seq`.
__device__ __forceinline__ bool any_came_before(const xksv_kv_append_args& a, uint64_t t, uint32_t begin) {
  const uint32_t lane = threadIdx.x & 31, last = 31 - __clz(begin);
  const bool one = begin >> lane & 1;
  const int32_t own = one ? a.seq[t + lane] : 0;  // (of a sequence: not negative)
  const int32_t low = __reduce_min_sync(0xffffffffu, one ? own : INT32_MAX), high = __reduce_max_sync(0xffffffffu, own);
  bool wrong = false;
  constexpr int kAtOnce = 16;
  for (uint64_t e = threadIdx.x; e + 1 < t + last; e += kAtOnce * blockDim.x) {
    int32_t other[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) other[i] = e + i * blockDim.x + 1 < t + last ? a.seq[e + i * blockDim.x] : -1;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i)
      if (other[i] >= low && other[i] <= high)
        for (uint32_t f = begin; f; f &= f - 1) {
          const uint64_t o = t + __ffs(f) - 1, at = e + i * blockDim.x;
          wrong |= at + 1 < o && a.seq[o] == other[i] && a.index[at] >= 0;
        }
  }
  return wrong;
}

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
      bool first;
      bool wrong = out_of_order(a, t, first) || at.page < 0;
      if (first && came_before(a, t)) wrong = true;
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
        if (kInteger<TC> && nan) atomicOr(p.status, kStatusHeader);  // (an integer holds none)
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
      float now = __int_as_float((kv_scale_exponent(need[!key][h], kInteger<TC>) + 127) << 23), less = 1.f;
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

// ---- many tokens: keys and values by runs, a warp a head (the queries go
// through the 16-bit caches' kernel) ----
constexpr int RT = 256;          // threads of a CTA
constexpr uint32_t kWarps = RT / 32;
constexpr uint32_t kChunk = 16;  // tokens whose runs a CTA takes
constexpr uint32_t kSpan = 32;   // tokens of a tile at most

// The magnitudes' largest, as the bits of FP32 numbers (infinity and NaN above all others).
__device__ __forceinline__ uint32_t largest(const float* x, uint32_t high) {
#pragma unroll
  for (int e = 0; e < 8; e += 2)
    high = __vimax3_u32(high, __float_as_uint(x[e]) & 0x7fffffffu, __float_as_uint(x[e + 1]) & 0x7fffffffu);
  return high;
}
// The same with what is no number left out, and whether there was NaN.
__device__ __forceinline__ uint32_t largest_finite(const float* x, uint32_t high, bool& nan) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t m = __float_as_uint(x[e]) & 0x7fffffffu;
    nan |= m > 0x7f800000u;
    high = m < 0x7f800000u ? max(high, m) : high;
  }
  return high;
}

// The largest magnitude of eight stored elements, as such bits: 16-bit ones two
// at a time, since their bits are ordered as they are.
__device__ __forceinline__ uint32_t largest(const Eight<__nv_bfloat16>& a) {
  // (no sign bits: as signed numbers, whose maximum of three is one instruction)
  const uint32_t m = __vimax3_s16x2(__vimax3_s16x2(a.w[0] & 0x7fff7fffu, a.w[1] & 0x7fff7fffu, a.w[2] & 0x7fff7fffu), a.w[3] & 0x7fff7fffu, 0);
  return max(m << 16, m & 0xffff0000u);
}
__device__ __forceinline__ uint32_t largest(const Eight<__half>& a) {
  // (no sign bits: as signed numbers, whose maximum of three is one instruction)
  const uint32_t m = __vimax3_s16x2(__vimax3_s16x2(a.w[0] & 0x7fff7fffu, a.w[1] & 0x7fff7fffu, a.w[2] & 0x7fff7fffu), a.w[3] & 0x7fff7fffu, 0);
  return __float_as_uint(__half2float(__ushort_as_half(uint16_t(max(m & 0xffffu, m >> 16)))));
}
__device__ __forceinline__ uint32_t largest(const Eight<float>& a) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, a.w[i] & 0x7fffffffu);
  return m;
}

// What the first warp finds for the CTA: the next runs, and their tokens' places.
struct Tile {
  uint64_t t;        // first token
  uint32_t len;      // tokens of the runs (0: no more)
  uint32_t firsts;   // the runs' first tokens, from t
  uint32_t good;     // tokens whose page is in the cache
  uint32_t begin;    // the firsts that begin a sequence
  uint32_t next;     // where this CTA goes on
  int32_t page[kSpan];
  uint32_t place[kSpan];
};

// A CTA takes the runs that begin among its 16 tokens, eight heads' keys or eight
// heads' values: as many as lie in a tile of 32, or a longer one tile by tile.
// Each warp has a head: it reads its rows into registers, all at once and, of
// keys, while the CTA computes the tile's angles; then, without a barrier, finds
// what they need, sets the scales and stores them.
template <class TI, class TC>
__global__ void __launch_bounds__(RT, 3) kv_append_runs_kernel(const AppendBlocksArgs p) {
  extern __shared__ __align__(16) float trig[];  // cosines [kSpan][pairs], then sines
  __shared__ Tile tile;
  __shared__ uint32_t need[kWarps][kSpan];                        // a warp's runs: what they need,
  __shared__ float inverse[kWarps][kSpan], ratio[kWarps][kSpan];  // their scales' inverses and rise
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  const xksv_kv_append_args& a = p.a;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t D = p.c.head_dim, rot = a.rot_dim, pairs = rot / 2, B = uint32_t(p.b.block), P = uint32_t(p.c.page_size);
  const bool inter = a.flags & XKSV_KV_INTERLEAVED;
  // this CTA's heads
  const uint32_t y = blockIdx.y, ys = gridDim.y;
  const bool key = y < ys / 2;  // (the others: values)
  const uint32_t group = key ? y : y - ys / 2, h0 = uint32_t(uint64_t(p.c.kv_heads) * group / (ys / 2));
  const uint32_t hn = uint32_t(uint64_t(p.c.kv_heads) * (group + 1) / (ys / 2)) - h0;
  float *const cs = trig, *const sn = trig + kSpan * pairs;
  // Lanes of a row: of values one a piece; a key's lane takes both elements of
  // its pairs, of rotated halves a piece and its partner (`both` such lanes)
  const uint32_t vper = D / 8, both = inter ? 0 : rot / 16, per = vper - both;

  auto seq_of = [&](uint64_t t) { return a.seq ? int64_t(a.seq[t]) : int64_t(t); };
  const uint64_t t0 = uint64_t(blockIdx.x) * p.chunk;
  // the first warp: of the 32 tokens from t0, which begin a run and which go on
  uint32_t follow = 0, begins = 0;
  if (warp == 0) {
    bool live = false, goes = false;
    if (t0 + lane < a.tokens) {
      live = seq_of(t0 + lane) >= 0 && a.index[t0 + lane] >= 0;
      goes = live && kv_follows(a.seq, a.index, t0 + lane, B);
    }
    follow = __ballot_sync(0xffffffffu, goes);
    begins = __ballot_sync(0xffffffffu, live) & ~follow;
  }
  auto find_places = [&](uint64_t t, uint32_t n) {  // of the tile's tokens, by the first warp
    KvPlace w{-1, 0};
    if (lane < n) {
      w = kv_place(a.table, a.table_rows, a.table_cols, a.table_stride, p.c.pages, P, seq_of(t + lane), a.index[t + lane]);
      tile.page[lane] = w.page;
      tile.place[lane] = w.place;
    }
    const uint32_t good = __ballot_sync(0xffffffffu, w.page >= 0);
    if (lane == 0) tile.good = good;
    if (lane < n && w.page < 0 && y == 0) atomicOr(p.status, kStatusHeader);
  };
  auto find_tile = [&](uint32_t at) {  // the first warp: the runs from token `at` on
    auto end_of = [&](uint32_t from) {  // of the run that begins at `from` (32: there or later)
      const uint32_t rest = from < 31 ? ~follow & ~((2u << from) - 1) : 0;
      return rest ? uint32_t(__ffs(rest)) - 1 : 32u;
    };
    const uint32_t starts = at < 32 ? begins & ~((1u << at) - 1) : 0;
    at = starts ? __ffs(starts) - 1 : 32;
    if (at >= p.chunk) {
      if (lane == 0) tile.len = 0;
      return;
    }
    const uint64_t t = t0 + at;
    uint32_t end = end_of(at), len = end - at, firsts = 1;
    if (end < 32 && len <= kSpan) {
      for (uint32_t next; end < p.chunk && (begins >> end & 1) && (next = end_of(end)) < 32 && next - at <= kSpan; end = next)
        firsts |= 1u << (end - at);
      len = end - at;
    } else if (end == 32) {
      for (uint32_t more = ~0u; more == ~0u; len += more == ~0u ? 32 : __ffs(~more) - 1) {
        const uint64_t o = t + len + lane;
        more = __ballot_sync(0xffffffffu, o < a.tokens && kv_follows(a.seq, a.index, o, B));
      }
    }
    find_places(t, min(len, kSpan));
    bool begin = false;
    if (y == 0 && lane < kSpan && (firsts >> lane & 1) && out_of_order(a, t + lane, begin)) atomicOr(p.status, kStatusHeader);
    const uint32_t begin_set = __ballot_sync(0xffffffffu, begin);
    if (lane == 0) tile.t = t, tile.len = len, tile.firsts = firsts, tile.next = end, tile.begin = begin_set;
  };
  auto tile_angles = [&](uint64_t t, uint32_t n) {  // of n tokens from t
    if (!key || !pairs) return;
    for (uint32_t k = tid / pairs, f = tid % pairs, at_k = RT / pairs, at_f = RT % pairs; k < n;) {
      // of rotated halves the pairs 8 j .. 8 j + 3 first, then 8 j + 4 .. 8 j + 7:
      // a row's lanes read next to each other
      const uint32_t where = k * pairs + (inter ? f : (f >> 2 & 1) * (pairs / 2) + (f >> 3) * 4 + (f & 3));
      angle_of(a.positions ? a.positions[t + k] : a.index[t + k], a.inv_freq[f], a.rot_scale, &cs[where], &sn[where]);
      k += at_k, f += at_f;
      if (f >= pairs) f -= pairs, ++k;
    }
  };
  auto run_of = [&](uint32_t i) { return tile.len <= kSpan ? 31 - __clz(tile.firsts & ((2u << i) - 1)) : 0; };

  // ---- a head's keys or values, by this warp: lanes that take row `sub` of
  // `once` at a time, from dim d on ----
  const uint32_t h = h0 + warp;
  const bool mine = warp < hn;
  const uint32_t lanes = key ? per : vper, once = 32 / lanes, sub = lane / lanes, c = lane - sub * lanes;
  const uint32_t d = key && c >= both ? 8 * (c + both) : 8 * c;
  const bool pair = key && c < both, idle = !mine || sub >= once;
  const uint64_t from_step = key ? a.k_stride[0] : a.v_stride[0];
  const TI* const from = static_cast<const TI*>(key ? a.k : a.v) + h * (key ? a.k_stride[1] : a.v_stride[1]) + d;
  const uint64_t to_page = key ? p.c.k_stride[0] : p.c.v_stride[0], to_place = key ? p.c.k_stride[1] : p.c.v_stride[1];
  TC* const to = static_cast<TC*>(key ? p.c.k : p.c.v) + h * (key ? p.c.k_stride[2] : p.c.v_stride[2]) + d;
  constexpr uint32_t kRaw = sizeof(TI) == 4 ? 4 : 8;  // pieces a lane holds: a key's with their partners
  const uint32_t batch = (key ? kRaw / 2 : kRaw) * once;
  Eight<TI> raw[kRaw];
  // the batch's rows of the tile's n tokens from t
  auto fetch = [&](uint64_t t, uint32_t n, uint32_t b0) {
    if (idle) return;
    const TI* row = from + (t + b0 + sub) * from_step;
    if (key) {
#pragma unroll
      for (uint32_t z = 0; z < kRaw / 2; ++z, row += once * from_step)
        if (b0 + sub + z * once < n) {
          raw[2 * z] = *reinterpret_cast<const Eight<TI>*>(row);
          if (pair) raw[2 * z + 1] = *reinterpret_cast<const Eight<TI>*>(row + pairs);
        }
    } else {
#pragma unroll
      for (uint32_t z = 0; z < kRaw; ++z, row += once * from_step)
        if (b0 + sub + z * once < n) raw[z] = *reinterpret_cast<const Eight<TI>*>(row);
    }
  };
  uint32_t high = 0;  // what a single run needs so far
  auto note = [&](uint32_t i, uint32_t m, auto again) {
    if (m >= 0x7f800000u) {  // an infinite element saturates, and an integer holds no NaN
      bool nan = false;
      m = again(nan);
      if (kInteger<TC> && nan && tile.good >> i & 1) atomicOr(p.status, kStatusHeader);
    }
    if (tile.firsts == 1)
      high = max(high, m);
    else
      atomicMax(&need[warp][run_of(i)], m);
  };
  auto held = [&](TC* at, float f, float* x) {
    if (f > 0.f) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= f;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = __fdiv_rn(x[e], -f);
    }
    Eight<TC> e;
    gather(x, e);
    *reinterpret_cast<Eight<TC>*>(at) = e;
  };
  // the batch: what it needs, or, `put`, into its places
  auto work = [&](uint32_t n, uint32_t b0, bool put) {
    if (idle) return;
    if (key) {
#pragma unroll
      for (uint32_t z = 0; z < kRaw / 2; ++z) {
        const uint32_t i = b0 + sub + z * once;
        if (i >= n) break;
        float x[8], o[8];
        spread(raw[2 * z], x);
        const float *co = cs + i * pairs, *si = sn + i * pairs;
        if (pair) {
          spread(raw[2 * z + 1], o);
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const uint32_t at = g * (pairs / 2) + 4 * c;
            const float4 c4 = *reinterpret_cast<const float4*>(co + at), s4 = *reinterpret_cast<const float4*>(si + at);
            const float cc[4] = {c4.x, c4.y, c4.z, c4.w}, ss[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float l = x[4 * g + j], w = o[4 * g + j];
              x[4 * g + j] = l * cc[j] - w * ss[j];
              o[4 * g + j] = w * cc[j] + l * ss[j];
            }
          }
        } else if (inter && d < rot) {
          const float4 c4 = *reinterpret_cast<const float4*>(co + 4 * c), s4 = *reinterpret_cast<const float4*>(si + 4 * c);
          const float cc[4] = {c4.x, c4.y, c4.z, c4.w}, ss[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float l = x[2 * j], w = x[2 * j + 1];
            x[2 * j] = l * cc[j] - w * ss[j];
            x[2 * j + 1] = w * cc[j] + l * ss[j];
          }
        }
        if (!put) {
          note(i, pair ? largest(o, largest(x, 0)) : largest(x, 0), [&](bool& nan) {
            const uint32_t m = largest_finite(x, 0, nan);
            return pair ? largest_finite(o, m, nan) : m;
          });
        } else if (tile.good >> i & 1) {
          const float f = inverse[warp][run_of(i)];
          TC* at = to + uint64_t(tile.page[i]) * to_page + tile.place[i] * to_place;
          held(at, f, x);
          if (pair) held(at + pairs, f, o);
        }
      }
    } else {
#pragma unroll
      for (uint32_t z = 0; z < kRaw; ++z) {
        const uint32_t i = b0 + sub + z * once;
        if (i >= n) break;
        if (!put) {
          note(i, largest(raw[z]), [&](bool& nan) {
            float x[8];
            spread(raw[z], x);
            return largest_finite(x, 0, nan);
          });
        } else if (tile.good >> i & 1) {
          float x[8];
          spread(raw[z], x);
          held(to + uint64_t(tile.page[i]) * to_page + tile.place[i] * to_place, inverse[warp][run_of(i)], x);
        }
      }
    }
  };
  // the runs' scales (lane: the run's first token), and where they rise the
  // blocks' earlier elements
  auto set_scales = [&] {
    if (tile.firsts == 1) {
      high = __reduce_max_sync(0xffffffffu, high);
      if (lane == 0) need[warp][0] = high;
    }
    __syncwarp();
    const uint64_t* st = key ? p.b.k_stride : p.b.v_stride;
    bool risen = false;
    if (lane < kSpan && (tile.firsts >> lane & 1) && tile.page[lane] >= 0) {
      float* where = (key ? p.b.k_scale : p.b.v_scale) + uint64_t(tile.page[lane]) * st[0] + tile.place[lane] / B * st[1] + h * st[2];
      float now = __int_as_float((kv_scale_exponent(need[warp][lane], kInteger<TC>) + 127) << 23), less = 1.f;
      if (tile.place[lane] % B) {
        const float had = *where;
        if (had < now)
          less = had / now;
        else if (had >= now)  // (not NaN)
          now = had;
      }
      *where = now;
      // a power of two's inverse is exact; another scale divides
      inverse[warp][lane] = (__float_as_uint(now) & 0x7fffffu) == 0 ? 1.f / now : -now;
      ratio[warp][lane] = less;
      risen = less != 1.f;
    }
    uint32_t some = __ballot_sync(0xffffffffu, risen);
    __syncwarp();
    const uint32_t v_once = 32 / vper, v_sub = lane / vper;
    for (; some; some &= some - 1) {
      const uint32_t i = __ffs(some) - 1, in = tile.place[i] % B;
      const float less = ratio[warp][i];
      for (uint32_t j = v_sub < v_once ? v_sub : ~0u; j < in; j += v_once) {
        TC* at = to - d + 8 * (lane - v_sub * vper) + uint64_t(tile.page[i]) * to_page + (tile.place[i] - in + j) * to_place;
        Eight<TC> e = *reinterpret_cast<const Eight<TC>*>(at);
        float x[8];
        spread(e, x);
#pragma unroll
        for (int z = 0; z < 8; ++z) x[z] *= less;
        gather(x, e);
        *reinterpret_cast<Eight<TC>*>(at) = e;
      }
    }
  };
  for (uint32_t at = 0;; at = tile.next) {
    __syncthreads();
    if (warp == 0) find_tile(at);
    __syncthreads();
    const uint32_t len = tile.len;
    if (!len) return;
    const uint64_t t = tile.t;
    high = 0;
    if (lane < kSpan) need[warp][lane] = 0;
    const bool small = len <= kSpan;
    for (int put = 0; put < 2; ++put) {
      for (uint32_t i0 = 0; i0 < len; i0 += kSpan) {
        const uint32_t n = min(kSpan, len - i0);
        const bool again = put && small;  // (the tile is as it was)
        if (!again || n > batch) fetch(t + i0, n, 0);
        if (!again) {
          if (!small) {
            __syncthreads();
            if (warp == 0) find_places(t + i0, n);
          }
          tile_angles(t + i0, n);
          __syncthreads();
        }
        for (uint32_t b0 = 0; b0 < n; b0 += batch) {
          if (b0) fetch(t + i0, n, b0);
          work(n, b0, put);
        }
      }
      if (put) break;
      if (tile.begin && any_came_before(a, t, tile.begin)) atomicOr(p.status, kStatusHeader);
      if (!small) {
        __syncthreads();
        if (warp == 0) find_places(t, kSpan);
        __syncthreads();
      }
      if (mine) set_scales();
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
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  const uint64_t room = 6 * uint64_t(sms);
  // Tokens up to which one kernel does all: it gives a run a CTA that goes over it
  // token by token; the other has a fixed price of two launches and its tiles.  First
  // kernel and runs, us, 32 + 8 heads of 128 E4M3: one-token sequences without `seq` 512
  // 11.1 and 17.1, 2048 20.3 and 21.9, 4096 36.5 and 33.5; blocks of one token (16 heads
  // of 64) 512 9.5 and 13.7, 4096 31 and 35.  With `seq` what a call holds is not known
  // here but for its tokens a row of the table at least.  A row, blocks of 16: 8
  // tokens 19 and 10, 64 35 and 14, 512 41 and 16; 64 rows, one token each 8.8 and 36, two
  // 11.6 and 17.5, four 16.0 and 17.7, eight 27 and 19; 20 + 20 heads of 80, blocks of 24,
  // four 24 and 16; one row of 64 tokens in a block of 64 (64 + 8 heads) 134 and 43, in
  // blocks of 4 13 and 15; 1024 of one token 44 and 47.
  const bool single = !p.a.seq || p.b.block == 1;
  const uint64_t few = single ? 2048 : p.a.tokens >= 8 * p.a.table_rows && p.b.block >= 8 ? 0 : 512;
  if (pieces && p.a.tokens > few) {
    if (p.a.q) {
      AppendArgs q{p.a, p.c, p.status};
      q.c.kv_heads = 0;
      const cudaError_t e = launch_kv_append(q, sms, st);
      if (e != cudaSuccess) return e;
    }
    p.chunk = kChunk;
    const uint64_t tiles = (p.a.tokens + kChunk - 1) / kChunk, splits = 2 * ((p.c.kv_heads + kWarps - 1) / kWarps);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(uint32_t(tiles), uint32_t(splits));
    cfg.blockDim = dim3(RT);
    cfg.dynamicSmemBytes = kSpan * p.a.rot_dim * sizeof(float);
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kv_append_runs_kernel<TI, TC>, p);
  }
  // few tokens, or runs of one: each its own CTA (a run's first one works); else as
  // many as a block has, up to a tile.  The heads are split where there are fewer runs
  // than the GPU holds CTAs (one-token sequences without `seq` taken for runs of a
  // block's tokens: 512 22 us, not 11).
  p.chunk = single || p.a.tokens <= 512 ? 1 : uint32_t(std::min<uint64_t>(kTile, p.b.block));
  const uint64_t runs = single ? p.a.tokens : (p.a.tokens + p.b.block - 1) / p.b.block;
  uint64_t splits = std::max<uint64_t>((p.c.kv_heads + kHeads - 1) / kHeads, std::min<uint64_t>(p.c.kv_heads, room / runs));
  splits = std::max<uint64_t>(1, std::min<uint64_t>(splits, 65535));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(uint32_t((p.a.tokens + p.chunk - 1) / p.chunk), uint32_t(splits));
  cfg.blockDim = dim3(BTH);
  cfg.dynamicSmemBytes = kTile * p.a.rot_dim * sizeof(float);
  cfg.stream = st;
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
