// Attention of one new token per sequence over the paged cache: a split over
// all cached tokens, one pass with running softmax statistics, and a join.
//
// Bound: every cached key and value is read once from HBM (a KV head's query
// heads share the read), so the kernel's task is to keep loads in flight.
//   * The unit of work is (sequence, KV head, up to 16 of its query heads).
//     All units' blocks of 16 or 32 tokens are shared evenly among all warps
//     of a grid that fills the GPU once (kv_index.h), whatever the lengths:
//     one long sequence and many uneven ones both keep every warp busy.
//   * A warp works alone, without block barriers: it copies its blocks through a ring of
//     kStages stages of shared memory by cp.async (16-byte pieces, XOR-swizzled
//     rows), across units' borders, so the next unit's keys are on their way
//     while one is finished.
//   * Scores and sums run on mma.sync m16n8k16, the query heads as the 16 rows
//     (the product needs 1 - 2 % of the tensor cores' rate; the wide tcgen05
//     forms need 128 rows): S = Q K^T gives each lane the weights in the very
//     layout that the second product reads them in.  Softmax statistics and
//     sums are FP32 registers.
//   * Weights reach the second product as 16-bit numbers.  BF16: as a pair
//     hi + lo of two products (2^-17 relative; one BF16 rounding, 2^-9, would
//     be as coarse as the output's own).  FP16 and E4M3: as FP16 scaled by 2^15,
//     so that weights down to 2^-29 of the largest keep 11 bits.
//   * E4M3 keys and values become FP16 exactly; the query is brought to FP16
//     after a power of two per row that puts its largest element in [2^14,
//     2^15), so that what FP16 drops is below 2^-39 of it.
//   * A unit that one warp holds alone is written at once; the others leave
//     their pieces (sums, maximum, weight) in slots, which the second kernel
//     joins in a fixed order: results do not depend on timing.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "kv_cache.h"
#include "kv_index.h"
#include "tcgen05.cuh"
#include "xksv_types.h"

namespace xksv {
namespace {

constexpr int kWarps = 4;   // per CTA
constexpr int kStages = 3;  // blocks in a warp's ring

// Shape of a kernel: the cache's elements (E8: E4M3), rows padded to DP dims.
template <bool E8, int DP>
struct Shape {
  static constexpr int ES = E8 ? 1 : 2;
  static constexpr int RB = DP * ES;              // bytes of a staged row
  static constexpr int CH = RB / 16;              // 16-byte pieces of a row (4 .. 32)
  static constexpr int BT = RB >= 256 ? 16 : 32;  // tokens of a block
  static constexpr int KV = BT * RB;              // bytes of a block's keys (or values)
  static constexpr bool QS = DP > 128;            // query fragments in shared memory, not registers
  static constexpr int QB = QS ? DP / 16 * 32 * 16 : 0;
  static constexpr int WARP = kStages * 2 * KV + QB + 16;  // + the stages' token masks
  static constexpr int CTA = kWarps * WARP;
  static constexpr int PER_SM = 2 * CTA <= 225 * 1024 ? 2 : 1;
};

// 16-byte piece c of row r: eight rows' pieces lie in eight bank groups.
template <int CH>
__device__ __forceinline__ uint32_t swz(uint32_t r, uint32_t c) {
  return CH >= 8 ? (c ^ (r & 7)) : (c ^ ((r >> 1) & 3));
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <bool BF>
__device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if (BF)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two E4M3 values (the low 16 bits of x) as FP16.
__device__ __forceinline__ uint32_t e4m3x2(uint32_t x) {
  uint32_t r;
  asm("{\n .reg .b16 t;\n cvt.u16.u32 t, %1;\n cvt.rn.f16x2.e4m3x2 %0, t;\n}\n" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <bool BF>
__device__ __forceinline__ float load16(const uint16_t* p) {
  return BF ? __uint_as_float(uint32_t(*p) << 16) : __half2float(*reinterpret_cast<const __half*>(p));
}
template <bool BF>
__device__ __forceinline__ void store16(uint16_t* p, float x) {
  if (BF)
    *reinterpret_cast<__nv_bfloat16*>(p) = __float2bfloat16_rn(x);
  else
    *reinterpret_cast<__half*>(p) = __float2half_rn(x);
}

// Position in the list of blocks: sequence, unit of the sequence, block of
// the unit; the sequence's attended tokens [first, length) (below 2^31).
struct Cursor {
  uint32_t seq, unit, block, blocks;
  int32_t first, length;
};

// Every warp's first block and the end of its range, found from the lengths.
struct Ranges {
  uint64_t total;
  uint32_t seq[kWarps];
  uint64_t before[kWarps];  // blocks ahead of that sequence
};

// FULL: head_dim is DP.
template <bool BF, bool E8, int DP, bool FULL>
__global__ void __launch_bounds__(kWarps * 32, Shape<E8, DP>::PER_SM) kv_attend_kernel(const AttendArgs p, const AttendPlan pl) {
  using Sh = Shape<E8, DP>;
  constexpr int CH = Sh::CH, BT = Sh::BT, RB = Sh::RB;
  constexpr bool MB = BF && !E8;       // BF16 products (else FP16)
  constexpr int KS = DP / 16;          // 16-dim steps
  constexpr int NB = BT / 8;           // 8-token columns of S
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Ranges R;
  __shared__ uint64_t wsum[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t D = FULL ? DP : p.c.head_dim;
  const uint32_t U = p.c.kv_heads * pl.chunks;  // units of a sequence
  // the join may start launching; it waits for this grid's end
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  asm volatile("griddepcontrol.wait;\n" ::: "memory");

  // ---- the blocks of all sequences, and where this CTA's warps start ----
  const uint64_t S = p.a.seqs;
  const uint64_t per = (S + kWarps * 32 - 1) / (kWarps * 32), s0 = min(S, per * threadIdx.x), s1 = min(S, s0 + per);
  auto span_of = [&](uint64_t s) { return kv_span(p.a.lens[s], p.a.table_cols, p.c.page_size, p.a.window); };
  auto blocks_of = [&](uint64_t s) { return kv_blocks(span_of(s), BT) * U; };
  uint64_t mine = 0;
  for (uint64_t s = s0; s < s1; ++s) {
    mine += blocks_of(s);
    if (blockIdx.x == 0 && !span_of(s).ok) atomicOr(p.status, kStatusHeader);
  }
  uint64_t incl = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint64_t x = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += x;
  }
  if (lane == 31) wsum[warp] = incl;
  __syncthreads();
  uint64_t total = 0, ahead = incl - mine;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) ahead += wsum[w];
    total += wsum[w];
  }
  const KvShare share = kv_share(total, pl.warps);
  for (int w = 0; w < kWarps; ++w) {
    const uint32_t i = blockIdx.x * kWarps + w;
    if (i >= share.workers) break;
    const uint64_t a = kv_start(share, i);
    if (a >= ahead && a < ahead + mine) {
      uint64_t at = ahead, s = s0;
      for (uint64_t n; at + (n = blocks_of(s)) <= a; ++s) at += n;
      R.seq[w] = uint32_t(s);
      R.before[w] = at;
    }
  }
  __syncthreads();
  const uint32_t me = blockIdx.x * kWarps + warp;
  if (me >= pl.warps) return;
  if (lane == 0) p.joins[me] = make_int4(0, 0, 0, 0);
  if (me >= share.workers) return;
  const uint64_t a = kv_start(share, me), b = kv_start(share, me + 1);

  uint8_t* ws = smem + warp * Sh::WARP;
  const uint32_t ring = smem_addr(ws), qsm = ring + kStages * 2 * Sh::KV;
  volatile uint32_t* masks = reinterpret_cast<volatile uint32_t*>(ws + kStages * 2 * Sh::KV + Sh::QB);
  // dims past head_dim stay zero: no copy writes there
  if (D < DP) {
    for (uint32_t i = lane; i < kStages * 2 * Sh::KV / 16; i += 32)
      reinterpret_cast<uint4*>(ws)[i] = make_uint4(0, 0, 0, 0);
    __syncwarp();
  }

  auto enter = [&](Cursor& c) {
    const KvSpan sp = span_of(c.seq);
    c.first = int32_t(sp.first);
    c.length = int32_t(sp.length);
    c.blocks = uint32_t(kv_blocks(sp, BT));
  };
  auto step = [&](Cursor& c) {
    if (++c.block < c.blocks) return;
    c.block = 0;
    if (++c.unit < U) return;
    c.unit = 0;
    if (++c.seq < S) enter(c);
  };

  // ---- copies: a block's rows, each lane one token's place ----
  const uint32_t row_ch = D * Sh::ES / 16;  // 16-byte pieces that a row really has
  const bool run = p.c.page_size % 16 == 0;  // a block's sixteen tokens lie in one page
  Cursor ld;  // of the next block to copy
  ld.seq = R.seq[warp];
  enter(ld);
  {
    const uint64_t in = a - R.before[warp];
    ld.unit = uint32_t(in / ld.blocks);
    ld.block = uint32_t(in - uint64_t(ld.unit) * ld.blocks);
  }
  Cursor cu = ld;  // of the block being worked on
  // this lane's token of the next block to copy: its rows' offsets in bytes
  bool ld_ok = false;
  uint64_t ld_k = 0, ld_v = 0;
  const uint32_t psize = uint32_t(p.c.page_size);
  auto look_up = [&]() {
    const uint32_t j = (uint32_t(ld.first) / BT + ld.block) * BT + lane;
    ld_ok = false;
    ld_k = ld_v = 0;
    if (lane < BT && j >= uint32_t(ld.first) && j < uint32_t(ld.length)) {
      const uint32_t col = pl.page_shift >= 0 ? j >> pl.page_shift : j / psize, place = j - col * psize;
      const int32_t page = p.a.table[ld.seq * p.a.table_stride + col];  // kv_span keeps the length inside the table
      if (uint32_t(page) < p.c.pages) {
        const uint32_t g = ld.unit / pl.chunks;
        ld_ok = true;
        ld_k = (uint32_t(page) * p.c.k_stride[0] + place * p.c.k_stride[1] + g * p.c.k_stride[2]) * Sh::ES;
        ld_v = (uint32_t(page) * p.c.v_stride[0] + place * p.c.v_stride[1] + g * p.c.v_stride[2]) * Sh::ES;
      } else {
        atomicOr(p.status, kStatusHeader);  // a page outside the cache
      }
    }
  };
  const uint8_t* const kb = static_cast<const uint8_t*>(p.c.k);
  const uint8_t* const vb = static_cast<const uint8_t*>(p.c.v);
  // a lane copies the same 16-byte piece of every 32 / CH-th row
  const uint32_t lr = lane / CH, lc = lane % CH;
  const uint64_t kstep = p.c.k_stride[1] * Sh::ES, vstep = p.c.v_stride[1] * Sh::ES;
  auto issue = [&](uint32_t stage) {  // copies the looked-up block into a stage, and steps on
    const uint32_t mask = __ballot_sync(0xffffffffu, ld_ok);
    if (lane == 0) masks[stage] = mask;
    const uint32_t kd = ring + stage * 2 * Sh::KV, vd = kd + Sh::KV;
    if (FULL && run && mask == (BT == 32 ? 0xffffffffu : 0xffffu)) {
      // sixteen tokens of a page lie one token's stride apart
#pragma unroll
      for (int h = 0; h < BT / 16; ++h) {
        const uint8_t* kp = kb + __shfl_sync(0xffffffffu, ld_k, 16 * h) + lr * kstep + lc * 16;
        const uint8_t* vp = vb + __shfl_sync(0xffffffffu, ld_v, 16 * h) + lr * vstep + lc * 16;
#pragma unroll
        for (int i = 0; i < CH / 2; ++i) {
          const uint32_t r = 16 * h + i * (32 / CH) + lr, off = r * RB + swz<CH>(r, lc) * 16;
          copy16(kd + off, kp);
          copy16(vd + off, vp);
          kp += (32 / CH) * kstep;
          vp += (32 / CH) * vstep;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < BT * CH / 32; ++i) {
        const uint32_t r = i * (32 / CH) + lr;
        const uint64_t kr = __shfl_sync(0xffffffffu, ld_k, r), vr = __shfl_sync(0xffffffffu, ld_v, r);
        // masked tokens are zeros: no garbage (NaN) meets their zero weight
        const uint32_t n = (mask >> r) & 1 ? 16u : 0u;
        if (FULL || lc < row_ch) {
          const uint32_t off = r * RB + swz<CH>(r, lc) * 16;
          cp_async16_zfill(kd + off, kb + kr + lc * 16, n);
          cp_async16_zfill(vd + off, vb + vr + lc * 16, n);
        }
      }
    }
    step(ld);
  };

  // ---- the unit being worked on ----
  constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;
  constexpr float kUp = MB ? 0.f : 15.f;  // weights are scaled by 2^kUp
  const int r0 = lane >> 2, qc = lane & 3;
  constexpr int QK = Sh::QS ? 1 : KS;
  uint32_t qf[QK][4];
  float o[2 * KS][4], m[2], l[2], qs[2];  // rows r0 and r0 + 8
  uint32_t head0 = 0, heads = 0;  // the unit's query heads
  auto begin = [&]() {
    const uint32_t group = p.a.q_heads / p.c.kv_heads, g = cu.unit / pl.chunks, ch = cu.unit % pl.chunks;
    head0 = g * group + ch * pl.heads;
    heads = min(pl.heads, group - ch * pl.heads);
    const uint16_t* q = static_cast<const uint16_t*>(p.a.q) + cu.seq * p.a.q_stride[0];
    float scale[2] = {p.a.scale, p.a.scale};
    if (E8 && p.c.k_scale) scale[0] = scale[1] = p.a.scale * p.c.k_scale[g];
    float up[2] = {1.f, 1.f};
    if (E8) {
      // the rows' powers of two
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float mx = 0.f;
        if (uint32_t(r0 + 8 * h) < heads) {
          const uint16_t* qr = q + (head0 + r0 + 8 * h) * p.a.q_stride[1];
          for (uint32_t d = qc; d < D; d += 4) mx = fmaxf(mx, fabsf(load16<BF>(qr + d)));
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        if (mx > 0.f && mx < INFINITY) {
          // an exponent whose inverse is a normal number too
          const int e = max(-110, min(126, 14 - ilogbf(mx)));
          up[h] = ldexpf(1.f, e);
          scale[h] = ldexpf(scale[h], -e);
        }
      }
    }
    // scores in powers of two (a softcap acts on the natural ones first)
    const float pw = p.a.softcap > 0.f ? 1.f : kLog2e;
    qs[0] = scale[0] * pw;
    qs[1] = scale[1] * pw;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      uint32_t f[4] = {0, 0, 0, 0};
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (uint32_t(r0 + 8 * h) < heads) {
          const uint16_t* qr = q + (head0 + r0 + 8 * h) * p.a.q_stride[1];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            // dims of this lane's element pairs: E4M3 rows give a lane four
            // dims in a row (both pairs), 16-bit rows two and two
            const uint32_t d = ks * 16 + (E8 ? 4 * qc + 2 * x : 2 * qc + 8 * x);
            if (d < D) {
              if (E8)
                f[h + 2 * x] = pack_f16(load16<BF>(qr + d) * up[h], load16<BF>(qr + d + 1) * up[h]);
              else
                f[h + 2 * x] = uint32_t(qr[d]) | (uint32_t(qr[d + 1]) << 16);
            }
          }
        }
      if (Sh::QS) {
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(qsm + (ks * 32 + lane) * 16), "r"(f[0]),
                     "r"(f[1]), "r"(f[2]), "r"(f[3])
                     : "memory");
      } else {
#pragma unroll
        for (int x = 0; x < 4; ++x) qf[Sh::QS ? 0 : ks][x] = f[x];
      }
    }
#pragma unroll
    for (int i = 0; i < 2 * KS; ++i)
#pragma unroll
      for (int x = 0; x < 4; ++x) o[i][x] = 0.f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
  };

  // dims of accumulator column i, element x (0, 1: row r0; 2, 3: row r0 + 8)
  auto dim_of = [&](int i, int x) -> uint32_t {
    return E8 ? (i >> 1) * 16 + 4 * qc + 2 * (x & 1) + (i & 1) : i * 8 + 2 * qc + (x & 1);
  };
  auto finish = [&](uint64_t t) {  // block t was the unit's last in this warp's range
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
    const uint64_t u0 = t - cu.block, u1 = u0 + cu.blocks;
    const KvPiece piece = kv_piece(share, me, a, b, u0, u1);
    if (piece.slot < 0) {
      const float vs = E8 && p.c.v_scale ? p.c.v_scale[cu.unit / pl.chunks] : 1.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t head = r0 + 8 * h;
        if (head >= heads) continue;
        const bool some = l[h] > 0.f || l[h] != l[h];
        const float f = some ? vs / l[h] : 0.f;
        uint16_t* out = static_cast<uint16_t*>(p.a.out) + cu.seq * p.a.out_stride[0] + (head0 + head) * p.a.out_stride[1];
#pragma unroll
        for (int i = 0; i < 2 * KS; ++i)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint32_t d = dim_of(i, x);
            if (d < D) store16<BF>(out + d, some ? o[i][2 * h + x] * f : 0.f);
          }
        if (qc == 0 && p.a.lse)
          p.a.lse[uint64_t(cu.seq) * p.a.q_heads + head0 + head] =
              some ? (m[h] == -INFINITY ? 0.f : m[h] + log2f(l[h]) - kUp) * kLn2 : -INFINITY;
      }
    } else {
      float* slot = p.slots + uint64_t(piece.slot) * pl.slot_floats;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t head = r0 + 8 * h;
        if (head >= heads) continue;
#pragma unroll
        for (int i = 0; i < 2 * KS; ++i)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            if (dim_of(i, x) < D) slot[head * DP + dim_of(i, x)] = o[i][2 * h + x];
        if (qc == 0) {
          slot[pl.heads * DP + 2 * head] = m[h];
          slot[pl.heads * DP + 2 * head + 1] = l[h];
        }
      }
      if (piece.parts && lane == 0) p.joins[me] = make_int4(int(cu.seq), int(cu.unit), int(piece.parts), 0);
    }
  };

  look_up();
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    if (a + i < b) {
      issue(i);
      if (a + i + 1 < b) look_up();
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  }
  begin();
  uint32_t stage = 0, put = kStages - 1;  // stages to read and to fill next
  for (uint64_t t = a; t < b; ++t) {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(kStages - 2) : "memory");
    __syncwarp();
    const uint32_t kd = ring + stage * 2 * Sh::KV, vd = kd + Sh::KV;
    const uint32_t mask = masks[stage];
    // the stage before this one is free: every lane has passed the barrier
    if (t + kStages - 1 < b) {
      issue(put);
      if (t + kStages < b) look_up();
    }
    stage = stage + 1 == kStages ? 0 : stage + 1;
    put = put + 1 == kStages ? 0 : put + 1;
    asm volatile("cp.async.commit_group;\n" ::: "memory");

    // ---- S = Q K^T ----
    float sc[NB][4];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) sc[n][x] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ks += E8 ? 2 : 1) {
      if (!FULL && uint32_t(ks * 16) >= D) break;
      uint32_t qa[2][4];
#pragma unroll
      for (int y = 0; y < (E8 ? 2 : 1); ++y) {
        if (Sh::QS)
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n"
                       : "=r"(qa[y][0]), "=r"(qa[y][1]), "=r"(qa[y][2]), "=r"(qa[y][3])
                       : "r"(qsm + ((ks + y) * 32 + lane) * 16)
                       : "memory");
        else
#pragma unroll
          for (int x = 0; x < 4; ++x) qa[y][x] = qf[Sh::QS ? 0 : ks + y][x];
      }
#pragma unroll
      for (int tb = 0; tb < BT / 16; ++tb) {
        const uint32_t row = tb * 16 + (lane >> 4) * 8 + (lane & 7);
        const uint32_t c = (E8 ? ks : 2 * ks) + ((lane >> 3) & 1);
        uint32_t r[4];
        ldsm4(kd + row * RB + swz<CH>(row, c) * 16, r);
        if (E8) {
          mma<false>(sc[2 * tb], qa[0], e4m3x2(r[0]), e4m3x2(r[0] >> 16));
          mma<false>(sc[2 * tb], qa[1], e4m3x2(r[1]), e4m3x2(r[1] >> 16));
          mma<false>(sc[2 * tb + 1], qa[0], e4m3x2(r[2]), e4m3x2(r[2] >> 16));
          mma<false>(sc[2 * tb + 1], qa[1], e4m3x2(r[3]), e4m3x2(r[3] >> 16));
        } else {
          mma<MB>(sc[2 * tb], qa[0], r[0], r[1]);
          mma<MB>(sc[2 * tb + 1], qa[0], r[2], r[3]);
        }
      }
    }
    // ---- softmax step, in powers of two ----
    float mx[2] = {m[0], m[1]};
    if (p.a.softcap > 0.f) {
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int x = 0; x < 4; ++x) sc[n][x] = kLog2e * p.a.softcap * tanhf(sc[n][x] * qs[x >> 1] / p.a.softcap);
    } else {
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int x = 0; x < 4; ++x) sc[n][x] *= qs[x >> 1];
    }
    if (mask != (BT == 32 ? 0xffffffffu : 0xffffu)) {
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if (!((mask >> (n * 8 + 2 * qc + (x & 1))) & 1)) sc[n][x] = -INFINITY;
    }
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) mx[x >> 1] = fmaxf(mx[x >> 1], sc[n][x]);
    float base[2];
    bool grew = false;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
      base[h] = mx[h] == -INFINITY ? 0.f : mx[h] - kUp;
      grew |= mx[h] != m[h];
    }
    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float f = exp2_fast(m[h] - (mx[h] == -INFINITY ? 0.f : mx[h]));
        l[h] *= f;
#pragma unroll
        for (int i = 0; i < 2 * KS; ++i) {
          o[i][2 * h] *= f;
          o[i][2 * h + 1] *= f;
        }
        m[h] = mx[h];
      }
    }
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        sc[n][x] = exp2_fast(sc[n][x] - base[x >> 1]);
        l[x >> 1] += sc[n][x];
      }
    // ---- O += P V ----
#pragma unroll
    for (int tb = 0; tb < BT / 16; ++tb) {
      const float* s0 = sc[2 * tb];
      const float* s1 = sc[2 * tb + 1];
      uint32_t hi[4], lo[4];
      if (MB) {
        hi[0] = pack_bf16(s0[0], s0[1]);
        hi[1] = pack_bf16(s0[2], s0[3]);
        hi[2] = pack_bf16(s1[0], s1[1]);
        hi[3] = pack_bf16(s1[2], s1[3]);
        auto rest = [](uint32_t h, float x, float y) {
          return pack_bf16(x - __uint_as_float(h << 16), y - __uint_as_float(h & 0xffff0000u));
        };
        lo[0] = rest(hi[0], s0[0], s0[1]);
        lo[1] = rest(hi[1], s0[2], s0[3]);
        lo[2] = rest(hi[2], s1[0], s1[1]);
        lo[3] = rest(hi[3], s1[2], s1[3]);
      } else {
        hi[0] = pack_f16(s0[0], s0[1]);
        hi[1] = pack_f16(s0[2], s0[3]);
        hi[2] = pack_f16(s1[0], s1[1]);
        hi[3] = pack_f16(s1[2], s1[3]);
      }
      const uint32_t row = tb * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
#pragma unroll
      for (int dc = 0; dc < CH; dc += 2) {  // two 16-byte pieces of every row
        if (!FULL && uint32_t(dc) >= row_ch) break;
        uint32_t r[4];
        ldsm4t(vd + row * RB + swz<CH>(row, dc + (lane >> 4)) * 16, r);
        if (E8) {
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            // bytes (dim 2n, 2n + 1) of two tokens -> dim 2n of both, dim 2n + 1 of both
            const uint32_t t0 = __byte_perm(r[2 * y], 0, 0x3120), t1 = __byte_perm(r[2 * y + 1], 0, 0x3120);
            mma<false>(o[2 * (dc + y)], hi, e4m3x2(t0), e4m3x2(t1));
            mma<false>(o[2 * (dc + y) + 1], hi, e4m3x2(t0 >> 16), e4m3x2(t1 >> 16));
          }
        } else {
          mma<MB>(o[dc], hi, r[0], r[1]);
          mma<MB>(o[dc + 1], hi, r[2], r[3]);
          if (MB) {
            mma<MB>(o[dc], lo, r[0], r[1]);
            mma<MB>(o[dc + 1], lo, r[2], r[3]);
          }
        }
      }
    }
    const bool last = cu.block + 1 == cu.blocks;
    if (last || t + 1 == b) finish(t);
    step(cu);
    if (last && t + 1 < b) begin();
  }
  asm volatile("cp.async.wait_group 0;\n" ::: "memory");
}

constexpr int JT = 256;                // threads of a join
constexpr uint32_t kJoin = JT / 32;    // workers whose units a CTA joins, and parts that a warp joins alone

// Joins the pieces of the units that workers 8 x .. 8 x + 7 begin, for query
// head y of their chunk.  A unit of few parts takes one warp, all its loads in
// flight at once; of the eight at most one has more than eight (its parts are
// successive workers), and that one takes the whole CTA: the parts' weights
// once in shared memory, then each warp every eighth part, lanes the dims;
// last the warps' sums in order.
template <bool BF>
__global__ void __launch_bounds__(JT) kv_join_kernel(const AttendArgs p, const AttendPlan pl, float up) {
  extern __shared__ float weight[];  // [workers]
  __shared__ __align__(16) float so[JT / 32][256];
  __shared__ float red[2][JT / 32];
  __shared__ int4 big;
  __shared__ uint32_t big_at;
  constexpr float kLn2 = 0.69314718055994531f;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t head = blockIdx.y, DP = pl.pad_dim, D = p.c.head_dim;
  const uint32_t group = p.a.q_heads / p.c.kv_heads, st = pl.heads * DP + 2 * head;
  if (threadIdx.x == 0) big_at = ~0u;
  __syncthreads();
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  auto slot = [&](uint32_t i, uint32_t k) { return p.slots + uint64_t(k ? 2 * (i + k) : 2 * i + 1) * pl.slot_floats; };
  struct Unit {
    uint32_t head, kv_head;
    bool mine;
  };
  auto unit_of = [&](int4 j) {
    const uint32_t g = uint32_t(j.y) / pl.chunks, ch = uint32_t(j.y) % pl.chunks;
    return Unit{g * group + ch * pl.heads + head, g, head < min(pl.heads, group - ch * pl.heads)};
  };
  auto out_of = [&](int4 j, const Unit& u) {
    return static_cast<uint16_t*>(p.a.out) + uint64_t(j.x) * p.a.out_stride[0] + u.head * p.a.out_stride[1];
  };
  auto scale_of = [&](const Unit& u, float l) {  // no weight at all: zeros
    return l > 0.f || l != l ? (p.c.v_scale ? p.c.v_scale[u.kv_head] : 1.f) / l : 0.f;
  };
  auto put_lse = [&](int4 j, const Unit& u, float base, float l) {
    if (p.a.lse)
      p.a.lse[uint64_t(j.x) * p.a.q_heads + u.head] = l > 0.f || l != l ? (base + log2f(l) - up) * kLn2 : -INFINITY;
  };
  const uint32_t i = blockIdx.x * kJoin + warp;
  const int4 j = i < pl.warps ? p.joins[i] : make_int4(0, 0, 0, 0);
  if (uint32_t(j.z) > kJoin) {
    if (lane == 0) {
      big = j;
      big_at = i;
    }
  } else if (j.z) {
    const Unit u = unit_of(j);
    if (u.mine) {
      float m[kJoin], w[kJoin], l = 0.f, base = -INFINITY;
#pragma unroll
      for (uint32_t k = 0; k < kJoin; ++k) {
        m[k] = k < uint32_t(j.z) ? slot(i, k)[st] : -INFINITY;
        w[k] = k < uint32_t(j.z) ? slot(i, k)[st + 1] : 0.f;
      }
      float acc[8] = {};
      float v[kJoin][4];  // 128 dims of every part at a time
      auto fetch = [&](uint32_t d0) {
#pragma unroll
        for (uint32_t k = 0; k < kJoin; ++k)
#pragma unroll
          for (uint32_t x = 0; x < 4; ++x) {
            const uint32_t d = d0 + x * 32 + lane;
            v[k][x] = k < uint32_t(j.z) && d < D ? slot(i, k)[head * DP + d] : 0.f;
          }
      };
      fetch(0);
#pragma unroll
      for (uint32_t k = 0; k < kJoin; ++k) base = fmaxf(base, m[k]);
      base = base == -INFINITY ? 0.f : base;
#pragma unroll
      for (uint32_t k = 0; k < kJoin; ++k) {
        m[k] = k < uint32_t(j.z) ? exp2f(m[k] - base) : 0.f;
        l += w[k] * m[k];
      }
#pragma unroll
      for (uint32_t k = 0; k < kJoin; ++k)
#pragma unroll
        for (uint32_t x = 0; x < 4; ++x) acc[x] += k < uint32_t(j.z) ? v[k][x] * m[k] : 0.f;
      if (D > 128) {
        fetch(128);
#pragma unroll
        for (uint32_t k = 0; k < kJoin; ++k)
#pragma unroll
          for (uint32_t x = 0; x < 4; ++x) acc[4 + x] += k < uint32_t(j.z) ? v[k][x] * m[k] : 0.f;
      }
      const float f = scale_of(u, l);
      const bool some = l > 0.f || l != l;
      uint16_t* out = out_of(j, u);
#pragma unroll
      for (int x = 0; x < 8; ++x)
        if (x * 32 + lane < D) store16<BF>(out + x * 32 + lane, some ? acc[x] * f : 0.f);
      if (lane == 0) put_lse(j, u, base, l);
    }
  }
  __syncthreads();
  const uint32_t many = big_at;
  const int4 jm = big;
  if (many == ~0u) return;
  const Unit u = unit_of(jm);
  if (!u.mine) return;
  const uint32_t parts = uint32_t(jm.z);
  float mt = -INFINITY;
  for (uint32_t k = threadIdx.x; k < parts; k += JT) {
    weight[k] = slot(many, k)[st];
    mt = fmaxf(mt, weight[k]);
  }
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, d));
  if (lane == 0) red[0][warp] = mt;
  __syncthreads();
  for (int w = 0; w < JT / 32; ++w) mt = fmaxf(mt, red[0][w]);
  const float base = mt == -INFINITY ? 0.f : mt;
  float l = 0.f;
  for (uint32_t k = threadIdx.x; k < parts; k += JT) {
    weight[k] = exp2f(weight[k] - base);
    l += slot(many, k)[st + 1] * weight[k];
  }
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
  if (lane == 0) red[1][warp] = l;
  __syncthreads();
  l = 0.f;
  for (int w = 0; w < JT / 32; ++w) l += red[1][w];
  // four dims a lane, two such rows for more than 128 dims
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    const uint32_t d = (y * 32 + lane) * 4;
    if (d >= D) break;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (uint32_t k = warp; k < parts; k += JT / 32) {
      const float4 v = *reinterpret_cast<const float4*>(slot(many, k) + head * DP + d);
      const float f = weight[k];
      acc.x += v.x * f;
      acc.y += v.y * f;
      acc.z += v.z * f;
      acc.w += v.w * f;
    }
    *reinterpret_cast<float4*>(&so[warp][d]) = acc;
  }
  __syncthreads();
  const float f = scale_of(u, l);
  const bool some = l > 0.f || l != l;
  uint16_t* out = out_of(jm, u);
  for (uint32_t d = threadIdx.x; d < D; d += JT) {
    float x = 0.f;
    for (int w = 0; w < JT / 32; ++w) x += so[w][d];
    store16<BF>(out + d, some ? x * f : 0.f);
  }
  if (threadIdx.x == 0) put_lse(jm, u, base, l);
}

int pad_dim(uint32_t d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

template <bool BF, bool E8, int DP, bool FULL>
cudaError_t launch_attend(const AttendArgs& p, const AttendPlan& pl, cudaStream_t st) {
  using Sh = Shape<E8, DP>;
  const cudaError_t e = cudaFuncSetAttribute(kv_attend_kernel<BF, E8, DP, FULL>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::CTA);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((pl.warps + kWarps - 1) / kWarps);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = Sh::CTA;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t f = cudaLaunchKernelEx(&cfg, kv_attend_kernel<BF, E8, DP, FULL>, p, pl);
  if (f != cudaSuccess) return f;
  cfg.gridDim = dim3((pl.warps + kJoin - 1) / kJoin, pl.heads);
  cfg.blockDim = dim3(JT);
  cfg.dynamicSmemBytes = pl.warps * sizeof(float);
  return cudaLaunchKernelEx(&cfg, kv_join_kernel<BF>, p, pl, BF && !E8 ? 0.f : 15.f);
}

template <bool BF, bool E8>
cudaError_t launch_dim(const AttendArgs& p, const AttendPlan& pl, cudaStream_t st) {
  const bool full = p.c.head_dim == pl.pad_dim;
  switch (pl.pad_dim) {
    case 64: return full ? launch_attend<BF, E8, 64, true>(p, pl, st) : launch_attend<BF, E8, 64, false>(p, pl, st);
    case 128: return full ? launch_attend<BF, E8, 128, true>(p, pl, st) : launch_attend<BF, E8, 128, false>(p, pl, st);
    default: return full ? launch_attend<BF, E8, 256, true>(p, pl, st) : launch_attend<BF, E8, 256, false>(p, pl, st);
  }
}

template <bool E8>
void shape_of(int dp, uint32_t* block, uint32_t* per_sm) {
  *block = dp == 64 ? Shape<E8, 64>::BT : dp == 128 ? Shape<E8, 128>::BT : Shape<E8, 256>::BT;
  *per_sm = dp == 64 ? Shape<E8, 64>::PER_SM : dp == 128 ? Shape<E8, 128>::PER_SM : Shape<E8, 256>::PER_SM;
}

}  // namespace

AttendPlan kv_attend_plan(const xksv_kv_desc& c, uint64_t seqs, uint32_t q_heads, uint64_t table_cols, int sms) {
  AttendPlan pl{};
  const uint32_t group = q_heads / c.kv_heads;
  pl.chunks = (group + 15) / 16;
  pl.heads = (group + pl.chunks - 1) / pl.chunks;
  pl.pad_dim = uint32_t(pad_dim(c.head_dim));
  pl.page_shift = -1;
  for (int k = 0; k < 31; ++k)
    if (c.page_size == 1ull << k) pl.page_shift = k;
  uint32_t block = 16, per_sm = 1;
  if (c.type == XKSV_E4M3)
    shape_of<true>(int(pl.pad_dim), &block, &per_sm);
  else
    shape_of<false>(int(pl.pad_dim), &block, &per_sm);
  // no more workers than blocks of the longest sequences the table can hold
  const uint64_t longest = table_cols * c.page_size / block + 1;
  const uint64_t blocks = seqs * c.kv_heads * pl.chunks;
  const uint64_t most = uint64_t(sms) * per_sm * kWarps;
  pl.warps = uint32_t(blocks >= most || longest >= most ? most : std::min<uint64_t>(most, blocks * longest));
  pl.slot_floats = (uint64_t(pl.heads) * (pl.pad_dim + 2) + 31) / 32 * 32;
  pl.joins_off = 2 * pl.warps * pl.slot_floats * sizeof(float);
  pl.bytes = pl.joins_off + pl.warps * sizeof(int4);
  return pl;
}

cudaError_t launch_kv_attend(const AttendArgs& p, const AttendPlan& pl, cudaStream_t st) {
  const bool bf = p.a.type == XKSV_BF16, e8 = p.c.type == XKSV_E4M3;
  if (bf) return e8 ? launch_dim<true, true>(p, pl, st) : launch_dim<true, false>(p, pl, st);
  return e8 ? launch_dim<false, true>(p, pl, st) : launch_dim<false, false>(p, pl, st);
}

}  // namespace xksv
