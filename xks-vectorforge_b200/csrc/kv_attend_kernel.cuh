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
//   * Scores and sums run on mma.sync m16n8k16 with the tokens, then the dims,
//     as its 16 rows and eight query heads as its columns: S^T = K Q^T, O^T =
//     V^T P^T (the product needs about 1 % of the tensor cores' rate; the wide
//     tcgen05 forms need 128 rows).  Up to eight heads of a KV head cost one
//     such product, and their softmax no padded rows; the weights pass from
//     the first product's layout to the second's by movmatrix.  Softmax
//     statistics and sums are FP32 registers.
//   * Weights reach the second product as 16-bit numbers, a pair hi + lo of two
//     products (BF16: 2^-17 relative, FP16 and E4M3: FP16, 2^-23): one rounding
//     would be as coarse as a result of the same type.  FP16 weights are scaled
//     by 2^15, so that less than 2^-40 of the largest falls out of FP16's range.  (One FP16
//     rounding: 64 uneven FP16 sequences 375 us against 377, E4M3 105 against
//     107, and an FP16 result 1.35 times as far from the exact one.)
//   * E4M3 keys and values become FP16 exactly; the query is brought to FP16
//     after a power of two per row that puts its largest element in [2^14,
//     2^15), so that what FP16 drops is below 2^-39 of it.
//   * Block scales: a token's scales travel with its rows through the ring. A
//     score is multiplied by its key's; a weight enters its product as its
//     value's part of the sixteen tokens' largest scale, which the FP32 sums take
//     in as they add the product, in units of the largest scale so far.  Integers become
//     FP16 exactly, as low bits of 1024.
//   * A unit that one warp holds alone is written at once; the others leave
//     their pieces (sums, maximum, weight) in slots, which the second kernel
//     joins in a fixed order: results do not depend on timing.
//   * Calls of few units over short tables give each unit a cluster of CTAs
//     instead, which joins its pieces through shared memory (CL, kShort).
// Measured on one B200 (32 query and 8 KV heads of 128, BF16): 131071 tokens
// of one sequence 100 us, 5370 GB/s with the join (a copy: 6554); 64 uneven
// sequences to 16384 tokens 395 us, 5440 GB/s; one of 777 tokens 7.6 us.  E4M3,
// 28 and 4 heads, 130 uneven sequences to 6000: 88 us, 4250 GB/s, the
// conversion's instructions besides the reads.  Block scales (of 16 tokens):
// 131071 tokens 65 us, 4130 GB/s (E4M3 with a scale per head 62); 64 uneven
// sequences to 16384 of integers 235 to 245 us, 4570 GB/s, under the power cap that they
// reach (217 in the first milliseconds; E4M3 per head 216); the 130 with a scale for
// each token 101 us against 88.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "kernels.h"
#include "kv_cache.h"
#include "kv_index.h"
#include "tcgen05.cuh"
#include "xksv_types.h"

namespace xksv {
namespace {

constexpr int kWarps = 4;   // per CTA
constexpr int kCluster = 8;  // CTAs of a unit whose pieces meet in shared memory (CL)
static_assert(kCluster * kWarps == 32, "the join reads a piece's statistics per lane");
constexpr int kStages = 2;  // blocks in a warp's ring: one landing while one is worked on

// The cache's elements: 16 bits; E4M3 with a scale per head; E4M3 or integers
// with one for each block of tokens.
enum : int { EL16 = 0, ELE4M3 = 1, ELE4M3Blocks = 2, ELInt8Blocks = 3 };

// Shape of a kernel: the cache's elements, rows padded to DP dims, NG groups of
// eight query heads.
template <int EL, int DP, int NG>
struct Shape {
  static constexpr bool E8 = EL != EL16, BS = EL >= ELE4M3Blocks;
  static constexpr int ES = E8 ? 1 : 2;
  static constexpr int RB = DP * ES;              // bytes of a staged row
  static constexpr int CH = RB / 16;              // 16-byte pieces of a row (4 .. 32)
  static constexpr int BT = RB >= 256 ? 16 : 32;  // tokens of a block
  static constexpr int KV = BT * RB;              // bytes of a block's keys (or values)
  static constexpr bool QS = DP * NG > 256;       // query fragments in shared memory, not registers
  static constexpr int QB = QS ? DP / 16 * 32 * 8 * NG : 0;
  static constexpr int SB = BS ? kStages * 2 * BT * 4 : 0;      // the stages' scales
  static constexpr int ST = BS ? 3 : 2;                         // a head's statistics in a piece: maximum, weight, the sums' unit
  static constexpr int WARP = kStages * 2 * KV + QB + SB + 16;  // + the stages' token masks
  static constexpr int CTA = kWarps * WARP;
  // CTAs an SM holds.  Three of two stages against two of three stages: 64
  // uneven sequences 399 us against 409, E4M3 85 against 92
  static constexpr int PER_SM = 3 * CTA <= 225 * 1024 ? 3 : 2 * CTA <= 225 * 1024 ? 2 : 1;
};

// The units of the sums with block scales: the least power of two that holds a
// scale, of [2^-64, 2^126]: the inverses are normal numbers too, and so is a unit
// divided by a sum of 2^31 weights of 2^15; the smallest scale is 2^-85 units.
constexpr float kLeastUnit = 0x1p-64f, kMostUnit = 0x1p126f;
__device__ __forceinline__ float unit_of(float scale) {
  return __uint_as_float(min((__float_as_uint(fmaxf(scale, kLeastUnit)) + 0x7fffffu) & 0x7f800000u, __float_as_uint(kMostUnit)));
}
__device__ __forceinline__ float inverse_of(float unit) { return __uint_as_float(0x7f000000u - __float_as_uint(unit)); }

// 16-byte piece c of row r: eight rows' pieces lie in eight bank groups.
template <int CH>
__device__ __forceinline__ uint32_t swz(uint32_t r, uint32_t c) {
  return CH >= 8 ? (c ^ (r & 7)) : (c ^ ((r >> 1) & 3));
}

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
}
// Four bytes, or zeros for n = 0.
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, uint32_t n) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(n) : "memory");
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
// Four E4M3 values as two pairs of FP16.
__device__ __forceinline__ void e4m3x4(uint32_t x, uint32_t& lo, uint32_t& hi) {
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;\n}\n"
      : "=r"(lo), "=r"(hi)
      : "r"(x));
}
// Four integers as two pairs of FP16: v + 128 as the low bits of 1024 + (v + 128).
// In order, or the first and third, then the second and fourth.
template <bool ACROSS>
__device__ __forceinline__ void int8x4(uint32_t x, uint32_t& lo, uint32_t& hi) {
  constexpr uint32_t kBase = 0x64806480u;  // 1152
  x ^= 0x80808080u;
  lo = __byte_perm(x, 0x64646464u, ACROSS ? 0x4240 : 0x4140);
  hi = __byte_perm(x, 0x64646464u, ACROSS ? 0x4341 : 0x4342);
  asm("sub.rn.f16x2 %0, %0, %1;\n" : "+r"(lo) : "r"(kBase));
  asm("sub.rn.f16x2 %0, %0, %1;\n" : "+r"(hi) : "r"(kBase));
}
// Four bytes of the cache, in order or across, as FP16.
template <int EL, bool ACROSS>
__device__ __forceinline__ void widen4(uint32_t x, uint32_t& lo, uint32_t& hi) {
  if (EL == ELInt8Blocks)
    int8x4<ACROSS>(x, lo, hi);
  else
    e4m3x4(ACROSS ? __byte_perm(x, 0, 0x3120) : x, lo, hi);
}
// The 8 x 8 matrix of 16-bit elements that the warp holds, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(x));
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
__device__ __forceinline__ float unpack16(bool bf, uint32_t x) {  // the low 16 bits
  return bf ? __uint_as_float(x << 16) : __half2float(__ushort_as_half(uint16_t(x)));
}
__device__ __forceinline__ void store16(bool bf, uint16_t* p, float x) {
  if (bf)
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

// A float of this shared-memory address in CTA `rank` of the cluster.
__device__ __forceinline__ float ld_cluster(uint32_t addr, uint32_t rank) {
  uint32_t r;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(r) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_barrier() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release;\n barrier.cluster.wait.acquire;\n" ::: "memory");
}

// MB: BF16 products (else FP16); FULL: head_dim is DP.
// CL (calls of few units and short tables): a unit's blocks are shared by the
// 32 warps of a cluster of CTAs, which then join their pieces from one
// another's shared memory: no second kernel and no workspace.
template <bool MB, int EL, int DP, int NG, bool FULL, bool CL>
__global__ void __launch_bounds__(kWarps * 32, Shape<EL, DP, NG>::PER_SM) kv_attend_kernel(const AttendArgs p, const AttendPlan pl) {
  using Sh = Shape<EL, DP, NG>;
  constexpr bool E8 = Sh::E8, BS = Sh::BS;
  constexpr int CH = Sh::CH, BT = Sh::BT, RB = Sh::RB;
  constexpr int KS = DP / 16;  // 16-dim steps
  constexpr int TB = BT / 16;  // 16-token steps
  const bool bf = E8 ? p.a.type == XKSV_BF16 : MB;
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
  KvShare share{};
  uint32_t me = 0;
  uint64_t a = 0, b = 0;
  const uint32_t cl_seq = CL ? blockIdx.x / kCluster / U : 0, cl_unit = CL ? blockIdx.x / kCluster % U : 0;
  const uint32_t cl_group = p.a.q_heads / p.c.kv_heads, cl_chunk = cl_unit % pl.chunks;
  const uint32_t cl_head0 = cl_unit / pl.chunks * cl_group + cl_chunk * pl.heads;
  const uint32_t cl_heads = CL ? min(pl.heads, cl_group - cl_chunk * pl.heads) : 0;
  auto span_of = [&](uint64_t s) { return kv_span(p.a.lens[s], p.a.table_cols, p.c.page_size, p.a.window); };
  auto blocks_of = [&](uint64_t s) { return kv_blocks(span_of(s), BT) * U; };
  if constexpr (CL) {
    const KvSpan sp = span_of(cl_seq);
    const uint32_t rank = blockIdx.x % kCluster;
    if (!sp.ok && cl_unit == 0 && rank == 0 && threadIdx.x == 0) atomicOr(p.status, kStatusHeader);
    share = kv_share(kv_blocks(sp, BT), kCluster * kWarps);
    if (!share.total) {  // the whole cluster: nothing to attend to
      if (rank) return;
      for (uint32_t h = warp; h < cl_heads; h += kWarps) {
        uint16_t* out = static_cast<uint16_t*>(p.a.out) + cl_seq * p.a.out_stride[0] + (cl_head0 + h) * p.a.out_stride[1];
        for (uint32_t d = lane; d < D; d += 32) out[d] = 0;
        if (lane == 0 && p.a.lse) p.a.lse[uint64_t(cl_seq) * p.a.q_heads + cl_head0 + h] = -INFINITY;
      }
      return;
    }
    me = rank * kWarps + warp;
    if (me < share.workers) a = kv_start(share, me), b = kv_start(share, me + 1);
  } else {
    const uint64_t per = (S + kWarps * 32 - 1) / (kWarps * 32), s0 = min(S, per * threadIdx.x), s1 = min(S, s0 + per);
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
    // sequences without a token to attend to: zeros, by the CTAs in turn
    for (uint64_t s = blockIdx.x; s < S; s += gridDim.x) {
      if (blocks_of(s)) continue;
      uint16_t* out = static_cast<uint16_t*>(p.a.out) + s * p.a.out_stride[0];
      for (uint32_t x = threadIdx.x; x < p.a.q_heads * D; x += kWarps * 32) out[x / D * p.a.out_stride[1] + x % D] = 0;
      for (uint32_t h = threadIdx.x; p.a.lse && h < p.a.q_heads; h += kWarps * 32) p.a.lse[s * p.a.q_heads + h] = -INFINITY;
    }
    share = kv_share(total, pl.warps);
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
    me = blockIdx.x * kWarps + warp;
    if (me >= pl.warps) return;
    if (lane == 0) p.joins[me] = make_int4(0, 0, 0, 0);
    if (me >= share.workers) return;  // all of them when there is no block
    a = kv_start(share, me), b = kv_start(share, me + 1);
  }

  uint8_t* ws = smem + warp * Sh::WARP;
  const uint32_t ring = smem_addr(ws), qsm = ring + kStages * 2 * Sh::KV;
  volatile uint32_t* masks = reinterpret_cast<volatile uint32_t*>(ws + kStages * 2 * Sh::KV + Sh::QB + Sh::SB);
  // a stage's scales: BT keys', BT values'; masked tokens' are zero
  const volatile float* scales = reinterpret_cast<const volatile float*>(ws + kStages * 2 * Sh::KV + Sh::QB);
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
    // the next sequence that has tokens, 32 looked at a time (there is one:
    // a range's last block is not stepped past)
    for (uint64_t s = c.seq + 1; s < S; s += 32) {
      const uint32_t some = __ballot_sync(0xffffffffu, s + lane < S && blocks_of(s + lane) != 0);
      if (some) {
        c.seq = uint32_t(s) + __ffs(some) - 1;
        break;
      }
    }
    enter(c);
  };

  // ---- copies: a block's rows, each lane one token's place ----
  const uint32_t row_ch = D * Sh::ES / 16;  // 16-byte pieces that a row really has
  const bool run = p.c.page_size % 16 == 0;  // a block's sixteen tokens lie in one page
  Cursor ld;  // of the next block to copy
  ld.seq = CL ? cl_seq : R.seq[warp];
  enter(ld);
  if (CL) {
    ld.unit = cl_unit;
    ld.block = uint32_t(a);
  } else {
    const uint64_t in = a - R.before[warp];
    ld.unit = uint32_t(in / ld.blocks);
    ld.block = uint32_t(in - uint64_t(ld.unit) * ld.blocks);
  }
  Cursor cu = ld;  // of the block being worked on
  // this lane's token of the next block to copy: its rows' offsets in bytes
  bool ld_ok = false;
  uint64_t ld_k = 0, ld_v = 0;
  uint32_t ld_page = 0, ld_place = 0;  // block scales: where it is, for `issue` (offsets take registers that they lack)
  const uint32_t psize = uint32_t(p.c.page_size);
  auto look_up = [&]() {
    const uint32_t j = (uint32_t(ld.first) / BT + ld.block) * BT + lane;
    ld_ok = false;
    ld_k = ld_v = 0;
    if (lane < BT && j >= uint32_t(ld.first) && j < uint32_t(ld.length)) {
      const uint32_t col = pl.page_shift >= 0 ? j >> pl.page_shift : j / psize, place = j - col * psize;
      const int32_t page = p.a.table[ld.seq * p.a.table_stride + col];  // kv_span keeps the length inside the table
      if (uint32_t(page) < p.c.pages) {
        ld_ok = true;
        if (BS) {
          ld_page = uint32_t(page), ld_place = place;
        } else {
          const uint32_t g = ld.unit / pl.chunks;
          ld_k = (uint32_t(page) * p.c.k_stride[0] + place * p.c.k_stride[1] + g * p.c.k_stride[2]) * Sh::ES;
          ld_v = (uint32_t(page) * p.c.v_stride[0] + place * p.c.v_stride[1] + g * p.c.v_stride[2]) * Sh::ES;
        }
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
  auto issue = [&](uint32_t stage) {  // copies the looked-up block into a stage
    const uint32_t mask = __ballot_sync(0xffffffffu, ld_ok);
    if (lane == 0) masks[stage] = mask;
    const uint32_t kd = ring + stage * 2 * Sh::KV, vd = kd + Sh::KV;
    if (BS) {
      const uint32_t g = ld.unit / pl.chunks, page = ld_ok ? ld_page : 0, place = ld_ok ? ld_place : 0;
      ld_k = page * p.c.k_stride[0] + place * p.c.k_stride[1] + g * p.c.k_stride[2];
      ld_v = page * p.c.v_stride[0] + place * p.c.v_stride[1] + g * p.c.v_stride[2];
      if (lane < BT) {
        const uint32_t block = pl.block_shift >= 0 ? place >> pl.block_shift : place / uint32_t(p.b.block);
        const uint32_t sd = qsm + Sh::QB + (stage * 2 * BT + lane) * 4;
        copy4(sd, p.b.k_scale + page * p.b.k_stride[0] + block * p.b.k_stride[1] + g * p.b.k_stride[2], ld_ok ? 4 : 0);
        copy4(sd + BT * 4, p.b.v_scale + page * p.b.v_stride[0] + block * p.b.v_stride[1] + g * p.b.v_stride[2], ld_ok ? 4 : 0);
      }
    }
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
  };

  // ---- the unit being worked on ----
  constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;
  constexpr float kUp = MB ? 0.f : 15.f;  // weights are scaled by 2^kUp
  // A lane's elements of a product's 16 x 8 result: rows hr and hr + 8
  // (elements 0, 1 and 2, 3), columns (query heads) 2 qc and 2 qc + 1.
  const int hr = lane >> 2, qc = lane & 3;
  uint32_t qf[Sh::QS ? 1 : KS][NG][2];
  float o[NG][KS][4], m[NG][2], l[NG][2], qs[NG][2];
  float unit = 1.f;  // block scales: what the sums are in units of
  uint32_t head0 = 0, heads = 0;  // the unit's query heads
  const bool q_pairs = ((reinterpret_cast<uintptr_t>(p.a.q) / 2 | p.a.q_stride[0] | p.a.q_stride[1]) & 1) == 0;
  auto begin = [&]() {
    unit = kLeastUnit;
    const uint32_t group = p.a.q_heads / p.c.kv_heads, g = cu.unit / pl.chunks, ch = cu.unit % pl.chunks;
    head0 = g * group + ch * pl.heads;
    heads = min(pl.heads, group - ch * pl.heads);
    const uint16_t* q = static_cast<const uint16_t*>(p.a.q) + cu.seq * p.a.q_stride[0];
    // scores in powers of two (a softcap acts on the natural ones first)
    float scale = p.a.scale * (p.a.softcap > 0.f ? 1.f : kLog2e);
    if (E8 && p.c.k_scale) scale *= p.c.k_scale[g];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const uint32_t head = 8 * n + hr;  // the head whose query this lane holds parts of
      const uint16_t* qr = q + (head0 + head) * p.a.q_stride[1];
      uint32_t f[KS][2];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          // dims of this lane's element pairs: E4M3 rows give a lane four
          // dims in a row (both pairs), 16-bit rows two and two
          const uint32_t d = ks * 16 + (E8 ? 4 * qc + 2 * x : 2 * qc + 8 * x);
          f[ks][x] = 0;
          if (head < heads && (FULL || d < D))
            f[ks][x] = q_pairs ? *reinterpret_cast<const uint32_t*>(qr + d) : uint32_t(qr[d]) | (uint32_t(qr[d + 1]) << 16);
        }
      float mine = scale;
      if (E8) {
        float mx = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int x = 0; x < 2; ++x) mx = fmaxf(mx, fmaxf(fabsf(unpack16(bf, f[ks][x])), fabsf(unpack16(bf, f[ks][x] >> 16))));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        float up = 1.f;
        if (mx > 0.f && mx < INFINITY) {
          // an exponent whose inverse is a normal number too
          const int e = max(-110, min(126, 14 - ilogbf(mx)));
          up = __int_as_float((e + 127) << 23);
          mine = ldexpf(scale, -e);
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int x = 0; x < 2; ++x) f[ks][x] = pack_f16(unpack16(bf, f[ks][x]) * up, unpack16(bf, f[ks][x] >> 16) * up);
      }
      qs[n][0] = __shfl_sync(0xffffffffu, mine, 8 * qc);
      qs[n][1] = __shfl_sync(0xffffffffu, mine, 8 * qc + 4);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if (Sh::QS) {
          asm volatile("st.shared.v2.b32 [%0], {%1, %2};\n" ::"r"(qsm + ((ks * NG + n) * 32 + lane) * 8), "r"(f[ks][0]),
                       "r"(f[ks][1])
                       : "memory");
        } else {
          qf[Sh::QS ? 0 : ks][n][0] = f[ks][0];
          qf[Sh::QS ? 0 : ks][n][1] = f[ks][1];
        }
      }
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[n][i][x] = 0.f;
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
    }
  };
  // dim of row hr + 8 y of accumulator i
  auto dim_of = [&](int i, int y) -> uint32_t { return i * 16 + (E8 ? 2 * hr + y : hr + 8 * y); };
  auto finish = [&](uint64_t t) {  // block t was the unit's last in this warp's range
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[n][h] += __shfl_xor_sync(0xffffffffu, l[n][h], d);
    const uint64_t u0 = t - cu.block, u1 = u0 + cu.blocks;
    const KvPiece piece = CL ? KvPiece{0, 0} : kv_piece(share, me, a, b, u0, u1);
    if (piece.slot < 0) {
      const float vs = BS ? unit : E8 && p.c.v_scale ? p.c.v_scale[cu.unit / pl.chunks] : 1.f;
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t head = 8 * n + 2 * qc + h;
          if (head >= heads) continue;
          const bool some = l[n][h] > 0.f || l[n][h] != l[n][h];
          const float f = some ? vs / l[n][h] : 0.f;
          uint16_t* out = static_cast<uint16_t*>(p.a.out) + cu.seq * p.a.out_stride[0] + (head0 + head) * p.a.out_stride[1];
#pragma unroll
          for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int y = 0; y < 2; ++y)
              if (FULL || dim_of(i, y) < D) store16(bf, out + dim_of(i, y), some ? o[n][i][2 * y + h] * f : 0.f);
          if (hr == 0 && p.a.lse)
            p.a.lse[uint64_t(cu.seq) * p.a.q_heads + head0 + head] =
                some ? ((m[n][h] == -INFINITY ? 0.f : m[n][h]) + log2f(l[n][h]) - kUp) * kLn2 : -INFINITY;
        }
    } else {
      // (CL: over the ring, whose last block every lane has read by now)
      if (CL) __syncwarp();
      float* slot = CL ? reinterpret_cast<float*>(ws) : p.slots + uint64_t(piece.slot) * pl.slot_floats;
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t head = 8 * n + 2 * qc + h;
          if (head >= heads) continue;
#pragma unroll
          for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int y = 0; y < 2; ++y)
              if (FULL || dim_of(i, y) < D) slot[head * DP + dim_of(i, y)] = o[n][i][2 * y + h];
          if (hr == 0) {
            float* const stat = slot + pl.heads * DP + Sh::ST * head;
            stat[0] = m[n][h], stat[1] = l[n][h];
            if (BS) stat[2] = unit;
          }
        }
      if (!CL && piece.parts && lane == 0) p.joins[me] = make_int4(int(cu.seq), int(cu.unit), int(piece.parts), 0);
    }
  };

  if (a < b) look_up();
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    if (a + i < b) {
      issue(i);
      if (a + i + 1 < b) {
        step(ld);
        look_up();
      }
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  }
  if (a < b) begin();
  uint32_t stage = 0, put = kStages - 1;  // stages to read and to fill next
  for (uint64_t t = a; t < b; ++t) {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(kStages - 2) : "memory");
    __syncwarp();
    const uint32_t kd = ring + stage * 2 * Sh::KV, vd = kd + Sh::KV;
    const uint32_t mask = masks[stage];
    float ks[TB][2];  // of this lane's tokens
    const volatile float* const vscale = scales + stage * 2 * BT + BT;  // of the block's tokens
    if (BS) {
#pragma unroll
      for (int tb = 0; tb < TB; ++tb)
#pragma unroll
        for (int y = 0; y < 2; ++y) ks[tb][y] = scales[stage * 2 * BT + tb * 16 + hr + 8 * y];
    }
    // the stage before this one is free: every lane has passed the barrier
    if (t + kStages - 1 < b) {
      issue(put);
      if (t + kStages < b) {
        step(ld);
        look_up();
      }
    }
    stage = stage + 1 == kStages ? 0 : stage + 1;
    put = put + 1 == kStages ? 0 : put + 1;
    asm volatile("cp.async.commit_group;\n" ::: "memory");

    // ---- S^T = K Q^T ----
    float sc[TB][NG][4];
#pragma unroll
    for (int tb = 0; tb < TB; ++tb)
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int x = 0; x < 4; ++x) sc[tb][n][x] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ks += E8 ? 2 : 1) {
      if (!FULL && uint32_t(ks * 16) >= D) break;
      constexpr int Y = E8 ? 2 : 1;
      uint32_t qb[Y][NG][2];
#pragma unroll
      for (int y = 0; y < Y; ++y)
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          if (Sh::QS) {
            asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];\n"
                         : "=r"(qb[y][n][0]), "=r"(qb[y][n][1])
                         : "r"(qsm + (((ks + y) * NG + n) * 32 + lane) * 8)
                         : "memory");
          } else {
            qb[y][n][0] = qf[Sh::QS ? 0 : ks + y][n][0];
            qb[y][n][1] = qf[Sh::QS ? 0 : ks + y][n][1];
          }
        }
#pragma unroll
      for (int tb = 0; tb < TB; ++tb) {
        // tokens 0 .. 7 and 8 .. 15 of one 16-byte piece, then of the next
        const uint32_t row = tb * 16 + (lane & 15), c = (E8 ? ks : 2 * ks) + (lane >> 4);
        uint32_t r[4];
        ldsm4(kd + row * RB + swz<CH>(row, c) * 16, r);
        if (E8) {
#pragma unroll
          for (int y = 0; y < Y; ++y) {
            uint32_t ka[4];
            widen4<EL, false>(r[2 * y], ka[0], ka[2]);
            widen4<EL, false>(r[2 * y + 1], ka[1], ka[3]);
#pragma unroll
            for (int n = 0; n < NG; ++n) mma<false>(sc[tb][n], ka, qb[y][n][0], qb[y][n][1]);
          }
        } else {
#pragma unroll
          for (int n = 0; n < NG; ++n) mma<MB>(sc[tb][n], r, qb[0][n][0], qb[0][n][1]);
        }
      }
    }
    // ---- softmax step, in powers of two ----
    if (p.a.softcap > 0.f) {
#pragma unroll
      for (int tb = 0; tb < TB; ++tb)
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            sc[tb][n][x] = kLog2e * p.a.softcap * tanhf(sc[tb][n][x] * qs[n][x & 1] * (BS ? ks[tb][x >> 1] : 1.f) / p.a.softcap);
    } else {
#pragma unroll
      for (int tb = 0; tb < TB; ++tb)
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) sc[tb][n][x] = sc[tb][n][x] * qs[n][x & 1] * (BS ? ks[tb][x >> 1] : 1.f);
    }
    if (mask != (BT == 32 ? 0xffffffffu : 0xffffu)) {
#pragma unroll
      for (int tb = 0; tb < TB; ++tb)
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (!((mask >> (tb * 16 + hr + 8 * (x >> 1))) & 1)) sc[tb][n][x] = -INFINITY;
    }
    float mx[NG][2], base[NG][2];
    bool grew = false;
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v = m[n][h];
#pragma unroll
        for (int tb = 0; tb < TB; ++tb) v = fmaxf(v, fmaxf(sc[tb][n][h], sc[tb][n][2 + h]));
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
        mx[n][h] = v;
        base[n][h] = v == -INFINITY ? 0.f : v - kUp;
        grew |= v != m[n][h];
      }
    // Block scales: the sums are in units of the least power of two that holds the
    // largest scale so far, since weights of 2^15 times a scale overflow where the result
    // does not.  It rises with the maximum's step (with a check at each product the
    // kernel took 7 to 17 % longer).
    const float own_vs = BS ? vscale[lane % BT] : 0.f;
    if (BS) grew |= own_vs > unit;
    if (__any_sync(0xffffffffu, grew)) {
      float down = 1.f;
      if (BS) {
        // (scales are ordered as their bits)
        const float most = unit_of(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(own_vs, unit)))));
        down = unit * inverse_of(most);
        unit = most;
      }
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float f = exp2_fast(m[n][h] - (mx[n][h] == -INFINITY ? 0.f : mx[n][h]));
          const float fo = BS ? f * down : f;
          l[n][h] *= f;
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            o[n][i][h] *= fo;
            o[n][i][2 + h] *= fo;
          }
          m[n][h] = mx[n][h];
        }
    }
#pragma unroll
    for (int tb = 0; tb < TB; ++tb)
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          sc[tb][n][x] = exp2_fast(sc[tb][n][x] - base[n][x & 1]);
          l[n][x & 1] += sc[tb][n][x];
        }
    const bool same = BS && pl.even && mask == (BT == 32 ? 0xffffffffu : 0xffffu);  // (no masked token's zero)
    // Block scales: a weight enters with its token's scale as a part of the
    // sixteen tokens' largest, which the FP32 sums take in.  Where they share
    // one there is nothing to do for it.
    float high[TB];
    if (BS) {
      if (same) {
#pragma unroll
        for (int tb = 0; tb < TB; ++tb) high[tb] = vscale[tb * 16];
      } else {
#pragma unroll
        for (int tb = 0; tb < TB; ++tb) {
          const float vs[2] = {vscale[tb * 16 + hr], vscale[tb * 16 + hr + 8]};
          high[tb] = fmaxf(vs[0], vs[1]);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) high[tb] = fmaxf(high[tb], __shfl_xor_sync(0xffffffffu, high[tb], d));
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            // (NaN scales stay NaN)
            const float part = vs[y] == high[tb] ? 1.f : vs[y] / high[tb];
#pragma unroll
            for (int n = 0; n < NG; ++n) sc[tb][n][2 * y] *= part, sc[tb][n][2 * y + 1] *= part;
          }
        }
      }
    }
    // ---- O^T += V^T P^T ----
#pragma unroll
    for (int tb = 0; tb < TB; ++tb) {
      const float part = BS ? high[tb] * inverse_of(unit) : 1.f;
      uint32_t hi[NG][2], lo[NG][2];
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float s0 = sc[tb][n][2 * y], s1 = sc[tb][n][2 * y + 1];
          const uint32_t w = MB ? pack_bf16(s0, s1) : pack_f16(s0, s1);
          hi[n][y] = transpose8(w);
          if (MB) {
            lo[n][y] = transpose8(pack_bf16(s0 - __uint_as_float(w << 16), s1 - __uint_as_float(w & 0xffff0000u)));
          } else {
            const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w));
            lo[n][y] = transpose8(pack_f16(s0 - h.x, s1 - h.y));
          }
        }
#pragma unroll
      for (int i = 0; i < KS; i += E8 ? 2 : 1) {  // 16 dims a product
        if (!FULL && uint32_t(i * 16) >= D) break;
        uint32_t r[4];
        if (E8) {
          // tokens 0 .. 7 and 8 .. 15 of one 16-byte piece, then of the next
          const uint32_t row = tb * 16 + (lane & 15);
          ldsm4t(vd + row * RB + swz<CH>(row, i + (lane >> 4)) * 16, r);
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            // bytes (dim 2n, 2n + 1) of two tokens -> dim 2n of both, dim 2n + 1 of both
            uint32_t va[4];
            widen4<EL, true>(r[2 * y], va[0], va[1]);
            widen4<EL, true>(r[2 * y + 1], va[2], va[3]);
#pragma unroll
            for (int n = 0; n < NG; ++n) {
              if (BS) {
                float some[4] = {};
                mma<false>(some, va, hi[n][0], hi[n][1]);
                mma<false>(some, va, lo[n][0], lo[n][1]);
#pragma unroll
                for (int x = 0; x < 4; ++x) o[n][i + y][x] += some[x] * part;
              } else {
                mma<false>(o[n][i + y], va, hi[n][0], hi[n][1]);
                mma<false>(o[n][i + y], va, lo[n][0], lo[n][1]);
              }
            }
          }
        } else {
          // dims 0 .. 7 and 8 .. 15 of tokens 0 .. 7, then of tokens 8 .. 15
          const uint32_t row = tb * 16 + (lane >> 4) * 8 + (lane & 7);
          ldsm4t(vd + row * RB + swz<CH>(row, 2 * i + ((lane >> 3) & 1)) * 16, r);
#pragma unroll
          for (int n = 0; n < NG; ++n) {
            mma<MB>(o[n][i], r, hi[n][0], hi[n][1]);
            mma<MB>(o[n][i], r, lo[n][0], lo[n][1]);
          }
        }
      }
    }
    const bool last = cu.block + 1 == cu.blocks;
    if (last || t + 1 == b) finish(t);
    if (t + 1 < b) {
      step(cu);
      if (last) begin();
    }
  }
  asm volatile("cp.async.wait_group 0;\n" ::: "memory");
  if constexpr (CL) {
    cluster_barrier();
    // warp `me`: a head, and every other run of 32 dims (or further apart)
    const uint32_t runs = 32 / cl_heads, head = me % cl_heads, run0 = me / cl_heads;
    if (run0 < runs) {
      auto piece = [&](uint32_t k) { return smem_addr(smem) + (k % kWarps) * Sh::WARP; };
      float m1 = -INFINITY, l1 = 0.f, u1 = kLeastUnit;
      if (uint32_t(lane) < share.workers) {
        const uint32_t stat = piece(lane) + (pl.heads * DP + Sh::ST * head) * 4;
        m1 = ld_cluster(stat, lane / kWarps);
        l1 = ld_cluster(stat + 4, lane / kWarps);
        if (BS) u1 = ld_cluster(stat + 8, lane / kWarps);
      }
      float base = m1;
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) base = fmaxf(base, __shfl_xor_sync(0xffffffffu, base, d));
      base = base == -INFINITY ? 0.f : base;
      const float w = uint32_t(lane) < share.workers ? exp2f(m1 - base) : 0.f;
      float lt = l1 * w;
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) lt += __shfl_xor_sync(0xffffffffu, lt, d);
      float u = 1.f, wo = w;  // of block scales' sums: the largest unit, and the weight in units of it
      if (BS) {
        u = u1;
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) u = fmaxf(u, __shfl_xor_sync(0xffffffffu, u, d));
        wo *= u1 * inverse_of(u);
      }
      const bool some = lt > 0.f || lt != lt;
      const float f = some ? (BS ? u : E8 && p.c.v_scale ? p.c.v_scale[cl_unit / pl.chunks] : 1.f) / lt : 0.f;
      uint16_t* out = static_cast<uint16_t*>(p.a.out) + cl_seq * p.a.out_stride[0] + (cl_head0 + head) * p.a.out_stride[1];
      for (uint32_t d0 = run0 * 32; d0 < D; d0 += runs * 32) {
        const uint32_t d = d0 + lane;
        float v[32];
#pragma unroll
        for (uint32_t k = 0; k < 32; ++k)
          v[k] = k < share.workers && d < D ? ld_cluster(piece(k) + (head * DP + d) * 4, k / kWarps) : 0.f;
        float acc = 0.f;
#pragma unroll
        for (uint32_t k = 0; k < 32; ++k) {
          const float wk = __shfl_sync(0xffffffffu, wo, k);
          acc += k < share.workers ? v[k] * wk : 0.f;
        }
        if (d < D) store16(bf, out + d, some ? acc * f : 0.f);
      }
      if (run0 == 0 && lane == 0 && p.a.lse)
        p.a.lse[uint64_t(cl_seq) * p.a.q_heads + cl_head0 + head] = some ? (base + log2f(lt) - kUp) * kLn2 : -INFINITY;
    }
    cluster_barrier();  // no CTA ends while another reads its shared memory
  }
}

constexpr int JT = 256;                // threads of a join
constexpr uint32_t kJoin = JT / 32;    // workers whose units a CTA joins, and parts that a warp joins alone

// Joins the pieces of the units that workers 8 x .. 8 x + 7 begin, for query
// head y of their chunk.  A unit of few parts takes one warp, all its loads in
// flight at once; of the eight at most one has more than eight (its parts are
// successive workers), and that one takes the whole CTA: the parts' weights
// once in shared memory, then each warp every eighth part, lanes the dims;
// last the warps' sums in order.
template <bool BS>
__global__ void __launch_bounds__(JT, 3) kv_join_kernel(const AttendArgs p, const AttendPlan pl, float up) {
  extern __shared__ float weight[];  // [workers]
  __shared__ __align__(16) float so[JT / 32][256];
  __shared__ float red[3][JT / 32];
  __shared__ int4 big;
  __shared__ uint32_t big_at;
  constexpr float kLn2 = 0.69314718055994531f;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t head = blockIdx.y, DP = pl.pad_dim, D = p.c.head_dim;
  const bool bf = p.a.type == XKSV_BF16;
  const uint32_t group = p.a.q_heads / p.c.kv_heads, st = pl.heads * DP + (BS ? 3 : 2) * head;
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
  auto scale_of = [&](const Unit& u, float l, float unit) {  // no weight at all: zeros
    return l > 0.f || l != l ? (!BS && p.c.v_scale ? p.c.v_scale[u.kv_head] : unit) / l : 0.f;
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
      float m[kJoin], w[kJoin], in[kJoin], l = 0.f, base = -INFINITY;
#pragma unroll
      for (uint32_t k = 0; k < kJoin; ++k) {
        m[k] = k < uint32_t(j.z) ? slot(i, k)[st] : -INFINITY;
        w[k] = k < uint32_t(j.z) ? slot(i, k)[st + 1] : 0.f;
        in[k] = BS && k < uint32_t(j.z) ? slot(i, k)[st + 2] : kLeastUnit;
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
      float most = 1.f;
      if (BS) {
        most = kLeastUnit;
#pragma unroll
        for (uint32_t k = 0; k < kJoin; ++k) most = fmaxf(most, in[k]);
#pragma unroll
        for (uint32_t k = 0; k < kJoin; ++k) m[k] *= in[k] * inverse_of(most);
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
      const float f = scale_of(u, l, most);
      const bool some = l > 0.f || l != l;
      uint16_t* out = out_of(j, u);
#pragma unroll
      for (int x = 0; x < 8; ++x)
        if (x * 32 + lane < D) store16(bf, out + x * 32 + lane, some ? acc[x] * f : 0.f);
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
  float mt = -INFINITY, most = BS ? kLeastUnit : 1.f;
  for (uint32_t k = threadIdx.x; k < parts; k += JT) {
    weight[k] = slot(many, k)[st];
    mt = fmaxf(mt, weight[k]);
    if (BS) most = fmaxf(most, slot(many, k)[st + 2]);
  }
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) {
    mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, d));
    if (BS) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
  }
  if (lane == 0) {
    red[0][warp] = mt;
    if (BS) red[2][warp] = most;
  }
  __syncthreads();
  for (int w = 0; w < JT / 32; ++w) {
    mt = fmaxf(mt, red[0][w]);
    if (BS) most = fmaxf(most, red[2][w]);
  }
  const float base = mt == -INFINITY ? 0.f : mt;
  float l = 0.f;
  for (uint32_t k = threadIdx.x; k < parts; k += JT) {
    weight[k] = exp2f(weight[k] - base);
    l += slot(many, k)[st + 1] * weight[k];
    if (BS) weight[k] *= slot(many, k)[st + 2] * inverse_of(most);
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
  const float f = scale_of(u, l, most);
  const bool some = l > 0.f || l != l;
  uint16_t* out = out_of(jm, u);
  for (uint32_t d = threadIdx.x; d < D; d += JT) {
    float x = 0.f;
    for (int w = 0; w < JT / 32; ++w) x += so[w][d];
    store16(bf, out + d, some ? x * f : 0.f);
  }
  if (threadIdx.x == 0) put_lse(jm, u, base, l);
}

int pad_dim(uint32_t d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

template <bool MB, int EL, int DP, int NG, bool FULL, bool CL>
cudaError_t launch_attend(const AttendArgs& p, const AttendPlan& pl, cudaStream_t st) {
  using Sh = Shape<EL, DP, NG>;
  static_assert(8 * NG * (DP + Sh::ST) * 4 <= Sh::WARP, "a piece fits the warp's shared memory");
  auto kernel = kv_attend_kernel<MB, EL, DP, NG, FULL, CL>;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = opt_in_smem(kernel, Sh::CTA, done);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(CL ? pl.clusters * kCluster : (pl.warps + kWarps - 1) / kWarps);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = Sh::CTA;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kCluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CL ? 2 : 1;
  const cudaError_t f = cudaLaunchKernelEx(&cfg, kernel, p, pl);
  if (f != cudaSuccess || CL) return f;
  cfg.gridDim = dim3((pl.warps + kJoin - 1) / kJoin, pl.heads);
  cfg.blockDim = dim3(JT);
  cfg.dynamicSmemBytes = pl.warps * sizeof(float);
  return cudaLaunchKernelEx(&cfg, kv_join_kernel<Sh::BS>, p, pl, MB ? 0.f : 15.f);
}

template <bool MB, int EL, int DP, int NG>
cudaError_t launch_full(const AttendArgs& p, const AttendPlan& pl, cudaStream_t st) {
  if (pl.clusters)
    return p.c.head_dim == DP ? launch_attend<MB, EL, DP, NG, true, true>(p, pl, st)
                              : launch_attend<MB, EL, DP, NG, false, true>(p, pl, st);
  return p.c.head_dim == DP ? launch_attend<MB, EL, DP, NG, true, false>(p, pl, st)
                            : launch_attend<MB, EL, DP, NG, false, false>(p, pl, st);
}
template <bool MB, int EL, int DP>
cudaError_t launch_heads(const AttendArgs& p, const AttendPlan& pl, cudaStream_t st) {
  return pl.heads <= 8 ? launch_full<MB, EL, DP, 1>(p, pl, st) : launch_full<MB, EL, DP, 2>(p, pl, st);
}
template <bool MB, int EL>
cudaError_t launch_dim(const AttendArgs& p, const AttendPlan& pl, cudaStream_t st) {
  switch (pl.pad_dim) {
    case 64: return launch_heads<MB, EL, 64>(p, pl, st);
    case 128: return launch_heads<MB, EL, 128>(p, pl, st);
    default: return launch_heads<MB, EL, 256>(p, pl, st);
  }
}

template <int EL, int NG>
void shape_of(uint32_t dp, uint32_t* block, uint32_t* per_sm) {
  using A = Shape<EL, 64, NG>;
  using B = Shape<EL, 128, NG>;
  using C = Shape<EL, 256, NG>;
  *block = dp == 64 ? A::BT : dp == 128 ? B::BT : C::BT;
  *per_sm = dp == 64 ? A::PER_SM : dp == 128 ? B::PER_SM : C::PER_SM;
}

}  // namespace
}  // namespace xksv
