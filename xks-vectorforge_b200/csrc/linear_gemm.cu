// Linear layer of a prompt: y[tokens, rows] = epilogue(x W^T) on the 5th-
// generation tensor cores, W decoded into a BF16 scratch before.
//
// Bound: the tensor cores (2 tokens rows cols operations) or the operands' way
// from L2, about 64 bytes a clock and SM: a 128 x 256 tile multiplies a
// 64-column slice in 512 clocks and reads 48 KB for it.  Two CTAs of a pair
// (PAIR) share a 256 x tn tile: each brings 128 tokens and half of the weight
// rows, 32 KB a slice, and tcgen05.mma cta_group::2 reads both.  A persistent
// CTA (or pair) per SM takes tiles; within it
//   * one thread loads 64-column slices of x and W by TMA (128-byte swizzled
//     rows, zero past the edges), two to a stage, into a ring of stages,
//   * one thread (of the pair's first CTA) issues tcgen05.mma kind::f16,
//     M = 128 (256) tokens, N = tn, K = 16, into one of two TMEM accumulators,
//   * eight warps read the other accumulator (a lane is a token, its registers
//     consecutive rows of y), apply bias, activation, factor and residual in
//     FP32 and write y: the epilogue of a tile runs behind the products of the next.
// The tensor cores add in FP32 but cut what falls below the sum's last place,
// always towards zero: 1.1e-9 of the result a column, 1.6e-5 at 14336.  A BF16
// result is rounded a hundred times coarser.  For FP32 results (EXACT) an
// accumulator holds 512 columns only, and the epilogue's warps add its sums to
// theirs, in registers, rounded to nearest: relative error 4.8e-7 at every
// length (1024 columns: 1.0e-6), with the decode 150 us against 141 at 77
// tokens, 272 against 244 at 2048 (4096 x 14336).
// gemm_plan chooses tn and the pair by a model of both costs.  Tokens as the
// MMA's rows rather than weight rows: y is token-major, so a lane's results
// are contiguous.
// Every wait is bounded: on a timeout the CTA sets an error bit, lets its
// copies and MMAs drain, frees its TMEM and returns.
#include <cuda.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <mutex>

#include "kernels.h"
#include "linear_epilogue.cuh"
#include "tcgen05.cuh"

namespace xksv {
namespace {

constexpr int GM = 128;          // tokens of a tile
constexpr int GK = 64;           // columns of a slice: 128-byte rows
constexpr int EPI = 256;         // epilogue threads: two warps for each 32 tokens
constexpr int GTHREADS = 64 + EPI;  // producer and MMA warps besides
// Slices of a stage.  The threads that copy and multiply wait once a stage, and
// those waits limited tiles of few rows: 4096 x 14336 with 77 tokens 75 us a
// slice at a time, 55 us two; with 2048 tokens and FP32 results 193, 182 us.
constexpr uint32_t SL = 2;
constexpr uint32_t kExact = 4;  // stages (512 columns) of an accumulator, EXACT
constexpr uint32_t kMaxStages = 8;
constexpr uint32_t kABytes = GM * GK * 2;
constexpr size_t kRing = 220 * 1024;  // stages' shared memory

struct GemmShared {
  uint64_t full[kMaxStages], empty[kMaxStages], tfull[2], tempty[2];
  uint32_t tmem;
  int abort_flag;
};

struct GemmArgs {
  Epilogue e;
  uint64_t row0;  // row of Y that the segment's first weight row gives
  uint32_t batch, rows, cols, tn, stages, tmem_cols;
  int* status;
};

// (Cluster scope: the pair's CTAs arrive on each other's barriers.)
__device__ __forceinline__ bool wait_or_abort(uint32_t bar, uint32_t parity, const volatile int* abort_flag) {
  for (uint32_t i = 0; i < kSpin; ++i) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return true;
    if ((i & 255) == 255 && *abort_flag) return false;
    if (i > 64) __nanosleep(32);
  }
  return false;
}

__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
}
// Box of `map` at (x, y) into dst; bytes counted on bar.
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, uint32_t x, uint32_t y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
// The same, its bytes counted on a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, uint32_t x, uint32_t y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
// A shared-memory address of this CTA in CTA `rank` of its cluster.
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n barrier.cluster.wait.aligned;\n" ::: "memory");
}
template <bool PAIR>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if (!PAIR) {
    umma_bf16(d, a, b, idesc, accumulate);
    return;
  }
  const uint32_t z = 0;
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(z)
      : "memory");
}
// Arrives on a barrier (of both CTAs) when the MMAs issued so far are done.
template <bool PAIR>
__device__ __forceinline__ void commit(uint32_t bar) {
  if (PAIR)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(bar),
                 "h"(uint16_t(3))
                 : "memory");
  else
    umma_commit(bar);
}

// Shared-memory descriptor of a K-major operand of 128-byte swizzled rows:
// eight rows are 1024 bytes (SBO), layout type 2 in bits 61-63.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr) {
  return uint64_t((addr >> 4) & 0x3FFFu) | (uint64_t(1) << 16) | (uint64_t(64) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
}

template <bool PAIR, bool EXACT>
__global__ void __launch_bounds__(GTHREADS, 1)
    linear_gemm_kernel(const __grid_constant__ CUtensorMap mx, const __grid_constant__ CUtensorMap mw, const GemmArgs a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ GemmShared S;
  constexpr uint32_t CTAS = PAIR ? 2 : 1, TM = GM * CTAS;  // tokens of a tile
  uint8_t* ring = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t rank = 0;
  if (PAIR) asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(rank));
  const uint32_t bn = a.tn / CTAS;  // weight rows that this CTA brings
  const uint32_t w_bytes = bn * GK * 2, stage_bytes = SL * (kABytes + w_bytes);
  const uint32_t mt = (a.batch + TM - 1) / TM, nt = (a.rows + a.tn - 1) / a.tn, tiles = mt * nt;
  const uint32_t ksteps = (a.cols + SL * GK - 1) / (SL * GK);
  const uint32_t kpart = EXACT ? kExact : ksteps;  // stages of an accumulator
  const uint32_t first = blockIdx.x / CTAS, stride = gridDim.x / CTAS;  // this CTA's (pair's) tiles
  if (warp == 1) {
    if (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_addr(&S.tmem)), "r"(a.tmem_cols)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_addr(&S.tmem)), "r"(a.tmem_cols)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
  }
  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < a.stages; ++s) {
      mbar_init(smem_addr(&S.full[s]), 1);
      mbar_init(smem_addr(&S.empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_addr(&S.tfull[b]), 1);
      mbar_init(smem_addr(&S.tempty[b]), EPI * CTAS);
    }
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    S.abort_flag = 0;
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();  // the other CTA's barriers are there
  tc_fence_after();
  const uint32_t tmem = S.tmem;
  bool ok = true;
  // the start above runs behind the decode's end; its weight is complete here
  asm volatile("griddepcontrol.wait;\n" ::: "memory");

  if (warp == 0) {
    if (lane == 0) {
      // stage and round of the next copy, stepped along: a division for each
      // would take this thread longer than the MMAs
      uint32_t n = 0, s = 0, round = 0;
      for (uint32_t t = first; t < tiles && ok; t += stride) {
        const uint32_t m0 = t % mt * TM + rank * GM, n0 = t / mt * a.tn + rank * bn;
        for (uint32_t k = 0; k < ksteps; ++k, ++n) {
          const uint32_t dst = smem_addr(ring) + s * stage_bytes;
          ok = wait_or_abort(smem_addr(&S.empty[s]), (round & 1) ^ 1, &S.abort_flag);
          if (!ok) break;
          // the first CTA's barrier counts both CTAs' bytes (the second's may
          // come before it is armed: its phase waits for the arming)
          if (rank == 0) expect_bytes(smem_addr(&S.full[s]), CTAS * stage_bytes);
          if (PAIR) {
            const uint32_t bar = in_cta(smem_addr(&S.full[s]), 0);
#pragma unroll
            for (uint32_t q = 0; q < SL; ++q) {
              tma_load_pair(dst + q * kABytes, &mx, (SL * k + q) * GK, m0, bar);
              tma_load_pair(dst + SL * kABytes + q * w_bytes, &mw, (SL * k + q) * GK, n0, bar);
            }
          } else {
            const uint32_t bar = smem_addr(&S.full[s]);
#pragma unroll
            for (uint32_t q = 0; q < SL; ++q) {
              tma_load(dst + q * kABytes, &mx, (SL * k + q) * GK, m0, bar);
              tma_load(dst + SL * kABytes + q * w_bytes, &mw, (SL * k + q) * GK, n0, bar);
            }
          }
          if (++s == a.stages) {
            s = 0;
            ++round;
          }
        }
      }
      if (!ok) S.abort_flag = 1;
      // every copy has landed before the CTA (the pair) ends
      if (rank == 0)
        for (uint32_t i = n > a.stages ? n - a.stages : 0; i < n; ++i)
          if (!mbar_wait(smem_addr(&S.full[i % a.stages]), (i / a.stages) & 1)) ok = false;
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = umma_idesc_bf16(TM, a.tn);
      uint32_t n = 0, ai = 0;  // stages multiplied, accumulators begun
      uint32_t s = 0, round = 0;
      const uint64_t desc0 = desc_sw128(smem_addr(ring));
      for (uint32_t t = first; t < tiles && ok; t += stride) {
        for (uint32_t k0 = 0; k0 < ksteps && ok; k0 += kpart, ++ai) {
          const uint32_t buf = ai & 1, d = tmem + buf * (a.tmem_cols / 2);
          const uint32_t parts = min(kpart, ksteps - k0);
          ok = wait_or_abort(smem_addr(&S.tempty[buf]), ((ai >> 1) & 1) ^ 1, &S.abort_flag);
          if (!ok) break;
          tc_fence_after();
          for (uint32_t k = 0; k < parts; ++k, ++n) {
            ok = wait_or_abort(smem_addr(&S.full[s]), round & 1, &S.abort_flag);
            if (!ok) break;
            tc_fence_after();
            // (addresses below 256 KB: a descriptor's address field does not overflow)
            const uint64_t da = desc0 + ((s * stage_bytes) >> 4), db = da + ((SL * kABytes) >> 4);
#pragma unroll
            for (uint32_t q = 0; q < SL; ++q)
#pragma unroll
              for (uint32_t j = 0; j < GK / 16; ++j)  // 32 bytes further along the rows
                mma_f16<PAIR>(d, da + q * (kABytes >> 4) + 2 * j, db + q * (w_bytes >> 4) + 2 * j, idesc, (k | q | j) != 0);
            commit<PAIR>(smem_addr(&S.empty[s]));
            if (++s == a.stages) {
              s = 0;
              ++round;
            }
          }
          if (ok) commit<PAIR>(smem_addr(&S.tfull[buf]));
        }
      }
      if (!ok) S.abort_flag = 1;
      // the MMAs issued are done before TMEM is freed: they complete in
      // order, and the last slice's commit follows them all
      if (n && !mbar_wait(smem_addr(&S.empty[(n - 1) % a.stages]), ((n - 1) / a.stages) & 1)) ok = false;
    }
  } else {
    const uint32_t ti0 = (warp & 3) * 32;            // this warp's TMEM lanes
    const uint32_t half = uint32_t(warp - 2) >> 2;   // 32-row groups half, half + 2, ... of a tile
    uint32_t ai = 0;
    for (uint32_t t = first; t < tiles && ok; t += stride) {
      const uint32_t m0 = t % mt * TM + rank * GM, n0 = t / mt * a.tn;
      const uint64_t b = m0 + ti0 + lane;
      const uint32_t top = min(a.tn, a.rows - n0);
      const auto store = [&](uint32_t c, float* v) {
        if (b >= a.batch) return;
#pragma unroll
        for (int g = 0; g < 4; ++g) epilogue_store8(a.e, b, a.row0 + n0 + c + 8 * g, v + 8 * g, int(top) - int(c + 8 * g));
      };
      float sum[EXACT ? 4 : 1][32];  // EXACT: of the tile's accumulators so far
      for (uint32_t k0 = 0; k0 < ksteps; k0 += kpart, ++ai) {
        const uint32_t buf = ai & 1, acc = tmem + (ti0 << 16) + buf * (a.tmem_cols / 2);
        ok = wait_or_abort(smem_addr(&S.tfull[buf]), (ai >> 1) & 1, &S.abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        if (EXACT) {
#pragma unroll
          for (uint32_t g = 0; g < 8; ++g) {
            const uint32_t c = 32 * (g & ~1u) + 32 * half + 16 * (g & 1);
            if (c < top) {
              float r[16];
              tmem_ld16(acc + c, r);
              float* z = sum[EXACT ? g / 2 : 0] + 16 * (g & 1);
#pragma unroll
              for (int x = 0; x < 16; ++x) z[x] = r[x] + (k0 ? z[x] : 0.f);
            }
          }
        } else {
          for (uint32_t c = 32 * half; c < top; c += 64) {
            uint32_t r[32];
            tmem_ld32(acc + c, r);
#pragma unroll
            for (int x = 0; x < 32; ++x) sum[0][x] = __uint_as_float(r[x]);
            store(c, sum[0]);
          }
        }
        tc_fence_before();
        if (PAIR)
          arrive_cluster(in_cta(smem_addr(&S.tempty[buf]), 0));
        else
          mbar_arrive(smem_addr(&S.tempty[buf]));
      }
      if (EXACT && ok)
#pragma unroll
        for (uint32_t g = 0; g < 4; ++g) {
          const uint32_t c = 32 * (2 * g + half);
          if (c < top) store(c, sum[EXACT ? g : 0]);
        }
    }
    if (!ok) S.abort_flag = 1;
  }
  if (!ok && lane == 0) atomicOr(a.status, kStatusInternal);
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();  // neither CTA ends (or frees TMEM) while the other's work needs it
  if (warp == 1) {
    tc_fence_after();
    if (PAIR)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(a.tmem_cols) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(a.tmem_cols) : "memory");
  }
}

// x's columns [0, cols) as BF16 rows of `pitch` elements (zeros behind), for
// rows that TMA cannot address.
__global__ void linear_rows_kernel(const uint16_t* __restrict__ x, uint64_t stride, uint64_t batch, uint64_t cols,
                                   uint64_t pitch, uint16_t* __restrict__ out) {
  for (uint64_t i = blockIdx.x * uint64_t(blockDim.x) + threadIdx.x; i < batch * pitch; i += uint64_t(gridDim.x) * blockDim.x) {
    const uint64_t b = i / pitch, c = i - b * pitch;
    out[i] = c < cols ? x[b * stride + c] : uint16_t(0);
  }
}

// Tile and pairing: the waves of tiles, each slice of a tile costing the
// slower of its products (2 tn clocks) and its copies (64 bytes a clock), a
// tile 2000 clocks besides (start and epilogue).
struct GemmPlan {
  bool pair;
  uint32_t tn;
};
GemmPlan gemm_plan(uint32_t batch, uint32_t rows, uint32_t cols, int sms) {
  GemmPlan best{false, 256};
  uint64_t least = ~uint64_t(0);
  for (const bool pair : {false, true}) {
    const uint32_t ctas = pair ? 2 : 1;
    const uint64_t mt = (batch + GM * ctas - 1) / (GM * ctas);
    // the MMA's N: steps of 16, of 32 for a pair
    for (uint32_t n = 256; n >= 32; n -= 16 * ctas) {
      const uint64_t tiles = mt * ((rows + n - 1) / n), waves = (tiles * ctas + sms - 1) / sms;
      const uint64_t slice = std::max<uint64_t>(2 * n, (kABytes + n / ctas * GK * 2) / 64);
      const uint64_t cost = waves * (slice * ((cols + GK - 1) / GK) + 2000);
      if (cost < least) {
        least = cost;
        best = GemmPlan{pair, n};
      }
    }
  }
  return best;
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
  static std::once_flag once;
  static EncodeTiled fn = nullptr;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiled>(p);
  });
  return fn;
}

// BF16 [rows, cols], rows `pitch` elements apart, read in boxes of 64 columns by `box` rows.
bool tensor_map(CUtensorMap* m, const void* base, uint64_t rows, uint64_t cols, uint64_t pitch, uint32_t box) {
  const EncodeTiled fn = encode_tiled();
  if (!fn) return false;
  const cuuint64_t dims[2] = {cols, rows}, strides[1] = {pitch * 2};
  const cuuint32_t boxes[2] = {GK, box}, steps[2] = {1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, boxes, steps,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

bool linear_rows_direct(const void* x, uint64_t stride, uint64_t xoff) {
  return ((reinterpret_cast<uintptr_t>(x) + xoff * 2) | stride * 2) % 16 == 0;
}

cudaError_t launch_linear_rows(const void* x, uint64_t stride, uint64_t batch, uint64_t cols, uint64_t pitch, void* out,
                               cudaStream_t st) {
  const uint64_t n = batch * pitch;
  linear_rows_kernel<<<uint32_t(std::min<uint64_t>((n + 255) / 256, 8192)), 256, 0, st>>>(
      static_cast<const uint16_t*>(x), stride, batch, cols, pitch, static_cast<uint16_t*>(out));
  return cudaGetLastError();
}

cudaError_t launch_linear_gemm(const void* w, uint32_t rows, uint32_t cols, const void* x, uint64_t x_pitch, uint32_t batch,
                               uint64_t row0, const Epilogue& e, int* status, int sms, cudaStream_t st) {
  GemmArgs a{};
  a.e = e;
  a.row0 = row0;
  a.batch = batch;
  a.rows = rows;
  a.cols = cols;
  a.status = status;
  const GemmPlan plan = gemm_plan(batch, rows, cols, sms);
  const uint32_t ctas = plan.pair ? 2 : 1;
  a.tn = plan.tn;
  const uint32_t stage = SL * (kABytes + a.tn / ctas * GK * 2);
  a.stages = std::min<uint32_t>(kMaxStages, uint32_t(kRing / stage));
  a.tmem_cols = 32;
  while (a.tmem_cols < 2 * ((a.tn + 31) / 32 * 32)) a.tmem_cols *= 2;
  CUtensorMap mx, mw;
  if (!tensor_map(&mx, x, batch, cols, x_pitch, GM) || !tensor_map(&mw, w, rows, cols, cols, a.tn / ctas)) return cudaErrorInvalidValue;
  const size_t smem = size_t(a.stages) * stage + 1024;
  // one CTA an SM, whatever the tile: its TMEM columns are its own
  const size_t ask = std::max<size_t>(smem, 120 * 1024);
  auto kernel = e.y_f32 ? plan.pair ? linear_gemm_kernel<true, true> : linear_gemm_kernel<false, true>
                        : plan.pair ? linear_gemm_kernel<true, false> : linear_gemm_kernel<false, false>;
  static std::atomic<uint64_t> done[2][2] = {};
  const cudaError_t err = opt_in_smem(kernel, kRing + 1024, done[e.y_f32][plan.pair]);
  if (err != cudaSuccess) return err;
  const uint64_t tiles = uint64_t((batch + GM * ctas - 1) / (GM * ctas)) * ((rows + a.tn - 1) / a.tn);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(uint32_t(std::min<uint64_t>(tiles, uint64_t(sms) / ctas)) * ctas);
  cfg.blockDim = dim3(GTHREADS);
  cfg.dynamicSmemBytes = ask;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, mx, mw, a);
}

}  // namespace xksv
