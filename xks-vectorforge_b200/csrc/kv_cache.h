// Launchers of the paged key/value cache's kernels.
#pragma once
#include <cuda_runtime.h>

#include "xksv_cuda.h"

namespace xksv {

struct AppendArgs {
  xksv_kv_append_args a;
  xksv_kv_desc c;
  int* status;
};
cudaError_t launch_kv_append(const AppendArgs& p, int sms, cudaStream_t st);

// The same into a cache with block scales.
struct AppendBlocksArgs {
  xksv_kv_append_args a;
  xksv_kv_desc c;
  int* status;
  xksv_kv_blocks b;
  uint32_t chunk;  // tokens whose runs a CTA takes
};
cudaError_t launch_kv_append_blocks(const AppendBlocksArgs& p, int sms, cudaStream_t st);

struct AttendArgs {
  xksv_kv_attend_args a;
  xksv_kv_desc c;
  int* status;
  // pieces of units that several workers share: per slot (two a worker) the
  // sums [heads][dims] and the heads' maxima and weights; per worker what the
  // join has to do
  float* slots;
  int4* joins;
  xksv_kv_blocks b;  // block 0: no block scales
};
// Warps that share the work of a call, and the workspace they need.
struct AttendPlan {
  uint32_t warps, chunks, heads, pad_dim;  // query-head chunks per KV head, heads per chunk, padded head_dim
  int page_shift, block_shift;  // log2 page_size and of a scale's tokens, -1 when that is no power of two
  bool even;                    // sixteen tokens from a multiple of sixteen on share a scale
  uint32_t clusters;  // clusters of CTAs, one a unit, that join by themselves (0: the split over all warps)
  uint64_t slot_floats, joins_off, bytes;
};
AttendPlan kv_attend_plan(const xksv_kv_desc& c, const xksv_kv_blocks& b, uint64_t seqs, uint32_t q_heads, uint64_t table_cols, int sms);
cudaError_t launch_kv_attend(const AttendArgs& p, const AttendPlan& plan, cudaStream_t st);
cudaError_t launch_kv_attend_blocks(const AttendArgs& p, const AttendPlan& plan, cudaStream_t st);

}  // namespace xksv
