// The attention's kernels for caches with block scales (a file of their own for
// the compiler's time).
#include "kv_attend_kernel.cuh"

namespace xksv {

cudaError_t launch_kv_attend_blocks(const AttendArgs& p, const AttendPlan& pl, cudaStream_t st) {
  return p.c.type == XKSV_INT8 ? launch_dim<false, ELInt8Blocks>(p, pl, st) : launch_dim<false, ELE4M3Blocks>(p, pl, st);
}

}  // namespace xksv
