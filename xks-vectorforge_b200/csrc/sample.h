// Launcher of the sampling kernel.
#pragma once
#include <cuda_runtime.h>

#include "xksv_cuda.h"

namespace xksv {

// Temperatures other than 0 lie in this range.
constexpr float kSampleColdest = 1e-6f, kSampleHottest = 1e6f;

struct SampleArgs {
  xksv_sample_args a;
  uint32_t cluster;   // CTAs that share a row
  uint32_t resident;  // the row fits their shared memory
  uint32_t held_off;  // where in it
};
cudaError_t launch_sample(const SampleArgs& p, int sms, cudaStream_t st);

}  // namespace xksv
