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
  uint32_t held_off;  // where the row lies in their shared memory
};
cudaError_t launch_sample(const SampleArgs& p, int sms, cudaStream_t st);

}  // namespace xksv
