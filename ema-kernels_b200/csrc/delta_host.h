// Buffers between the chunked gated delta rule's kernels, and the kernel families' host entry points.
#pragma once

#include <cuda_runtime.h>

#include "delta_common.cuh"

namespace emab {
namespace delta {

// All per (chunk slot, head), slot-major.
struct Buffers {
  // fp32 family
  float* T;    // 64 x 64
  float* P;    // 64 x 64
  float* S0;   // headdim x dstate: the state entering the chunk (kept for a backward, else null)
  float* E;    // 64 x headdim (the same)
  float* dU;   // 64 x headdim
  float* dX;   // 64 x headdim
  float* dS1;  // headdim x dstate
};

cudaError_t simt_fwd(const Params& p, const Buffers& w, int dtype, cudaStream_t st);
cudaError_t simt_bwd(const Params& p, const Buffers& w, int dtype, cudaStream_t st);

}  // namespace delta
}  // namespace emab
