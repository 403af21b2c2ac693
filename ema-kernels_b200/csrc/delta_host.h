// Buffers between the chunked gated delta rule's kernels, and the kernel families' host entry points.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include "delta_common.cuh"
#include "delta_tc.cuh"

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

// bf16 on the tensor cores.  mk, mq: tiles of 64 tokens x 64 channels, 128-byte swizzle; mv: 64 tokens x headdim.
cudaError_t tc_prep(const CUtensorMap& mk, const CUtensorMap& mq, const Params& p, const TcBuffers& w, uint32_t* status,
                    cudaStream_t st);
cudaError_t tc_fwd_walk(const CUtensorMap& mk, const CUtensorMap& mq, const CUtensorMap& mv, const Params& p,
                        const TcBuffers& w, uint32_t* status, cudaStream_t st);

// (dout and dv as tiles of 64 tokens x 64 channels, 128-byte swizzle)
cudaError_t tc_bwd_walk(const CUtensorMap& mk, const CUtensorMap& mq, const CUtensorMap& mo, const Params& p,
                        const TcBuffers& w, uint32_t* status, cudaStream_t st);
cudaError_t tc_grads(const CUtensorMap& mk, const CUtensorMap& mq, const CUtensorMap& mo, const CUtensorMap& mdv,
                     const Params& p, const TcBuffers& w, uint32_t* status, cudaStream_t st);

}  // namespace delta
}  // namespace emab
