// What the chunked gated delta rule's kernels share: the sequence and chunk indices, the parameters of a
// call, and where the buffers between the kernels lie.
//
// A sequence is cut into chunks of kC = 64 tokens from its own start.  Inside a chunk, with b the
// running sum of g (clamped at -100), Gam_ij = exp(b_i - b_j) for j <= i, S0 the state entering it:
//
//   A_ij = Gam_ij (k_i . k_j) beta_j  (j < i),   T = (I + A)^-1
//   X_i = v_i - exp(b_i) S0 k_i,   E = T X,   U = beta E
//   o_i = exp(b_i) scale S0 q_i + sum_{j <= i} P_ij U_j,   P_ij = scale Gam_ij (q_i . k_j)
//   S1 = exp(b_end) S0 + sum_j U_j (exp(b_end - b_j) k_j)^T
//
// and backwards, from dO and dS1 (the gradient of S1):
//
//   dU_j = sum_{i >= j} P_ij dO_i + exp(b_end - b_j) dS1 k_j,   dX = T^t (beta dU),   dV = dX
//   dS0 = exp(b_end) dS1 + sum_i (scale exp(b_i) dO_i) q_i^T - sum_i (exp(b_i) dX_i) k_i^T
//   N_ij = scale Gam_ij (dO_i . U_j),  F_ij = Gam_ij (dX_i . E_j) for j < i,  M_ij = -F_ij beta_j
//   dQ = N K + scale exp(b) dO S0,   dK = (M + M^t) K + N^t Q - exp(b) dX S0 + exp(b_end - b) U dS1
//   dbeta_j = dU_j . E_j - sum_{i > j} F_ij (k_i . k_j)
//   dg_t = sum_{j < t <= i} Z_ij + sum_{i >= t} r_i + sum_{j < t} c_j + exp(b_end) <dS1, S0>,
//     Z_ij = N_ij (q_i . k_j) + M_ij (k_i . k_j),
//     r_i = exp(b_i) (scale dO_i . S0 q_i - dX_i . S0 k_i),  c_j = exp(b_end - b_j) U_j . dS1 k_j
//
// (dg_t gathers every pair whose decay spans token t; the sums over pairs are taken as they are, not as
// differences of running totals, so nothing cancels that does not cancel in dg itself.)
//
// Chunk slots: sequence n of a plain batch has slots [n ceil(L / 64), ...); sequence n of a packed call, starting
// at token t, has slots [t / 64 + n, ...) -- disjoint whatever the lengths, known without a prefix
// sum, and at most L / 64 + nseq of them.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "delta_b200.h"
#include "ema_common.cuh"

namespace emab {
namespace delta {

constexpr int kC = 64;              // tokens of a chunk
constexpr float kMinGate = -100.f;  // exp(-100) = 4e-44: a reset; keeps sums and their differences finite
// (not fmaxf, which would make a reset of a gate that is no number)
__device__ __forceinline__ float clamp_gate(float g) { return g < kMinGate ? kMinGate : g; }

// The running sum of a chunk's gates is taken in 64 bits and kept as two floats: a decay between two tokens is a difference of
// such sums, and in 32 bits it would have the digits of what steep gates before both have summed to (one reset in four
// tokens: 3e-5 of o).
struct GateSum {
  float hi, lo;
};
__device__ __forceinline__ GateSum gate_sum(double b) {
  const float hi = static_cast<float>(b);
  return GateSum{hi, static_cast<float>(b - hi)};
}
__device__ __forceinline__ float operator-(GateSum a, GateSum b) { return (a.hi - b.hi) + (a.lo - b.lo); }
// Inclusive sums of the warp's 64 gates, two a lane: up to the lane's second one.
__device__ __forceinline__ double gate_scan(const float (&g)[2], int lane) {
  double run = static_cast<double>(g[0]) + g[1];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double v = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += v;
  }
  return run;
}

struct View {
  long long b, t, h;  // element strides of batch, token, head / group
};

struct Params {
  int B, L, H, G, V, K, nseq;
  int nc;        // chunks of a sequence (plain batch)
  int slots;     // chunk slots of the call
  float scale;
  const void* q;  View vq;
  const void* k;  View vk;
  const void* v;  View vv;
  const float* g;
  const float* beta;
  const int32_t* cu;
  const float* s0;
  void* o;        View vo;
  float* s1;
  const void* dout; View vd;
  const float* ds1;
  void* dq;       View vdq;
  void* dk;       View vdk;
  void* dv;       View vdv;
  float* dg;
  float* dbeta;
  float* ds0;
};

// One sequence: its batch row, first token, length and first chunk slot.
struct Seq {
  int b, t0, len, slot;
};
__device__ __forceinline__ Seq seq_at(const Params& p, int n) {
  if (p.cu == nullptr) return Seq{n, 0, p.L, n * p.nc};
  const int t0 = min(max(p.cu[n], 0), p.L);
  const int t1 = min(max(p.cu[n + 1], t0), p.L);
  return Seq{0, t0, t1 - t0, t0 / kC + n};
}
// The sequence of a chunk slot and the chunk's first token in it; false for a slot that holds none.
__device__ __forceinline__ bool chunk_at(const Params& p, int slot, int* n, Seq* s, int* tok) {
  if (p.cu == nullptr) {
    *n = slot / p.nc;
  } else {  // the last sequence whose first slot is not behind this one (first slots rise strictly)
    int lo = 0, hi = p.nseq;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (min(max(p.cu[mid], 0), p.L) / kC + mid <= slot) lo = mid;
      else hi = mid;
    }
    *n = lo;
  }
  *s = seq_at(p, *n);
  *tok = (slot - s->slot) * kC;
  return *tok >= 0 && *tok < s->len;
}

template <class T>
__device__ __forceinline__ const T* row_of(const void* base, const View& v, int b, int t, int h) {
  return static_cast<const T*>(base) + b * v.b + t * v.t + h * v.h;
}
template <class T>
__device__ __forceinline__ T* row_of(void* base, const View& v, int b, int t, int h) {
  return static_cast<T*>(base) + b * v.b + t * v.t + h * v.h;
}

}  // namespace delta
}  // namespace emab
