// The chunked gated delta rule in fp32 on the CUDA cores: every element type and shape the entry points take.
// The formulas stand in delta_common.cuh.  Four kernels:
//
//   prep   (chunk, head): running gate sums, T and P of the chunk
//   fwd    (32 value channels, head, sequence): walks the chunks with its rows of the state
//   bwd    (the same, last chunk first): dU, dX, the state gradient at every chunk end
//   grads  (chunk, group): dq, dk summed over the group's heads, dg and dbeta
//
// All operands are staged in shared memory as fp32 with rows padded to an odd stride (no bank conflicts by
// row or by column); products are register tiles of 4 rows x every 16th column a thread.  Bound: the
// shared-memory reads of those products, and on few chunks the walks' chain (2 x 333 tokens of 4 heads of 64 x 64 in fp32:
// 125 and 115 us for 6 chunks, 20 us a chunk; preparation 46, gradients 123).  The tensor-core kernels serve bf16; this family
// serves fp32 and fp16 inputs (an fp16 number is a bf16 pair and an fp32 one three pieces, but no kernel stages them so).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "delta_common.cuh"
#include "delta_host.h"
#include "ema_scan_dispatch.h"

namespace emab {
namespace delta {
namespace simt {

constexpr int kThreads = 256;
constexpr int kVB = 32;        // value channels of a walking block
constexpr int kS = kC + 1;     // row stride of a 64 x 64 matrix in shared memory
constexpr int kVS = kVB + 1;   // of a 64 x 32 tile

// acc[i][j] += sum over kk < n of a(row0 + i, kk) b(kk, col + 16 j), operands through accessors.
template <int RM, int CN, class FA, class FB>
__device__ __forceinline__ void product(float (&acc)[RM][CN], int n, FA a, FB b) {
  const int r0 = (threadIdx.x >> 4) * RM, c0 = threadIdx.x & 15;
#pragma unroll 4
  for (int kk = 0; kk < n; ++kk) {
    float x[RM], y[CN];
#pragma unroll
    for (int i = 0; i < RM; ++i) x[i] = a(r0 + i, kk);
#pragma unroll
    for (int j = 0; j < CN; ++j) y[j] = b(kk, c0 + 16 * j);
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
      for (int j = 0; j < CN; ++j) acc[i][j] = fmaf(x[i], y[j], acc[i][j]);
  }
}
template <int RM, int CN>
__device__ __forceinline__ void zero(float (&acc)[RM][CN]) {
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int j = 0; j < CN; ++j) acc[i][j] = 0.f;
}
// f(row, column, value) over a thread's tile.
template <int RM, int CN, class F>
__device__ __forceinline__ void each(float (&acc)[RM][CN], F f) {
  const int r0 = (threadIdx.x >> 4) * RM, c0 = threadIdx.x & 15;
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int j = 0; j < CN; ++j) f(r0 + i, c0 + 16 * j, acc[i][j]);
}

// `rows` token rows from t (those at or past `end` as zeros), columns [c0, c0 + n) of which `have` exist.
template <class T>
__device__ __forceinline__ void load_rows(float* dst, int stride, const void* src, const View& v, int b, int t, int end,
                                          int h, int c0, int n, int have) {
  for (int i = threadIdx.x; i < kC * n; i += kThreads) {
    const int r = i / n, c = i - r * n;
    dst[r * stride + c] =
        (t + r < end && c0 + c < have) ? to_f32(row_of<T>(src, v, b, t + r, h)[c0 + c]) : 0.f;
  }
}
__device__ __forceinline__ void load_flat(float* dst, int stride, const float* src, int src_stride, int rows, int n,
                                          int have_rows) {
  for (int i = threadIdx.x; i < rows * n; i += kThreads) {
    const int r = i / n, c = i - r * n;
    dst[r * stride + c] = r < have_rows ? src[static_cast<long long>(r) * src_stride + c] : 0.f;
  }
}

// The chunk's gates: b (running sums), beta; both zero-extended past the sequence (b stays at its last value).
__device__ __forceinline__ void load_gates(const Params& p, const Seq& s, int tok, int h, GateSum* sb, float* sbeta) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    float g[2], be[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = tok + 2 * lane + i;
      const long long at = (static_cast<long long>(s.b) * p.L + s.t0 + t) * p.H + h;
      g[i] = t < s.len ? clamp_gate(p.g[at]) : 0.f;
      be[i] = t < s.len ? p.beta[at] : 0.f;
    }
    const double run = gate_scan(g, lane);
    sb[2 * lane] = gate_sum(run - g[1]);
    sb[2 * lane + 1] = gate_sum(run);
    sbeta[2 * lane] = be[0];
    sbeta[2 * lane + 1] = be[1];
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads) prep_kernel(const Params p, const Buffers w) {
  extern __shared__ float smem[];
  const int K = p.K, ks = K + 1;
  float* sk = smem;
  float* sq = sk + kC * ks;
  float* sa = sq + kC * ks;
  float* st = sa + kC * kS;
  GateSum* sb = reinterpret_cast<GateSum*>(st + kC * kS);
  float* sbeta = reinterpret_cast<float*>(sb + kC);
  const int slot = blockIdx.x, h = blockIdx.y, gr = h / (p.H / p.G);
  int n, tok;
  Seq s;
  if (!chunk_at(p, slot, &n, &s, &tok)) return;
  load_rows<T>(sk, ks, p.k, p.vk, s.b, s.t0 + tok, s.t0 + s.len, gr, 0, K, K);
  load_rows<T>(sq, ks, p.q, p.vq, s.b, s.t0 + tok, s.t0 + s.len, gr, 0, K, K);
  load_gates(p, s, tok, h, sb, sbeta);
  __syncthreads();
  const long long at = (static_cast<long long>(slot) * p.H + h) * kC * kC;
  float acc[4][4];
  zero(acc);
  product(acc, K, [&](int i, int kk) { return sq[i * ks + kk]; }, [&](int kk, int j) { return sk[j * ks + kk]; });
  each(acc, [&](int i, int j, float v) { w.P[at + i * kC + j] = j <= i ? p.scale * v * expf(sb[i] - sb[j]) : 0.f; });
  zero(acc);
  product(acc, K, [&](int i, int kk) { return sk[i * ks + kk]; }, [&](int kk, int j) { return sk[j * ks + kk]; });
  each(acc, [&](int i, int j, float v) { sa[i * kS + j] = j < i ? v * expf(sb[i] - sb[j]) * sbeta[j] : 0.f; });
  __syncthreads();
  if (threadIdx.x < kC) {  // column c of T by forward substitution
    const int c = threadIdx.x;
    for (int i = 0; i < kC; ++i) {
      float v = i == c ? 1.f : 0.f;
      for (int j = c; j < i; ++j) v = fmaf(-sa[i * kS + j], st[j * kS + c], v);
      st[i * kS + c] = v;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kC * kC; i += kThreads) w.T[at + i] = st[(i / kC) * kS + i % kC];
}

template <class T, int KJ>  // dstate = 16 KJ
__global__ void __launch_bounds__(kThreads) fwd_kernel(const Params p, const Buffers w) {
  extern __shared__ float smem[];
  const int K = p.K, ks = K + 1;
  float* sk = smem;
  float* sq = sk + kC * ks;
  float* ss = sq + kC * ks;       // state rows [32][K]
  float* st = ss + kVB * ks;
  float* sp = st + kC * kS;
  float* sx = sp + kC * kS;       // X, then U
  float* su = sx + kC * kVS;
  GateSum* sb = reinterpret_cast<GateSum*>(su + kC * kVS);
  float* sbeta = reinterpret_cast<float*>(sb + kC);
  const int v0 = blockIdx.x * kVB, h = blockIdx.y, n = blockIdx.z, gr = h / (p.H / p.G);
  const Seq s = seq_at(p, n);
  const int have = min(kVB, p.V - v0);
  const long long srow = ((static_cast<long long>(n) * p.H + h) * p.V + v0) * K;
  for (int i = threadIdx.x; i < kVB * K; i += kThreads) {
    const int r = i / K, c = i - r * K;
    ss[r * ks + c] = (p.s0 != nullptr && r < have) ? p.s0[srow + i] : 0.f;
  }
  for (int tok = 0; tok < s.len; tok += kC) {
    const long long ch = static_cast<long long>(s.slot + tok / kC) * p.H + h;
    __syncthreads();
    load_rows<T>(sk, ks, p.k, p.vk, s.b, s.t0 + tok, s.t0 + s.len, gr, 0, K, K);
    load_rows<T>(sq, ks, p.q, p.vq, s.b, s.t0 + tok, s.t0 + s.len, gr, 0, K, K);
    load_rows<T>(sx, kVS, p.v, p.vv, s.b, s.t0 + tok, s.t0 + s.len, h, v0, kVB, p.V);
    load_flat(st, kS, w.T + ch * kC * kC, kC, kC, kC, kC);
    load_flat(sp, kS, w.P + ch * kC * kC, kC, kC, kC, kC);
    load_gates(p, s, tok, h, sb, sbeta);
    if (w.S0 != nullptr)
      for (int i = threadIdx.x; i < have * K; i += kThreads)
        w.S0[ch * p.V * K + v0 * K + i] = ss[(i / K) * ks + i % K];
    __syncthreads();
    float acc[4][2];
    zero(acc);
    product(acc, K, [&](int i, int kk) { return sk[i * ks + kk]; }, [&](int kk, int j) { return ss[j * ks + kk]; });
    each(acc, [&](int i, int j, float v) { sx[i * kVS + j] = fmaf(-expf(sb[i].hi), v, sx[i * kVS + j]); });
    __syncthreads();
    zero(acc);
    product(acc, kC, [&](int i, int kk) { return st[i * kS + kk]; }, [&](int kk, int j) { return sx[kk * kVS + j]; });
    each(acc, [&](int i, int j, float v) {
      su[i * kVS + j] = sbeta[i] * v;
      if (w.E != nullptr && j < have) w.E[(ch * kC + i) * p.V + v0 + j] = v;
    });
    zero(acc);
    product(acc, K, [&](int i, int kk) { return sq[i * ks + kk]; }, [&](int kk, int j) { return ss[j * ks + kk]; });
    each(acc, [&](int i, int j, float& v) { v *= p.scale * expf(sb[i].hi); });
    __syncthreads();
    product(acc, kC, [&](int i, int kk) { return sp[i * kS + kk]; }, [&](int kk, int j) { return su[kk * kVS + j]; });
    each(acc, [&](int i, int j, float v) {
      if (tok + i < s.len && j < have)
        row_of<T>(p.o, p.vo, s.b, s.t0 + tok + i, h)[v0 + j] = from_f32<T>(v);
    });
    const GateSum end = sb[kC - 1];
    for (int i = threadIdx.x; i < kC * K; i += kThreads) {
      const int r = i / K, c = i - r * K;
      sk[r * ks + c] *= expf(end - sb[r]);
    }
    __syncthreads();
    float up[2][KJ];
    zero(up);
    product(up, kC, [&](int i, int kk) { return su[kk * kVS + i]; }, [&](int kk, int j) { return sk[kk * ks + j]; });
    const float dec = expf(end.hi);
    each(up, [&](int i, int j, float v) { ss[i * ks + j] = fmaf(dec, ss[i * ks + j], v); });
  }
  __syncthreads();
  if (p.s1 != nullptr)
    for (int i = threadIdx.x; i < have * K; i += kThreads) p.s1[srow + i] = ss[(i / K) * ks + i % K];
}

template <class T, int KJ>
__global__ void __launch_bounds__(kThreads) bwd_kernel(const Params p, const Buffers w) {
  extern __shared__ float smem[];
  const int K = p.K, ks = K + 1;
  float* sk = smem;
  float* sq = sk + kC * ks;
  float* ss = sq + kC * ks;       // state-gradient rows [32][K]
  float* st = ss + kVB * ks;
  float* sp = st + kC * kS;
  float* so = sp + kC * kS;       // dO
  float* su = so + kC * kVS;      // beta dU, then dX
  GateSum* sb = reinterpret_cast<GateSum*>(su + kC * kVS);
  float* sbeta = reinterpret_cast<float*>(sb + kC);
  const int v0 = blockIdx.x * kVB, h = blockIdx.y, n = blockIdx.z, gr = h / (p.H / p.G);
  const Seq s = seq_at(p, n);
  const int have = min(kVB, p.V - v0);
  const long long srow = ((static_cast<long long>(n) * p.H + h) * p.V + v0) * K;
  for (int i = threadIdx.x; i < kVB * K; i += kThreads) {
    const int r = i / K, c = i - r * K;
    ss[r * ks + c] = (p.ds1 != nullptr && r < have) ? p.ds1[srow + i] : 0.f;
  }
  for (int tok = (s.len - 1) / kC * kC; s.len > 0 && tok >= 0; tok -= kC) {
    const long long ch = static_cast<long long>(s.slot + tok / kC) * p.H + h;
    __syncthreads();
    load_rows<T>(sk, ks, p.k, p.vk, s.b, s.t0 + tok, s.t0 + s.len, gr, 0, K, K);
    load_rows<T>(sq, ks, p.q, p.vq, s.b, s.t0 + tok, s.t0 + s.len, gr, 0, K, K);
    load_rows<T>(so, kVS, p.dout, p.vd, s.b, s.t0 + tok, s.t0 + s.len, h, v0, kVB, p.V);
    load_flat(st, kS, w.T + ch * kC * kC, kC, kC, kC, kC);
    load_flat(sp, kS, w.P + ch * kC * kC, kC, kC, kC, kC);
    load_gates(p, s, tok, h, sb, sbeta);
    for (int i = threadIdx.x; i < have * K; i += kThreads)
      w.dS1[ch * p.V * K + v0 * K + i] = ss[(i / K) * ks + i % K];
    __syncthreads();
    const GateSum end = sb[kC - 1];
    float acc[4][2];
    zero(acc);
    product(acc, K, [&](int i, int kk) { return sk[i * ks + kk]; }, [&](int kk, int j) { return ss[j * ks + kk]; });
    each(acc, [&](int i, int j, float& v) { v *= expf(end - sb[i]); });
    product(acc, kC, [&](int i, int kk) { return sp[kk * kS + i]; }, [&](int kk, int j) { return so[kk * kVS + j]; });
    each(acc, [&](int i, int j, float v) {
      su[i * kVS + j] = sbeta[i] * v;
      if (j < have) w.dU[(ch * kC + i) * p.V + v0 + j] = v;
    });
    __syncthreads();
    zero(acc);
    product(acc, kC, [&](int i, int kk) { return st[kk * kS + i]; }, [&](int kk, int j) { return su[kk * kVS + j]; });
    __syncthreads();
    each(acc, [&](int i, int j, float v) {
      su[i * kVS + j] = v * -expf(sb[i].hi);
      so[i * kVS + j] *= p.scale * expf(sb[i].hi);
      if (j < have) {
        w.dX[(ch * kC + i) * p.V + v0 + j] = v;
        if (tok + i < s.len) row_of<T>(p.dv, p.vdv, s.b, s.t0 + tok + i, h)[v0 + j] = from_f32<T>(v);
      }
    });
    __syncthreads();
    float up[2][KJ];
    zero(up);
    product(up, kC, [&](int i, int kk) { return so[kk * kVS + i]; }, [&](int kk, int j) { return sq[kk * ks + j]; });
    product(up, kC, [&](int i, int kk) { return su[kk * kVS + i]; }, [&](int kk, int j) { return sk[kk * ks + j]; });
    const float dec = expf(end.hi);
    each(up, [&](int i, int j, float v) { ss[i * ks + j] = fmaf(dec, ss[i * ks + j], v); });
  }
  __syncthreads();
  if (p.ds0 != nullptr)
    for (int i = threadIdx.x; i < have * K; i += kThreads) p.ds0[srow + i] = ss[(i / K) * ks + i % K];
}

// Sum over the 16 threads that share a tile's rows.
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <class T, int KJ>
__global__ void __launch_bounds__(kThreads) grads_kernel(const Params p, const Buffers w) {
  extern __shared__ float smem[];
  const int K = p.K, ks = K + 1;
  float* sk = smem;
  float* sq = sk + kC * ks;
  float* s0 = sq + kC * ks;       // 32 rows of S0
  float* s1 = s0 + kVB * ks;      // of dS1
  float* so = s1 + kVB * ks;      // dO
  float* sx = so + kC * kVS;      // dX
  float* se = sx + kC * kVS;      // E
  float* sn = se + kC * kVS;      // N, then M + M^t
  float* sz = sn + kC * kS;       // Z, then M
  GateSum* sb = reinterpret_cast<GateSum*>(sz + kC * kS);
  float* sbeta = reinterpret_cast<float*>(sb + kC);
  float* sr = sbeta + kC;         // r_i
  float* sc = sr + kC;            // c_j
  float* sdb = sc + kC;           // dU_j . E_j
  float* sdot = sdb + kC;         // <dS1, S0> by warp
  const int slot = blockIdx.x, gr = blockIdx.y, hpg = p.H / p.G;
  int n, tok;
  Seq s;
  if (!chunk_at(p, slot, &n, &s, &tok)) return;
  load_rows<T>(sk, ks, p.k, p.vk, s.b, s.t0 + tok, s.t0 + s.len, gr, 0, K, K);
  load_rows<T>(sq, ks, p.q, p.vq, s.b, s.t0 + tok, s.t0 + s.len, gr, 0, K, K);
  __syncthreads();
  float kk[4][4], qk[4][4], dq[4][KJ], dk[4][KJ];
  zero(kk);
  zero(qk);
  zero(dq);
  zero(dk);
  product(kk, K, [&](int i, int c) { return sk[i * ks + c]; }, [&](int c, int j) { return sk[j * ks + c]; });
  product(qk, K, [&](int i, int c) { return sq[i * ks + c]; }, [&](int c, int j) { return sk[j * ks + c]; });
  const int ty4 = (threadIdx.x >> 4) * 4, tx = threadIdx.x & 15;
  for (int h = gr * hpg; h < (gr + 1) * hpg; ++h) {
    const long long ch = static_cast<long long>(slot) * p.H + h;
    __syncthreads();
    load_gates(p, s, tok, h, sb, sbeta);
    float fx[4][4], fn[4][4], r[4] = {}, c[4] = {}, db[4] = {}, dot = 0.f;
    zero(fx);
    zero(fn);
    for (int v0 = 0; v0 < p.V; v0 += kVB) {
      const int have = min(kVB, p.V - v0);
      __syncthreads();
      load_rows<T>(so, kVS, p.dout, p.vd, s.b, s.t0 + tok, s.t0 + s.len, h, v0, kVB, p.V);
      for (int i = threadIdx.x; i < kC * kVB; i += kThreads) {
        const int a = i / kVB, b = i - a * kVB;
        const long long at = (ch * kC + a) * p.V + v0 + b;
        sx[a * kVS + b] = b < have ? w.dX[at] : 0.f;
        se[a * kVS + b] = b < have ? w.E[at] : 0.f;
      }
      load_flat(s0, ks, w.S0 + ch * p.V * K + v0 * K, K, kVB, K, have);
      load_flat(s1, ks, w.dS1 + ch * p.V * K + v0 * K, K, kVB, K, have);
      __syncthreads();
      const GateSum end = sb[kC - 1];
      product(fx, kVB, [&](int i, int v) { return sx[i * kVS + v]; }, [&](int v, int j) { return se[j * kVS + v]; });
      product(fn, kVB, [&](int i, int v) { return so[i * kVS + v]; }, [&](int v, int j) { return se[j * kVS + v]; });
      float acc[4][KJ];
      zero(acc);
      product(acc, kVB, [&](int i, int v) { return so[i * kVS + v]; }, [&](int v, int j) { return s0[v * ks + j]; });
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f = p.scale * expf(sb[ty4 + i].hi);
#pragma unroll
        for (int j = 0; j < KJ; ++j) {
          const float x = f * acc[i][j];
          dq[i][j] += x;
          r[i] = fmaf(x, sq[(ty4 + i) * ks + tx + 16 * j], r[i]);
        }
      }
      zero(acc);
      product(acc, kVB, [&](int i, int v) { return sx[i * kVS + v]; }, [&](int v, int j) { return s0[v * ks + j]; });
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f = -expf(sb[ty4 + i].hi);
#pragma unroll
        for (int j = 0; j < KJ; ++j) {
          const float x = f * acc[i][j];
          dk[i][j] += x;
          r[i] = fmaf(x, sk[(ty4 + i) * ks + tx + 16 * j], r[i]);
        }
      }
      zero(acc);
      product(acc, kVB, [&](int i, int v) { return se[i * kVS + v]; }, [&](int v, int j) { return s1[v * ks + j]; });
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f = sbeta[ty4 + i] * expf(end - sb[ty4 + i]);
#pragma unroll
        for (int j = 0; j < KJ; ++j) {
          const float x = f * acc[i][j];
          dk[i][j] += x;
          c[i] = fmaf(x, sk[(ty4 + i) * ks + tx + 16 * j], c[i]);
        }
#pragma unroll
        for (int j = 0; j < kVB / 16; ++j) {
          const int v = tx + 16 * j;
          if (v < have) db[i] = fmaf(w.dU[(ch * kC + ty4 + i) * p.V + v0 + v], se[(ty4 + i) * kVS + v], db[i]);
        }
      }
      for (int i = threadIdx.x; i < kVB * K; i += kThreads)
        dot = fmaf(s0[(i / K) * ks + i % K], s1[(i / K) * ks + i % K], dot);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = row_sum(r[i]), b = row_sum(c[i]), d = row_sum(db[i]);
      if (tx == 0) {
        sr[ty4 + i] = a;
        sc[ty4 + i] = b;
        sdb[ty4 + i] = d;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if ((threadIdx.x & 31) == 0) sdot[threadIdx.x >> 5] = dot;
    __syncthreads();
    // N in sn, Z in sz; F kk (the column sums of dbeta) beside them afterwards
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int a = ty4 + i, b = tx + 16 * j;
        const float gam = b <= a ? expf(sb[a] - sb[b]) : 0.f;
        const float N = p.scale * gam * fn[i][j] * sbeta[b];
        const float F = b < a ? gam * fx[i][j] : 0.f;
        fx[i][j] = F;
        sn[a * kS + b] = N;
        sz[a * kS + b] = N * qk[i][j] - F * sbeta[b] * kk[i][j];
      }
    __syncthreads();
    product(dq, kC, [&](int i, int c2) { return sn[i * kS + c2]; }, [&](int c2, int j) { return sk[c2 * ks + j]; });
    product(dk, kC, [&](int i, int c2) { return sn[c2 * kS + i]; }, [&](int c2, int j) { return sq[c2 * ks + j]; });
    if (threadIdx.x < kC && tok + threadIdx.x < s.len) {
      const int t = threadIdx.x;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < kThreads / 32; ++i) sum += sdot[i];
      sum *= expf(sb[kC - 1].hi);
      for (int i = t; i < kC; ++i) {
        float x = sr[i];
        for (int j = 0; j < t; ++j) x += sz[i * kS + j];
        sum += x;
      }
      for (int j = 0; j < t; ++j) sum += sc[j];
      const long long at = (static_cast<long long>(s.b) * p.L + s.t0 + tok + t) * p.H + h;
      p.dg[at] = p.g[at] <= kMinGate ? 0.f : sum;  // a clamped gate has no gradient
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int a = ty4 + i, b = tx + 16 * j;
        sz[a * kS + b] = -fx[i][j] * sbeta[b];
        sn[a * kS + b] = fx[i][j] * kk[i][j];
      }
    __syncthreads();
    product(dk, kC, [&](int i, int c2) { return sz[i * kS + c2] + sz[c2 * kS + i]; },
            [&](int c2, int j) { return sk[c2 * ks + j]; });
    if (threadIdx.x < kC && tok + threadIdx.x < s.len) {
      const int j = threadIdx.x;
      float sum = sdb[j];
      for (int i = j + 1; i < kC; ++i) sum -= sn[i * kS + j];
      p.dbeta[(static_cast<long long>(s.b) * p.L + s.t0 + tok + j) * p.H + h] = sum;
    }
  }
  each(dq, [&](int i, int j, float v) {
    if (tok + i < s.len) row_of<T>(p.dq, p.vdq, s.b, s.t0 + tok + i, gr)[j] = from_f32<T>(v);
  });
  each(dk, [&](int i, int j, float v) {
    if (tok + i < s.len) row_of<T>(p.dk, p.vdk, s.b, s.t0 + tok + i, gr)[j] = from_f32<T>(v);
  });
}

int smem_prep(int K) { return (2 * kC * (K + 1) + 2 * kC * kS + 3 * kC) * 4; }
int smem_walk(int K) { return ((2 * kC + kVB) * (K + 1) + 2 * kC * kS + 2 * kC * kVS + 3 * kC) * 4; }
int smem_grads(int K) {
  return ((2 * kC + 2 * kVB) * (K + 1) + 3 * kC * kVS + 2 * kC * kS + 6 * kC + kThreads / 32) * 4;
}

template <class F>
cudaError_t opt_in(F fn, int bytes, unsigned long long* mask) {
  return static_cast<cudaError_t>(ensure_smem_attr(reinterpret_cast<const void*>(fn), bytes, mask));
}

template <class T, int KJ>
cudaError_t fwd_t(const Params& p, const Buffers& w, cudaStream_t st) {
  static unsigned long long m0 = 0, m1 = 0;
  // prep_kernel serves both dstates: the larger need
  cudaError_t e = opt_in(prep_kernel<T>, smem_prep(128), &m0);
  if (e == cudaSuccess) e = opt_in(fwd_kernel<T, KJ>, smem_walk(p.K), &m1);
  if (e != cudaSuccess) return e;
  if (p.slots > 0) prep_kernel<T><<<dim3(p.slots, p.H), kThreads, smem_prep(p.K), st>>>(p, w);
  fwd_kernel<T, KJ><<<dim3((p.V + kVB - 1) / kVB, p.H, p.nseq), kThreads, smem_walk(p.K), st>>>(p, w);
  return cudaGetLastError();
}
template <class T, int KJ>
cudaError_t bwd_t(const Params& p, const Buffers& w, cudaStream_t st) {
  static unsigned long long m0 = 0, m1 = 0;
  cudaError_t e = opt_in(bwd_kernel<T, KJ>, smem_walk(p.K), &m0);
  if (e == cudaSuccess) e = opt_in(grads_kernel<T, KJ>, smem_grads(p.K), &m1);
  if (e != cudaSuccess) return e;
  bwd_kernel<T, KJ><<<dim3((p.V + kVB - 1) / kVB, p.H, p.nseq), kThreads, smem_walk(p.K), st>>>(p, w);
  if (p.slots > 0) grads_kernel<T, KJ><<<dim3(p.slots, p.G), kThreads, smem_grads(p.K), st>>>(p, w);
  return cudaGetLastError();
}

}  // namespace simt

template <bool BWD>
static cudaError_t simt_any(const Params& p, const Buffers& w, int dtype, cudaStream_t st) {
  auto go = [&](auto zero) {
    using T = decltype(zero);
    if (p.K == 64) return BWD ? simt::bwd_t<T, 4>(p, w, st) : simt::fwd_t<T, 4>(p, w, st);
    return BWD ? simt::bwd_t<T, 8>(p, w, st) : simt::fwd_t<T, 8>(p, w, st);
  };
  if (dtype == EMA_DTYPE_F32) return go(float{});
  if (dtype == EMA_DTYPE_BF16) return go(__nv_bfloat16{});
  return go(__half{});
}
cudaError_t simt_fwd(const Params& p, const Buffers& w, int dtype, cudaStream_t st) {
  return simt_any<false>(p, w, dtype, st);
}
cudaError_t simt_bwd(const Params& p, const Buffers& w, int dtype, cudaStream_t st) {
  return simt_any<true>(p, w, dtype, st);
}

}  // namespace delta
}  // namespace emab
