// Gated delta rule, tensor-core family: what a chunk needs before the states are known.
//
//   gates:  b_i (running sum of g), exp(b_i), exp(b_end - b_i), beta_i, exp(b_end)
//   P_ij = scale exp(b_i - b_j) (q_i . k_j)  for j <= i
//   T - I,  T = (I + A)^-1,  A_ij = exp(b_i - b_j) (k_i . k_j) beta_j  for j < i
//
// One block per (chunk, group, up to kHeads of its heads).  K K^t and Q K^t are one M = 128 MMA chain,
// [K; Q] K^t, read once into registers (a thread owns one of the 128 rows) and scaled per head.  The
// inverse of the unit lower triangular matrix is substitution: the four diagonal 16 x 16 blocks by columns in
// fp32, the blocks below them one block diagonal after the other with 16 x 16 products on the warp's tensor cores
// (16 products a head; tf32 pairs, so still 2^-21).  (A product of powers of A would be fewer steps but loses
// everything when keys repeat and the powers grow binomially.)
// Decays take the approximate exponential (2 + 1.2 |b_i - b_j| ulp of fp32 of a number that falls as fast: below the 2^-16 of the
// pairs that P and T are stored as).
// Bound: latency of these short dependent phases; four blocks a SM overlap them (4 x 4096 tokens of 32 heads: 135 us, 6 of
// them for the 64-bit gate sums; five blocks, whose registers spill, 138 against 130 before those).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "delta_host.h"
#include "delta_tc.cuh"
#include "ema_scan_dispatch.h"

namespace emab {
namespace delta {
namespace {

constexpr int kHeads = 2;   // heads of a group per block
constexpr int kThreads = 128;
constexpr int kLd = 68;     // row stride of the fp32 matrices: 16-byte rows, conflict-free fragment reads
constexpr int kWLd = 20;    // row stride of a warp's 16 x 16 block
struct Matrices {  // over the operand tiles, once their product is read
  float A[kC][kLd];
  float T[kC][kLd];
  float W[4][16][kWLd];
};
struct Shared {
  GateSum b[kHeads][kC];
  float beta[kHeads][kC], key[kHeads][kC];  // key: exp(b_r - b_j), or 1 in a wide group
  uint32_t wide[kHeads];
  uint64_t full, mma;
  uint32_t taddr, fail;
};

__device__ __forceinline__ float4 ld4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ void st4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }

// c (16 x 16, two 8-column tiles) += a (16 x 16, row-major, stride lda) b (16 x 16, row-major, stride ldb) on the
// warp's tensor cores: each fp32 operand as two tf32 pieces, three products, 2^-21 of the sum.
__device__ __forceinline__ void block_product(float (&c)[2][4], const float* a, int lda, const float* b, int ldb) {
  const int lane = threadIdx.x & 31, r = lane >> 2, q = lane & 3;
  auto split = [](float x, uint32_t& hi, uint32_t& lo) {
    hi = __float_as_uint(x) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi));
  };
  auto mma = [](float (&d)[4], const uint32_t (&x)[4], uint32_t y0, uint32_t y1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(y0), "r"(y1));
  };
#pragma unroll
  for (int k = 0; k < 16; k += 8) {
    uint32_t ah[4], al[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) split(a[(r + 8 * (i & 1)) * lda + k + q + 4 * (i >> 1)], ah[i], al[i]);
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      uint32_t bh[2], bl[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) split(b[(k + q + 4 * i) * ldb + 8 * n + r], bh[i], bl[i]);
      mma(c[n], ah, bh[0], bh[1]);
      mma(c[n], ah, bl[0], bl[1]);
      mma(c[n], al, bh[0], bh[1]);
    }
  }
}
__device__ __forceinline__ void store_block(float* d, int ld, const float (&c)[2][4], float sign) {
  const int lane = threadIdx.x & 31, r = lane >> 2, q = 2 * (lane & 3);
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    *reinterpret_cast<float2*>(d + r * ld + 8 * n + q) = make_float2(sign * c[n][0], sign * c[n][1]);
    *reinterpret_cast<float2*>(d + (r + 8) * ld + 8 * n + q) = make_float2(sign * c[n][2], sign * c[n][3]);
  }
}

// T = (I + A)^-1 for the strictly lower triangular A, in 16 x 16 blocks: the diagonal ones by substitution, then one
// block diagonal after the other, T_IJ = -T_II sum_{J <= K < I} A_IK T_KJ.  All 128 threads; blocks above the
// diagonal are left as they are.
__device__ __forceinline__ void unit_lower_inverse(Matrices& s) {
  const int t = threadIdx.x, warp = t >> 5;
  if (t < kC) {  // a column of a diagonal block each
    const int r0 = t & ~15, c = t & 15;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = i == c ? 1.f : 0.f;
#pragma unroll
      for (int j4 = 0; j4 < i; j4 += 4) {
        const float4 a = ld4(&s.A[r0 + i][r0 + j4]);
        v = fmaf(-a.x, x[j4], v);
        if (j4 + 1 < i) v = fmaf(-a.y, x[j4 + 1], v);
        if (j4 + 2 < i) v = fmaf(-a.z, x[j4 + 2], v);
        if (j4 + 3 < i) v = fmaf(-a.w, x[j4 + 3], v);
      }
      x[i] = v;
      s.T[r0 + i][r0 + c] = v;
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int d = 1; d < 4; ++d) {
    if (warp < 4 - d) {
      const int I = 16 * (warp + d), J = 16 * warp;
      float c[2][4] = {};
#pragma unroll 1
      for (int K = J; K < I; K += 16) block_product(c, &s.A[I][K], kLd, &s.T[K][J], kLd);
      store_block(&s.W[warp][0][0], kWLd, c, 1.f);
      __syncwarp();
      float x[2][4] = {};
      block_product(x, &s.T[I][I], kLd, &s.W[warp][0][0], kWLd);
      store_block(&s.T[I][J], kLd, x, -1.f);
    }
    __syncthreads();
  }
}

// 16 numbers of row `row`, columns c0 .. c0 + 15, as hi and lo chunks of an image.
__device__ __forceinline__ void store_row16(char* hi, char* lo, int row, int c0, const float (&v)[16]) {
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) split2(make_float2(v[8 * q + 2 * k], v[8 * q + 2 * k + 1]), h[k], l[k]);
    const uint32_t at = tc::chunk_off(row, c0 / 8 + q);
    *reinterpret_cast<uint4*>(hi + at) = make_uint4(h[0], h[1], h[2], h[3]);
    *reinterpret_cast<uint4*>(lo + at) = make_uint4(l[0], l[1], l[2], l[3]);
  }
}

template <int K>
constexpr int kOperands = (K / 64) * 128 * 128 > static_cast<int>(sizeof(Matrices)) ? (K / 64) * 128 * 128
                                                                                     : (sizeof(Matrices) + 127) / 128 * 128;

template <int K>
__global__ void __launch_bounds__(kThreads, 4) prep_tc_kernel(const __grid_constant__ CUtensorMap mk,
                                                           const __grid_constant__ CUtensorMap mq, const Params p,
                                                           const TcBuffers w, uint32_t* status) {
  extern __shared__ __align__(1024) unsigned char smem[];
  constexpr int kReg = 128 * 128;  // 64 key rows, then 64 query rows
  Matrices& m = *reinterpret_cast<Matrices*>(smem);
  Shared& s = *reinterpret_cast<Shared*>(smem + kOperands<K>);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int hpg = p.H / p.G, splits = (hpg + kHeads - 1) / kHeads;
  const int slot = blockIdx.x, gr = blockIdx.y / splits, h0 = gr * hpg + (blockIdx.y % splits) * kHeads;
  const int h1 = min(h0 + kHeads, (gr + 1) * hpg);
  int n, tok;
  Seq q;
  if (!chunk_at(p, slot, &n, &q, &tok)) return;
  const int have = min(kC, q.len - tok);
  if (tid == 0) {
    mbar_init(&s.full, 1);
    mbar_init(&s.mma, 1);
    s.fail = 0;
    fence_mbar_init();
    mbar_arrive_expect_tx(&s.full, (K / 64) * kReg);
    for (int r = 0; r < K / 64; ++r) {
      tma_load_4d(smem + r * kReg, &mk, &s.full, 64 * r, gr, q.t0 + tok, q.b);
      tma_load_4d(smem + r * kReg + kTile, &mq, &s.full, 64 * r, gr, q.t0 + tok, q.b);
    }
  }
  if (warp == 0) tc::tmem_alloc(&s.taddr, 64);
  if (warp >= 2 && h0 + warp - 2 < h1) {  // gates of one head
    const int e = warp - 2, h = h0 + e;
    float g[2], be[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int t = 2 * lane + k;
      const long long at = (static_cast<long long>(q.b) * p.L + q.t0 + tok + t) * p.H + h;
      g[k] = t < have ? clamp_gate(p.g[at]) : 0.f;
      be[k] = t < have ? p.beta[at] : 0.f;
    }
    const double run = gate_scan(g, lane), left = run - g[1];
    const double end = __shfl_sync(0xffffffffu, run, 31);
    const double first = __shfl_sync(0xffffffffu, left, lane & ~7);  // b of the 16-token group's first token
    const double last = __shfl_sync(0xffffffffu, run, lane | 7);
    const bool wide = fabs(first - last) > kWideSpan;
    const uint32_t wb = __ballot_sync(0xffffffffu, wide);
    float* rec = w.gates + (static_cast<long long>(slot) * p.H + h) * kGateFloats;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const double b = k == 0 ? left : run;
      const GateSum bs = gate_sum(b);
      const int t = 2 * lane + k;
      s.b[e][t] = bs;
      s.beta[e][t] = be[k];
      const float key = wide ? 1.f : expf(static_cast<float>(first - b)), tail = expf(static_cast<float>(end - b));
      s.key[e][t] = key;
      rec[kGateE + t] = -expf(bs.hi);
      rec[kGateW + t] = be[k] * tail;
      rec[kGateBeta + t] = be[k];
      rec[kGateB + t] = bs.hi;
      rec[kGateBLo + t] = bs.lo;
      rec[kGateKey + t] = key;
      rec[kGateTail + t] = tail;
    }
    if (lane == 0) {
      rec[kGateEnd] = expf(static_cast<float>(end));
      s.wide[e] = wb;  // bit 8 g: group g
      rec[kGateWide] = __uint_as_float(wb);
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tb = s.taddr;
  if (warp == 0) {
    const bool ok = mbar_wait_bounded(&s.full, 0, status, 32);
    if (have < kC && p.cu != nullptr) {  // rows of the next sequence
      zero_rows(smem, K / 64, kReg, have);
      zero_rows(smem + kTile, K / 64, kReg, have);
      fence_proxy_async_smem();
    }
    __syncwarp();
    if (lane == 0) {
      if (ok) {
        const uint64_t d = tc::smem_desc_sw128(smem_u32(smem), 16, 1024);
        const uint32_t id = tc::idesc_bf16(128, 64, false, false);
#pragma unroll
        for (int k = 0; k < K / 16; ++k) {
          const uint64_t at = static_cast<uint64_t>(((k >> 2) * kReg + (k & 3) * 32) >> 4);
          tc::mma_bf16(tb, d + at, d + at, id, k > 0);
        }
        tc::mma_commit(&s.mma);
      } else {
        s.fail = 1;
        mbar_arrive(&s.mma);
      }
    }
    __syncwarp();
  }
  const bool ok = mbar_wait_bounded(&s.mma, 0, status, 32);
  tc::fence_after_sync();
  float x[64];  // row tid of [K K^t; Q K^t]
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    float v[16];
    tc::tmem_ld16(tc::tmem_at(tb, 32 * warp, 16 * c), v);
    tc::tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 16; ++i) x[16 * c + i] = v[i];
  }
  tc::fence_before_sync();
  const int failed = __syncthreads_or(!ok || s.fail != 0);
  if (failed && warp == 0) {  // the copies and the product in flight end before the block does
    mbar_wait_bounded(&s.full, 0, status);
    mbar_wait_bounded(&s.mma, 0, status);
    __syncwarp();
  }
  if (warp == 0) {
    tc::tmem_relinquish();
    tc::tmem_dealloc(tb, 64);
  }
  if (failed) return;  // the status word tells the host

  const int i = tid & 63;
  for (int h = h0; h < h1; ++h) {
    const long long ch = static_cast<long long>(slot) * p.H + h;
    const int e = h - h0;
    const GateSum bi = s.b[e][i];
    const uint32_t wide = s.wide[e];
    char* hi = w.P + ch * 2 * kTile;
#pragma unroll
    for (int g = 0; g < 4; ++g) {  // 16 columns of the row of A (first 64 threads) or of P
      float f[16];
      if ((wide >> (8 * g)) & 1u) {
#pragma unroll
        for (int c = 0; c < 16; ++c) f[c] = __expf(bi - s.b[e][16 * g + c]);
      } else {
        const float rf = __expf(bi - s.b[e][16 * g]);
#pragma unroll
        for (int c = 0; c < 16; c += 4) {
          const float4 k4 = ld4(&s.key[e][16 * g + c]);
          f[c] = rf * k4.x, f[c + 1] = rf * k4.y, f[c + 2] = rf * k4.z, f[c + 3] = rf * k4.w;
        }
      }
      if (tid < kC) {
#pragma unroll
        for (int c = 0; c < 16; ++c) f[c] = 16 * g + c < i ? x[16 * g + c] * f[c] * s.beta[e][16 * g + c] : 0.f;
#pragma unroll
        for (int c = 0; c < 16; c += 4) st4(&m.A[i][16 * g + c], make_float4(f[c], f[c + 1], f[c + 2], f[c + 3]));
      } else {
#pragma unroll
        for (int c = 0; c < 16; ++c) f[c] = 16 * g + c <= i ? p.scale * x[16 * g + c] * f[c] : 0.f;
        store_row16(hi, hi + kTile, i, 16 * g, f);
      }
    }
    __syncthreads();
    unit_lower_inverse(m);
    {
      const int r = tid >> 1, c0 = (tid & 1) * 32;
      char* to = w.T + ch * 2 * kTile;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        float v[16];
#pragma unroll
        for (int c = 0; c < 16; c += 4) {
          const float4 f = ld4(&m.T[r][c0 + 16 * g + c]);
          v[c] = f.x, v[c + 1] = f.y, v[c + 2] = f.z, v[c + 3] = f.w;
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = c0 + 16 * g + k < r ? v[k] : 0.f;
        store_row16(to, to + kTile, r, c0 + 16 * g, v);
      }
    }
    __syncthreads();
  }
}

template <int K>
cudaError_t launch(const CUtensorMap& mk, const CUtensorMap& mq, const Params& p, const TcBuffers& w, uint32_t* status, cudaStream_t st) {
  static unsigned long long mask = 0;
  const int bytes = kOperands<K> + static_cast<int>(sizeof(Shared));
  const cudaError_t e = static_cast<cudaError_t>(
      ensure_smem_attr(reinterpret_cast<const void*>(prep_tc_kernel<K>), bytes, &mask));
  if (e != cudaSuccess) return e;
  const int hpg = p.H / p.G;
  prep_tc_kernel<K><<<dim3(p.slots, p.G * ((hpg + kHeads - 1) / kHeads)), kThreads, bytes, st>>>(mk, mq, p, w,
                                                                                              status);
  return cudaGetLastError();
}

}  // namespace

cudaError_t tc_prep(const CUtensorMap& mk, const CUtensorMap& mq, const Params& p, const TcBuffers& w, uint32_t* status, cudaStream_t st) {
  if (p.slots == 0) return cudaSuccess;
  return p.K == 64 ? launch<64>(mk, mq, p, w, status, st) : launch<128>(mk, mq, p, w, status, st);
}

}  // namespace delta
}  // namespace emab
