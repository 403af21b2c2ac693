// Gated delta rule, tensor-core family: the gradients of q, k, g and beta, chunk by chunk and in parallel, once the
// forward walk has left S0 and E and the backward walk dS1 and dX (formulas in delta_common.cuh).
//
// With lanes as token rows (M = 128: 64 query rows over 64 key rows, [dO; dX] and [Q; K]) one chain gives both
// 64 x 64 matrices of a head and one the products they are weighted with:
//   [dO; dX] E^t = [f; F'],   [Q; K] K^t = [qk; kk]
//   N = scale Gam f beta, M = -Gam F' beta (bf16 pairs, for dq and dk);  y = scale Gam f qk  over  -Gam F' kk
// with lanes as state columns (M = dstate) everything that ends in dq or dk:
//   a1 = S0^t dO^t, a2 = S0^t dX^t, a3 = dS1^t E^t, a4 = K^t N^t, a5 = K^t (M + M^t) + Q^t N
//   dq = scale exp(b) a1 + a4,   dk = -exp(b) a2 + beta w a3 + a5      (w_j = exp(b_end - b_j))
// and what the gates need, by transposed butterflies over the lanes of fp32 values:
//   dbeta_j = sum of y over its column + w_j k_j . a3_j
//   dg_t = sum over rows of (prefix of beta y up to t) + sum_{i >= t} r_i + sum_{j < t} c_j + exp(b_end) <dS1, S0>
// dg and dbeta are fp32 results, and sums that cancel: S0, dS1 and E enter as three bf16 pieces each, dX as two (dv and
// the rest), with all products of them down to 2^-24.  N and M are pairs: single bf16 would show beside the rounding of dk
// itself (2.0e-3 off where that alone is 1.7e-3), and dq's two terms cancel where keys repeat.
//
// One block a SM, persistent over (chunk, group) and the group's heads, whose dq and dk add up in registers.  E's pieces
// and dX's come as operand tiles, a head ahead.  S0 and dS1 come as fp32 images; warps 8-11 take them through registers in
// steps of 16 value channels (one MMA step), sum <dS1, S0> on the way and write the pieces to tensor memory as the left
// operand: a step whose left operand is there takes 14 + N / 2 cycles, from shared memory 48 + N / 2, and the pieces need
// neither 48 KB nor a proxy fence.  (Through shared memory, with E as fp32 too, the kernel took 700 us at 4 x 4096 x 32
// heads of 128 x 128; so, 569.)  Order of a head: F; the steps, and half-way the Q and K products of a new group, whose
// tiles arrive late; a4 and a5.  The next head's F runs under this one's epilogue of a1 to a3.  Bound: the staging warps, 8
// steps of about 1500 cycles of loads, turns, splits and hand-overs a head, near 17000 in all; the tensor pipe has 10000, the
// epilogues 10000, and the bytes (S0 and dS1 are 2 x 64 KB) would allow 9000.  Roles: warps 0-7 epilogues (lane quarter
// w % 4, column half w / 4), warps 8-11 staging, warp 12 the MMAs, warp 13 the loads, warp 14 dg and dbeta from the
// epilogues' sums.  The long loops are kept rolled where they can be: at twice the code the block ran at a third of the
// speed, waiting for instructions.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "delta_host.h"
#include "delta_tc.cuh"
#include "ema_scan_dispatch.h"

namespace emab {
namespace delta {
namespace {

constexpr int kEpi = 8, kAux = 4;
constexpr int kMma = 12, kLoad = 13, kGates = 14;  // (15 only fills its warpgroup)
constexpr int kThreads = 16 * 32;
constexpr int kRegEpi = 152, kRegAux = 128, kRegCtl = 80;
static_assert(2 * kRegEpi + kRegAux + kRegCtl == 4 * 128 && kRegAux >= 128 && kRegCtl <= 128, "register split");
constexpr int kRing = 2;
constexpr int kReg = 128 * 128;  // two 64-row tiles of 64 columns, one over the other

// tensor-memory columns
constexpr uint32_t cKQ = 0;     // [qk; kk]
constexpr uint32_t cF = 64;     // [f; F']; then a4
constexpr uint32_t cFX = 128;   // F' of dX lo (its rows alone); then a5
constexpr uint32_t cA = 192;    // a1, a2
constexpr uint32_t cA3 = 320;   // a3
constexpr uint32_t cRing = 384; // 16 value channels of S0, then of dS1, state columns as lanes: hi, mid, lo (8 columns each)
constexpr uint32_t kSlot = 48;

struct Bars {
  uint64_t qk_full, qk_empty, ox_full, ox_empty, ex_full[2], ex_empty[2];
  uint64_t s_full[kRing], s_empty[kRing];  // 16 value channels of S0 and dS1
  uint64_t g_full[2], g_empty[2];
  uint64_t f, a45;             // MMA groups done
  uint64_t nm, free_f, free_a; // N, M written; a4 and a5, a1 to a3 read
  uint64_t sums, fin;          // the epilogues' sums and <dS1, S0> written; dg, dbeta done with them
  uint64_t epi_sync;           // meeting of the epilogue warps (bounded, unlike a barrier instruction)
  uint64_t drain;
  uint32_t taddr, fail;
  int n_g, n_ex, n_ox, n_qk;  // loads issued
};

struct Small {
  float gate[2][kGateFloats];
  float y[4][kC], r[4][kC], R[4][kC], c[4][kC];  // column sums by lane quarter
  float base[128];                                // row sums of a row's first 32 columns
  float dot[kAux];
  Bars bar;
};

// Offsets from the 1024-byte aligned base.
template <int K, int VP>
struct Layout {
  static constexpr int ox = (K / 64) * kReg;             // after [Q; K]
  static constexpr int ex = ox + (VP / 64) * kReg;       // E hi, mid, dX lo, of this head and the next
  static constexpr int kEx = 3 * VP * 128;
  static constexpr int el = ex + 2 * kEx;                // E lo, of one head as dO and dv are
  static constexpr int nm = el + VP * 128;               // N hi, M hi, N lo, M lo: two tiles of 128 rows
  static constexpr int out = nm + 2 * kTile;             // over N lo: 32 rows of dq or dk on their way out
  static constexpr int small = nm + 4 * kTile;           // (32 x dstate bf16 fit a tile)
  static constexpr int bytes = small + static_cast<int>(sizeof(Small));
};

// Sums of 16 columns over the warp's 32 lanes: lane l gets column l / 2.
__device__ __forceinline__ float column_sums(float (&x)[16], int lane) {
#pragma unroll
  for (int o = 16, n = 8; n >= 1; o >>= 1, n >>= 1) {
    const bool up = (lane & o) != 0;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float give = up ? x[i] : x[i + n];
      x[i] = (up ? x[i + n] : x[i]) + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
  return x[0] + __shfl_xor_sync(0xffffffffu, x[0], 1);
}

// Four lanes' 4 x 4 turned: lane j of them gives element i to lane i's place j.
__device__ __forceinline__ float4 turn4(float4 v, int lane) {
  const bool b0 = (lane & 1) != 0, b1 = (lane & 2) != 0;
  const float g0 = __shfl_xor_sync(0xffffffffu, b0 ? v.x : v.y, 1), g1 = __shfl_xor_sync(0xffffffffu, b0 ? v.z : v.w, 1);
  v = b0 ? make_float4(g0, v.y, g1, v.w) : make_float4(v.x, g0, v.z, g1);
  const float h0 = __shfl_xor_sync(0xffffffffu, b1 ? v.x : v.z, 2), h1 = __shfl_xor_sync(0xffffffffu, b1 ? v.y : v.w, 2);
  return b1 ? make_float4(h0, h1, v.z, v.w) : make_float4(v.x, v.y, h0, h1);
}

template <int K, int VP>
__global__ void __launch_bounds__(kThreads, 1)
    grads_tc_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mq,
                    const __grid_constant__ CUtensorMap mo, const __grid_constant__ CUtensorMap mdv, const Params p,
                    const TcBuffers w, uint32_t* status) {
  extern __shared__ __align__(1024) unsigned char smem[];
  using Lay = Layout<K, VP>;
  constexpr int img = VP * 128, steps = VP / 16;
  Small& sm = *reinterpret_cast<Small*>(smem + Lay::small);
  Bars& bar = sm.bar;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int hpg = p.H / p.G;
  const int tasks = p.slots * p.G;
  volatile uint32_t* fail = &bar.fail;

  if (tid == 0) {
    uint64_t* one[] = {&bar.qk_full, &bar.ox_full, &bar.ox_empty, &bar.ex_full[0], &bar.ex_full[1], &bar.ex_empty[0],
                       &bar.ex_empty[1], &bar.s_empty[0], &bar.s_empty[1], &bar.g_full[0], &bar.g_full[1], &bar.f,
                       &bar.a45, &bar.fin, &bar.drain};
    for (uint64_t* b : one) mbar_init(b, 1);
    mbar_init(&bar.qk_empty, 1 + kEpi);
    for (int i = 0; i < kRing; ++i) mbar_init(&bar.s_full[i], kAux);
    for (int i = 0; i < 2; ++i) mbar_init(&bar.g_empty[i], kEpi + 1);
    mbar_init(&bar.nm, kEpi);
    mbar_init(&bar.free_f, kEpi);
    mbar_init(&bar.free_a, kEpi);
    mbar_init(&bar.sums, kEpi + kAux);
    mbar_init(&bar.epi_sync, kEpi);
    bar.fail = 0;
    fence_mbar_init();
  }
  if (warp == kMma) tc::tmem_alloc(&bar.taddr, 512);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  constexpr uint32_t tb = 0;  // the whole of tensor memory is this block's: its base is 0 (checked below)
  if (bar.taddr != 0u) {
    if (tid == 0) {
      atomicOr(status, kStatusTmem);
      bar.fail = 1;
    }
    __syncthreads();
  }
  auto wait1 = [&](uint64_t* b, uint32_t parity) { return chain_wait(b, parity, status, fail); };
  auto wait = [&](uint64_t* b, uint32_t parity) { return chain_wait_warp(b, parity, status, fail); };
  uint32_t meetings = 0;
  auto meet = [&](uint64_t* b) {
    __syncwarp();
    if (lane == 0) mbar_arrive(b);
    return wait(b, meetings++ & 1);
  };

  if (warp >= kMma) {
    set_regs_down<kRegCtl>();
    if (warp == kLoad && lane == 0) {  // ---- loads
      int n, tok, task = 0, hc = 0;    // tasks and heads begun
      int n_g = 0, n_ex = 0, n_ox = 0;
      Seq q;
      bool ok = true;
      for (int t = blockIdx.x; ok && t < tasks; t += gridDim.x) {
        const int slot = t / p.G, gr = t - slot * p.G;
        if (!chunk_at(p, slot, &n, &q, &tok)) continue;
        const int tt = q.t0 + tok;
        for (int h = gr * hpg; h < (gr + 1) * hpg; ++h, ++hc) {
          const long long ch = static_cast<long long>(slot) * p.H + h;
          const uint32_t last = (hc - 1) & 1;
          bulk_prefetch_l2(w.S + ch * state_image(p.V, K), VP * K * 4);  // warps 8-11 read these next
          bulk_prefetch_l2(w.dS + ch * state_image(p.V, K), VP * K * 4);
          for (int i = 0; i < VP / 64; ++i) {
            tma_prefetch_4d(&mo, 64 * i, h, tt, q.b);
            tma_prefetch_4d(&mdv, 64 * i, h, tt, q.b);
          }
          if (hc > 1 && !(ok = wait1(&bar.g_empty[hc & 1], (hc / 2 - 1) & 1))) break;
          mbar_arrive_expect_tx(&bar.g_full[hc & 1], kGateFloats * 4);
          bulk_g2s(sm.gate[hc & 1], w.gates + ch * kGateFloats, kGateFloats * 4, &bar.g_full[hc & 1]);
          ++n_g;
          if (hc > 1 && !(ok = wait1(&bar.ex_empty[hc & 1], (hc / 2 - 1) & 1))) break;
          mbar_arrive_expect_tx(&bar.ex_full[hc & 1], 3 * img);
          unsigned char* ex = smem + Lay::ex + (hc & 1) * Lay::kEx;
          bulk_g2s(ex, w.E + ch * 3 * img, 2 * img, &bar.ex_full[hc & 1]);
          bulk_g2s(ex + 2 * img, w.dX + ch * img, img, &bar.ex_full[hc & 1]);
          ++n_ex;
          bulk_prefetch_l2(w.E + ch * 3 * img + 2 * img, img);
          if (hc > 0 && !(ok = wait1(&bar.ox_empty, last))) break;
          mbar_arrive_expect_tx(&bar.ox_full, (VP / 64) * kReg + img);
          bulk_g2s(smem + Lay::el, w.E + ch * 3 * img + 2 * img, img, &bar.ox_full);
          for (int i = 0; i < VP / 64; ++i) {
            tma_load_4d(smem + Lay::ox + i * kReg, &mo, &bar.ox_full, 64 * i, h, tt, q.b);
            tma_load_4d(smem + Lay::ox + i * kReg + kTile, &mdv, &bar.ox_full, 64 * i, h, tt, q.b);
          }
          ++n_ox;
          if (h == gr * hpg) {  // Q and K, which the products with E do not need
            if (task > 0 && !(ok = wait1(&bar.qk_empty, (task - 1) & 1))) break;
            mbar_arrive_expect_tx(&bar.qk_full, (K / 64) * kReg);
            for (int i = 0; i < K / 64; ++i) {
              tma_load_4d(smem + i * kReg, &mq, &bar.qk_full, 64 * i, gr, tt, q.b);
              tma_load_4d(smem + i * kReg + kTile, &mk, &bar.qk_full, 64 * i, gr, tt, q.b);
            }
            ++task;
          }
        }
      }
      bar.n_g = n_g, bar.n_ex = n_ex, bar.n_ox = n_ox, bar.n_qk = task;
    }
    if (warp == kMma) {  // ---- MMAs
      constexpr uint32_t idKQ = tc::idesc_bf16(128, 64, false, false);
      constexpr uint32_t idF = tc::idesc_bf16(128, 64, false, true);
      constexpr uint32_t idA = tc::idesc_bf16(128, 128, false, false);
      constexpr uint32_t idA64 = tc::idesc_bf16(128, 64, false, true);
      constexpr uint32_t idMM = tc::idesc_bf16(128, 64, true, true);
      constexpr uint32_t idMK = tc::idesc_bf16(128, 128, true, false);
      auto kstep = [](int s) { return static_cast<uint32_t>(((s >> 2) * kReg + (s & 3) * 32) >> 4); };
      auto nstep = [](int s) { return static_cast<uint32_t>((s * 2048) >> 4); };
      auto jstep = [](int s) { return static_cast<uint32_t>((s * 32) >> 4); };
      const uint32_t sb = smem_u32(smem);
      // state columns as lanes: two 64-column regions (dstate 64: the same one twice, the upper lanes are not read)
      constexpr uint32_t qreg = K == 128 ? kReg : 0u;
      const uint32_t dQK = desc_lo(sb, 16), dK = desc_lo(sb + kTile, 16);
      const uint32_t dQn = desc_lo(sb, qreg), dKn = desc_lo(sb + kTile, qreg);
      const uint32_t dOX = desc_lo(sb + Lay::ox, 16);
      const uint32_t dN = desc_lo(sb + Lay::nm, 16), dM = desc_lo(sb + Lay::nm + kTile, 16);  // hi; M follows N
      const uint32_t dNl = desc_lo(sb + Lay::nm + 2 * kTile, 16), dMl = desc_lo(sb + Lay::nm + 3 * kTile, 16);
      const uint32_t dEl = desc_lo(sb + Lay::el, img);
      constexpr uint32_t im = img >> 4;  // from one piece of E to the next
      int n, tok, task = 0, hc = 0, rc = 0;
      Seq q;
      bool ok = true;
      for (int t = blockIdx.x; ok && t < tasks; t += gridDim.x) {
        const int slot = t / p.G;
        if (!chunk_at(p, slot, &n, &q, &tok)) continue;
        const int have = q.len - tok;
        const bool cut = have < kC && p.cu != nullptr;  // rows of the next sequence in the tiles
        for (int h = 0; h < hpg; ++h, ++hc) {
          const uint32_t ph = hc & 1;
          const uint32_t dE = desc_lo(sb + Lay::ex, img) + ph * (Lay::kEx >> 4);       // E hi, mid, dX lo
          const uint32_t dEX = desc_lo(sb + Lay::ex, 2 * img) + ph * (Lay::kEx >> 4);  // [E hi | dX lo]
          ok = wait(&bar.ox_full, ph) && wait(&bar.ex_full[ph], (hc >> 1) & 1);
          if (!ok) break;
          if (cut) {
            zero_rows(smem + Lay::ox, VP / 64, kReg, have);
            zero_rows(smem + Lay::ox + kTile, VP / 64, kReg, have);
            fence_proxy_async_smem();
            __syncwarp();
          }
          if (hc > 0) ok = wait(&bar.free_f, (hc - 1) & 1);
          if (!ok) break;
          tc::fence_after_sync();
          if (elect_one()) {
#pragma unroll 1
            for (int s4 = 0; s4 < steps / 4; ++s4) {  // 64 value channels
              const uint32_t ox = dOX + s4 * (kReg >> 4), vo = s4 * 512;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const bool more = s4 > 0 || i > 0;
                mma_ss(tb + cF, ox + 2 * i, dE + vo + 128 * i, idF, more);
                mma_ss(tb + cF, ox + 2 * i, dE + im + vo + 128 * i, idF, true);
                mma_ss(tb + cF, ox + 2 * i, dEl + vo + 128 * i, idF, true);
                mma_ss(tb + cFX, dEX + vo + 128 * i, dE + vo + 128 * i, idMM, more);
                mma_ss(tb + cFX, dEX + vo + 128 * i, dE + im + vo + 128 * i, idMM, true);
              }
            }
          }
          __syncwarp();
          if (h > 0 && elect_one()) tc::mma_commit(&bar.f);
          __syncwarp();
          if (hc > 0) ok = wait(&bar.free_a, (hc - 1) & 1);
#pragma unroll 1
          for (int s2 = 0; ok && s2 < steps / 2; ++s2, ++rc) {  // the ring once around
            if (h == 0 && s2 == steps / 4) {  // Q K^t and K K^t, late: Q and K come when the last group is done with theirs
              ok = wait(&bar.qk_full, task & 1);
              if (!ok) break;
              if (cut) {
                zero_rows(smem, K / 64, kReg, have);
                zero_rows(smem + kTile, K / 64, kReg, have);
                fence_proxy_async_smem();
                __syncwarp();
              }
              ++task;
              if (elect_one()) {
#pragma unroll 1
                for (int s = 0; s < K / 16; ++s) mma_ss(tb + cKQ, dQK + kstep(s), dK + kstep(s), idKQ, s > 0);
                tc::mma_commit(&bar.f);
              }
              __syncwarp();
            }
            const uint32_t ox = dOX + (s2 >> 1) * (kReg >> 4) + (s2 & 1) * 4, vo = s2 * 256;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              constexpr uint32_t pc = kSlot / 6;
              const uint32_t aS = tb + cRing + i * kSlot, aD = aS + 3 * pc;
              const uint32_t e = dE + vo + 128 * i;
              const bool more = s2 > 0 || i > 0;
              ok = ok && wait(&bar.s_full[i], rc & 1);
              if (!ok) break;
              tc::fence_after_sync();
              if (elect_one()) {
                mma_ts_lo(tb + cA, aS, ox + 2 * i, idA, more);
                mma_ts_lo(tb + cA, aS + pc, ox + 2 * i, idA, true);
                mma_ts_lo(tb + cA, aS + 2 * pc, ox + 2 * i, idA, true);
                mma_ts_lo(tb + cA + 64, aS, e + 2 * im, idA64, true);
                mma_ts_lo(tb + cA + 64, aS + pc, e + 2 * im, idA64, true);
                mma_ts_lo(tb + cA3, aD, e, idA64, more);
                mma_ts_lo(tb + cA3, aD + pc, e, idA64, true);
                mma_ts_lo(tb + cA3, aD + 2 * pc, e, idA64, true);
                mma_ts_lo(tb + cA3, aD, e + im, idA64, true);
                mma_ts_lo(tb + cA3, aD + pc, e + im, idA64, true);
                mma_ts_lo(tb + cA3, aD, dEl + vo + 128 * i, idA64, true);
                tc::mma_commit(&bar.s_empty[i]);
              }
              __syncwarp();
            }
          }
          if (!ok) break;
          if (elect_one()) {
            tc::mma_commit(&bar.ox_empty);
            tc::mma_commit(&bar.ex_empty[ph]);
          }
          __syncwarp();
          ok = wait(&bar.nm, ph);
          if (!ok) break;
          tc::fence_after_sync();
          if (elect_one()) {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
              mma_ss(tb + cF, dKn + nstep(s), dN + jstep(s), idMK, s > 0);  // K^t [N; M]^t: a4 and the first part of a5
              mma_ss(tb + cF, dKn + nstep(s), dNl + jstep(s), idMK, true);
              mma_ss(tb + cFX, dKn + nstep(s), dM + nstep(s), idMM, true);
              mma_ss(tb + cFX, dKn + nstep(s), dMl + nstep(s), idMM, true);
              mma_ss(tb + cFX, dQn + nstep(s), dN + nstep(s), idMM, true);
              mma_ss(tb + cFX, dQn + nstep(s), dNl + nstep(s), idMM, true);
            }
            tc::mma_commit(&bar.a45);  // and with them a1 to a3
            if (h == hpg - 1) tc::mma_commit(&bar.qk_empty);
          }
          __syncwarp();
        }
      }
      if (*fail != 0u && elect_one()) {
        tc::mma_commit(&bar.drain);
        mbar_wait_bounded(&bar.drain, 0, status);
      }
      __syncwarp();
    }
    if (warp == kGates) {  // ---- dg, dbeta
      int n, tok, hc = 0;
      Seq q;
      bool ok = true;
      for (int t = blockIdx.x; ok && t < tasks; t += gridDim.x) {
        const int slot = t / p.G, gr = t - slot * p.G;
        if (!chunk_at(p, slot, &n, &q, &tok)) continue;
        for (int h = gr * hpg; h < (gr + 1) * hpg; ++h, ++hc) {
          ok = wait(&bar.g_full[hc & 1], (hc / 2) & 1) && wait(&bar.sums, hc & 1);
          if (!ok) break;
          const float* gate = sm.gate[hc & 1];
          const float all = ((sm.dot[0] + sm.dot[1]) + (sm.dot[2] + sm.dot[3])) * gate[kGateEnd];
          float y[2], r[2], R[2], c[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int j = 2 * lane + k;
            y[k] = (sm.y[0][j] + sm.y[1][j]) + (sm.y[2][j] + sm.y[3][j]);
            r[k] = (sm.r[0][j] + sm.r[1][j]) + (sm.r[2][j] + sm.r[3][j]);
            R[k] = (sm.R[0][j] + sm.R[1][j]) + (sm.R[2][j] + sm.R[3][j]);
            c[k] = (sm.c[0][j] + sm.c[1][j]) + (sm.c[2][j] + sm.c[3][j]);  // w_j k_j . a3_j
          }
          const float b0 = gate[kGateBeta + 2 * lane], b1 = gate[kGateBeta + 2 * lane + 1];
          // the rows' sums over their first 32 columns, which R lacks past them
          const float s0 = sm.base[2 * lane] + sm.base[64 + 2 * lane], s1 = sm.base[2 * lane + 1] + sm.base[65 + 2 * lane];
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&bar.fin);
            mbar_arrive(&bar.g_empty[hc & 1]);
          }
          float pre = b0 * c[0] + b1 * c[1], suf = r[0] + r[1], left = s0 + s1;  // sums up to and from this lane's tokens
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const float a = __shfl_up_sync(0xffffffffu, pre, o), b = __shfl_down_sync(0xffffffffu, suf, o);
            const float e = __shfl_down_sync(0xffffffffu, left, o);
            if (lane >= o) pre += a;
            if (lane + o < 32) suf += b, left += e;
          }
          if (lane >= 16) {
            R[0] += left;
            R[1] += left - s0;
          }
          const float before = __shfl_up_sync(0xffffffffu, pre, 1);
          const float after = __shfl_down_sync(0xffffffffu, suf, 1);
          const float pre0 = lane > 0 ? before : 0.f, suf1 = r[1] + (lane < 31 ? after : 0.f);
          const float dg[2] = {R[0] + (suf1 + r[0]) + pre0 + all, R[1] + suf1 + (pre0 + b0 * c[0]) + all};
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int j = 2 * lane + k;
            if (tok + j < q.len) {
              const long long to = (static_cast<long long>(q.b) * p.L + q.t0 + tok + j) * p.H + h;
              p.dg[to] = p.g[to] <= kMinGate ? 0.f : dg[k];  // a clamped gate has no gradient
              p.dbeta[to] = y[k] + c[k];
            }
          }
        }
      }
    }
  } else if (warp >= kEpi) {  // ---- staging, <dS1, S0>
    set_regs_up<kRegAux>();
    const int quarter = warp & 3;
    const bool staging = 32 * quarter < K;  // (dstate 64: the upper lanes of S0 and dS1 hold nothing and are not read)
    int n, tok, hc = 0, rc = 0;
    Seq q;
    bool ok = true;
    for (int t = blockIdx.x; ok && t < tasks; t += gridDim.x) {
      const int slot = t / p.G, gr = t - slot * p.G;
      if (!chunk_at(p, slot, &n, &q, &tok)) continue;
      for (int h = gr * hpg; h < (gr + 1) * hpg; ++h, ++hc) {
        const long long ch = static_cast<long long>(slot) * p.H + h;
        const float *gS = w.S + ch * state_image(p.V, K), *gD = w.dS + ch * state_image(p.V, K);
        // S0 and dS1, 16 value channels a step, two steps in flight.  A thread's lane is a state column; four lanes load
        // four columns of four channels, four times, and turn them among themselves.
        float2 acc = make_float2(0, 0);
        float4 s0[2][4], d1[2][4];
        const int piece = 8 * quarter + (lane >> 2);
        auto fetch = [&](int s, int into) {
          if (staging) {
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              s0[into][m] = __ldcs(reinterpret_cast<const float4*>(gS + image_at(VP, 16 * s + 4 * m + (lane & 3), piece)));
              d1[into][m] = __ldcs(reinterpret_cast<const float4*>(gD + image_at(VP, 16 * s + 4 * m + (lane & 3), piece)));
            }
          }
        };
        auto put = [&](float4 (&f)[4], uint32_t to) {
          uint32_t o[24];
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const float4 v = turn4(f[m], lane);
            split3(make_float2(v.x, v.y), o[2 * m], o[8 + 2 * m], o[16 + 2 * m]);
            split3(make_float2(v.z, v.w), o[2 * m + 1], o[9 + 2 * m], o[17 + 2 * m]);
          }
          tmem_st16u(to, o);
          tmem_st8u(to + 16, o + 16);
        };
        fetch(0, 0);
        fetch(1, 1);
#pragma unroll 1
        for (int s2 = 0; ok && s2 < steps; s2 += 2, ++rc) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            ok = ok && (rc == 0 || wait(&bar.s_empty[u], (rc - 1) & 1));
            if (!ok) break;
            tc::fence_after_sync();
            if (staging) {
              const uint32_t to = tb + cRing + u * kSlot + (static_cast<uint32_t>(32 * quarter) << 16);
#pragma unroll
              for (int m = 0; m < 4; ++m) {
                acc = f2_fma(make_float2(s0[u][m].x, s0[u][m].y), make_float2(d1[u][m].x, d1[u][m].y), acc);
                acc = f2_fma(make_float2(s0[u][m].z, s0[u][m].w), make_float2(d1[u][m].z, d1[u][m].w), acc);
              }
              put(s0[u], to);
              put(d1[u], to + kSlot / 2);
              tc::tmem_wait_st();
            }
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar.s_full[u]);
            if (s2 + 2 < steps) fetch(s2 + 2 + u, u);
          }
        }
        if (!ok) break;
        float d = staging ? acc.x + acc.y : 0.f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
        ok = hc == 0 || wait(&bar.fin, (hc - 1) & 1);  // the last head's sums have been read
        if (!ok) break;
        if (lane == 0) {
          sm.dot[warp - kEpi] = d;
          mbar_arrive(&bar.sums);
        }
        __syncwarp();
      }
    }
  } else {  // ---- epilogues
    set_regs_up<kRegEpi>();
    const int quarter = warp & 3, hf = warp >> 2, row = 32 * quarter + lane, c0 = 32 * hf;
    const uint32_t tl = static_cast<uint32_t>(32 * quarter) << 16;
    const bool klive = row < K;
    int n, tok, hc = 0;
    Seq q;
    bool ok = true;
    auto arrive = [&](uint64_t* b) {
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(b);
    };
    for (int t = blockIdx.x; ok && t < tasks; t += gridDim.x) {
      const int slot = t / p.G, gr = t - slot * p.G;
      if (!chunk_at(p, slot, &n, &q, &tok)) continue;
      float dq[32], dk[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) dq[i] = dk[i] = 0.f;
      for (int h = 0; h < hpg; ++h, ++hc) {
        const uint32_t ph = hc & 1;
        const float* gate = sm.gate[hc & 1];
        ok = wait(&bar.g_full[hc & 1], (hc / 2) & 1) && wait(&bar.f, ph);
        if (!ok) break;
        tc::fence_after_sync();
        {  // rows: f and qk (lanes 0-63), F' and kk (64-127); columns c0 .., 16 at a time
          const int i = row & 63;
          const bool second = quarter >= 2;
          const float own = second ? 1.f : 0.f;  // (the upper rows of cFX are E E^t)
          const GateSum bi = {gate[kGateB + i], gate[kGateBLo + i]};
          const float sc = second ? -1.f : p.scale;
          const uint32_t wide = __float_as_uint(gate[kGateWide]);
          unsigned char* tile = smem + Lay::nm + (second ? kTile : 0);
          ok = hc == 0 || wait(&bar.fin, (hc - 1) & 1);  // the last head's sums have been read
          if (!ok) break;
          float run = 0.f;
#pragma unroll 1
          for (int g = 0; g < 2; ++g) {
            const int cg = c0 + 16 * g, lim = (second ? i - 1 : i) - cg;  // last of these columns in the row
            float x[16];
            {
              float b[16];
              tc::tmem_ld16(tb + tl + cF + cg, x);
              tc::tmem_ld16(tb + tl + cFX + cg, b);
              tc::tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 16; ++k) x[k] = fmaf(own, b[k], x[k]);
            }
            if ((wide >> (cg / 2)) & 1u) {  // bit 8 of a 16-token group
#pragma unroll
              for (int k = 0; k < 16; ++k) x[k] *= sc * __expf(bi - GateSum{gate[kGateB + cg + k], gate[kGateBLo + cg + k]});
            } else {
              const float rf = sc * __expf(bi - GateSum{gate[kGateB + cg], gate[kGateBLo + cg]});
#pragma unroll
              for (int k = 0; k < 16; k += 4) {
                const float4 k4 = *reinterpret_cast<const float4*>(gate + kGateKey + cg + k);
                x[k] *= rf * k4.x, x[k + 1] *= rf * k4.y, x[k + 2] *= rf * k4.z, x[k + 3] *= rf * k4.w;
              }
            }
            float R[16];  // beta y later; first beta x, which is N or M
#pragma unroll
            for (int k = 0; k < 16; k += 4) {
              const float4 b4 = *reinterpret_cast<const float4*>(gate + kGateBeta + cg + k);
              const float be[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
              for (int m = 0; m < 4; ++m) {
                x[k + m] = k + m <= lim ? x[k + m] : 0.f;
                R[k + m] = be[m] * x[k + m];
              }
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              uint32_t o[4], l[4];
#pragma unroll
              for (int m = 0; m < 4; ++m) split2(make_float2(R[8 * k + 2 * m], R[8 * k + 2 * m + 1]), o[m], l[m]);
              const uint32_t to = tc::chunk_off(i, cg / 8 + k);
              *reinterpret_cast<uint4*>(tile + to) = make_uint4(o[0], o[1], o[2], o[3]);
              *reinterpret_cast<uint4*>(tile + 2 * kTile + to) = make_uint4(l[0], l[1], l[2], l[3]);
            }
            // y, and the prefixes of beta y along the row that reach column t <= i
            float prod[16];
            tc::tmem_ld16(tb + tl + cKQ + cg, prod);
            tc::tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              x[k] *= prod[k];
              const float by = R[k] * prod[k];
              R[k] = k <= i - cg ? run : 0.f;
              run += by;
            }
            const float y = column_sums(x, lane), Rs = column_sums(R, lane);
            if ((lane & 1) == 0) {
              sm.y[quarter][cg + (lane >> 1)] = y;
              sm.R[quarter][cg + (lane >> 1)] = Rs;
            }
          }
          if (hf == 0) sm.base[row] = run;
          fence_proxy_async_smem();
          arrive(&bar.nm);
        }
        // state columns as lanes: a4, a5, whose place the next head waits for; then a1, a2, a3
        ok = wait(&bar.a45, ph);
        if (!ok) break;
        tc::fence_after_sync();
        {
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            float a[16], b[16];
            tc::tmem_ld16(tb + tl + cF + c0 + 16 * g, a);
            tc::tmem_ld16(tb + tl + cFX + c0 + 16 * g, b);
            tc::tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              dq[16 * g + k] += a[k];
              dk[16 * g + k] += b[k];
            }
          }
        }
        arrive(&bar.free_f);
        {
          // (dstate 64: lanes 64 and above hold nothing; they read the lower lanes' elements and count for nothing)
          const unsigned char* tq = smem + (K == 128 ? (row >> 6) * kReg : 0) + c0 * 128;
          const uint32_t col = (row & 63) * 2;
          auto elem = [&](const unsigned char* tile, int k) {
            return to_f32(*reinterpret_cast<const __nv_bfloat16*>(tile + k * 128 + (col ^ ((k & 7) << 4))));
          };
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const int cg = c0 + 16 * g;
            float s[16], kv[16], a[16], b[16], a3[16];
            tc::tmem_ld16(tb + tl + cA + cg, a);
            tc::tmem_ld16(tb + tl + cA + 64 + cg, b);
            tc::tmem_ld16(tb + tl + cA3 + cg, a3);
#pragma unroll
            for (int k = 0; k < 16; ++k) kv[k] = elem(tq + kTile, 16 * g + k);
            tc::tmem_wait_ld();
            if (g == 1) arrive(&bar.free_a);
#pragma unroll
            for (int k = 0; k < 16; k += 2) {
              const float2 e = *reinterpret_cast<const float2*>(gate + kGateE + cg + k);
              const float v0 = -p.scale * e.x * a[k], v1 = -p.scale * e.y * a[k + 1];
              const float u0 = e.x * b[k], u1 = e.y * b[k + 1];
              dq[16 * g + k] += v0;
              dq[16 * g + k + 1] += v1;
              dk[16 * g + k] += u0;
              dk[16 * g + k + 1] += u1;
              s[k] = fmaf(u0, kv[k], v0 * elem(tq, 16 * g + k));
              s[k + 1] = fmaf(u1, kv[k + 1], v1 * elem(tq, 16 * g + k + 1));
            }
            if (K == 64 && !klive) {
#pragma unroll
              for (int k = 0; k < 16; ++k) s[k] = 0.f;
            }
            const float r = column_sums(s, lane);
#pragma unroll
            for (int k = 0; k < 16; k += 2) {
              const float2 bw = *reinterpret_cast<const float2*>(gate + kGateW + cg + k);
              const float2 wt = *reinterpret_cast<const float2*>(gate + kGateTail + cg + k);
              const float v0 = a3[k], v1 = a3[k + 1];
              dk[16 * g + k] = fmaf(bw.x, v0, dk[16 * g + k]);
              dk[16 * g + k + 1] = fmaf(bw.y, v1, dk[16 * g + k + 1]);
              s[k] = wt.x * v0 * kv[k];
              s[k + 1] = wt.y * v1 * kv[k + 1];
            }
            if (K == 64 && !klive) {
#pragma unroll
              for (int k = 0; k < 16; ++k) s[k] = 0.f;
            }
            const float c = column_sums(s, lane);
            if ((lane & 1) == 0) {
              sm.r[quarter][cg + (lane >> 1)] = r;
              sm.c[quarter][cg + (lane >> 1)] = c;
            }
          }
        }
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&bar.sums);
          mbar_arrive(&bar.g_empty[hc & 1]);
        }
      }
      if (!ok) break;
      if (lane == 0) mbar_arrive(&bar.qk_empty);  // (its tiles were last read before bar.sums)
      // dq and dk, 32 tokens at a time: through a tile in shared memory to whole 16-byte pieces of their rows
      const int have = min(kC, q.len - tok);
      uint32_t qo[16], ko[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        qo[k] = pack_pair<__nv_bfloat16>(make_float2(dq[2 * k], dq[2 * k + 1]));
        ko[k] = pack_pair<__nv_bfloat16>(make_float2(dk[2 * k], dk[2 * k + 1]));
      }
#pragma unroll 1
      for (int part = 0; part < 4; ++part) {
        const int which = part >> 1, half = part & 1;
        ok = meet(&bar.epi_sync);  // the tile's last pieces have been read
        if (!ok) break;
        if (klive && hf == half) {
          uint16_t* so = reinterpret_cast<uint16_t*>(smem + Lay::out) + row;
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const uint32_t v = which == 0 ? qo[k] : ko[k];
            so[2 * k * K] = static_cast<uint16_t>(v);
            so[(2 * k + 1) * K] = static_cast<uint16_t>(v >> 16);
          }
        }
        ok = meet(&bar.epi_sync);
        if (!ok) break;
        constexpr int kPieces = K / 8, kRows = kEpi * 32 / kPieces;
        const int pc = tid % kPieces;
        void* out = which == 0 ? p.dq : p.dk;
        const View& v = which == 0 ? p.vdq : p.vdk;
        for (int tk = tid / kPieces; tk < 32 && 32 * half + tk < have; tk += kRows)
          __stcs(reinterpret_cast<uint4*>(row_of<__nv_bfloat16>(out, v, q.b, q.t0 + tok + 32 * half + tk, gr)) + pc,
                 *reinterpret_cast<const uint4*>(smem + Lay::out + (tk * kPieces + pc) * 16));
      }
      ok = ok && meet(&bar.epi_sync);  // N lo of the next head goes where they were
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (*fail != 0u && tid == 0) {  // the copies in flight land before the block ends: each barrier's last phase
    auto last = [&](uint64_t* b, int n) {
      if (n > 0) mbar_wait_bounded(b, (n - 1) & 1, status);
    };
    for (int i = 0; i < 2; ++i) {
      last(&bar.g_full[i], (bar.n_g + 1 - i) / 2);
      last(&bar.ex_full[i], (bar.n_ex + 1 - i) / 2);
    }
    last(&bar.ox_full, bar.n_ox);
    last(&bar.qk_full, bar.n_qk);
  }
  if (warp == kMma) {
    tc::tmem_relinquish();
    tc::tmem_dealloc(bar.taddr, 512);
  }
}

template <int K, int VP>
cudaError_t launch(const CUtensorMap& mk, const CUtensorMap& mq, const CUtensorMap& mo, const CUtensorMap& mdv,
                   const Params& p, const TcBuffers& w, uint32_t* status, cudaStream_t st) {
  static unsigned long long mask = 0;
  constexpr int bytes = Layout<K, VP>::bytes;
  static_assert(bytes <= kMaxDynSmem, "shared memory");
  const cudaError_t e = static_cast<cudaError_t>(
      ensure_smem_attr(reinterpret_cast<const void*>(grads_tc_kernel<K, VP>), bytes, &mask));
  if (e != cudaSuccess) return e;
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const long long tasks = static_cast<long long>(p.slots) * p.G;
  grads_tc_kernel<K, VP><<<static_cast<unsigned>(tasks < sms ? tasks : sms), kThreads, bytes, st>>>(mk, mq, mo, mdv, p, w,
                                                                                                 status);
  return cudaGetLastError();
}

}  // namespace

cudaError_t tc_grads(const CUtensorMap& mk, const CUtensorMap& mq, const CUtensorMap& mo, const CUtensorMap& mdv,
                     const Params& p, const TcBuffers& w, uint32_t* status, cudaStream_t st) {
  if (p.slots == 0) return cudaSuccess;
  const bool wide = pad_channels(p.V) == 128;
  if (p.K == 64)
    return wide ? launch<64, 128>(mk, mq, mo, mdv, p, w, status, st) : launch<64, 64>(mk, mq, mo, mdv, p, w, status, st);
  return wide ? launch<128, 128>(mk, mq, mo, mdv, p, w, status, st) : launch<128, 64>(mk, mq, mo, mdv, p, w, status, st);
}

}  // namespace delta
}  // namespace emab
