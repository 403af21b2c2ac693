// Gated delta rule, tensor-core family: the backward walk, last chunk first.
//
// One block per (sequence, head) carries dS, the gradient of the state, with a tensor-memory lane per value channel as
// in the forward walk, whose mirror it is:
//
//   Z = dS K^t,  Y = dO^t P  ->  W = beta Y + (beta w) Z  ->  dX = W + W (T - I)  ->  dS = exp(b_end) dS + dO~ Q - (exp(b) dX) K
//
// with w_j = exp(b_end - b_j) and dO~_i = scale exp(b_i) dO_i.  W, dX and dS are the chain; Y (from P and dO as they
// lie in shared memory) and dO~ Q are ready before it needs them.  Operands that are not bf16 by nature are hi + lo
// pairs (delta_tc.cuh), dO~, whose rounding stays in dS, three pieces.  exp(b) dX, whose rounding stays there too, is a pair:
// it comes from the pairs W and T, and a third piece would take the error of d initial states from 2.2e-6 to 1.9e-6 for
// four more steps in the chain.  dv = dX; for the gradient kernel dS at every chunk's
// end is left as an fp32 image, and what dX has beyond dv as a bf16 tile.
//
// Bound: the chain's latency, as in the forward walk (three dependent MMA groups of about 900, 750 and 950 cycles with
// their hand-overs, and an epilogue after each): 264 us at 4 x 4096 tokens of 32 heads of 128 x 128, 175 on 9 packed
// sequences of 8 heads.  dS's image leaves in parts, one in every gap of the chain (at once: 283).  Roles: warps 0-7 the
// chain's epilogues, warps 8-11 dO~ and the copy of dv to its rows, warp 12 the MMAs, warp 13 the loads.
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
constexpr int kMma = 12, kLoad = 13;  // (14 and 15 only fill their warpgroup)
constexpr int kThreads = 16 * 32;
constexpr int kRegEpi = 168, kRegAux = 96, kRegCtl = 80;
static_assert(2 * kRegEpi + kRegAux + kRegCtl == 4 * 128, "register split");
constexpr int kStages = 2;
constexpr int kReg = 128 * 128;  // 64 query rows, then 64 key rows of 64 columns

// tensor-memory columns
constexpr uint32_t cZ = 0;     // Z; then W T hi
constexpr uint32_t cY = 64;    // Y; then W T lo
constexpr uint32_t cW = 128;   // W hi, lo; then -exp(b) dX hi, lo (32 columns each)
constexpr uint32_t cDS = 256;
constexpr uint32_t cDh = 384;  // dS hi (K / 2 columns)
constexpr uint32_t cDl = 448;  // dS lo
constexpr uint32_t cO = 384;   // dO~ hi, mid, lo (32 columns each), once Z has read dS

struct Bars {
  uint64_t full[kStages], empty[kStages];
  uint64_t z, dx, ds;            // MMA groups done
  uint64_t s, w, wx, dot, dv;    // epilogues done: dS, W, exp(b) dX, dO~ ready; dv staged
  uint64_t drain;
  uint32_t taddr, fail;
  int issued;  // chunks whose loads were issued
};

template <int K>
struct Stage {
  static constexpr int oKQ = 0;                     // per 64 columns: 64 rows of Q, 64 of K
  static constexpr int oT = oKQ + (K / 64) * kReg;  // T hi, lo
  static constexpr int oP = oT + 2 * kTile;         // P hi, lo
  static constexpr int oO = oP + 2 * kTile;         // dO: two 64-channel regions; later dv, rows of headdim
  static constexpr int oG = oO + 2 * kTile;
  static constexpr int kBytes = (oG + kGateFloats * 4 + 1023) / 1024 * 1024;
};

__device__ __forceinline__ float2 pair(const float (&a)[2][16], int i) {
  return make_float2(a[i / 8][(2 * i) % 16], a[i / 8][(2 * i) % 16 + 1]);
}

template <int K>
__global__ void __launch_bounds__(kThreads, 1)
    bwd_tc_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mq,
                  const __grid_constant__ CUtensorMap mo, const Params p, const TcBuffers w, uint32_t* status) {
  using St = Stage<K>;
  extern __shared__ __align__(1024) unsigned char smem[];
  Bars& bar = *reinterpret_cast<Bars*>(smem + kStages * St::kBytes);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int h = blockIdx.x, n = blockIdx.y, gr = h / (p.H / p.G);
  const Seq q = seq_at(p, n);
  const int nc = (q.len + kC - 1) / kC;
  const int VP = pad_channels(p.V);
  volatile uint32_t* fail = &bar.fail;

  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bar.full[i], 1);
      mbar_init(&bar.empty[i], kEpi + kAux);
    }
    mbar_init(&bar.z, 1);
    mbar_init(&bar.dx, 1);
    mbar_init(&bar.ds, 1);
    mbar_init(&bar.s, kEpi);
    mbar_init(&bar.w, kEpi);
    mbar_init(&bar.wx, kEpi);
    mbar_init(&bar.dot, kAux);
    mbar_init(&bar.dv, kEpi);
    mbar_init(&bar.drain, 1);
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
  auto chunk = [&](int r) { return nc - 1 - r; };  // of step r

  if (warp >= kMma) {
    set_regs_down<kRegCtl>();
    if (warp == kLoad && lane == 0) {  // ---- loads
      const int regions = VP / 64;
      int r = 0;
      for (; r < nc; ++r) {
        const int st = r % kStages, c = chunk(r);
        if (r >= kStages && !wait1(&bar.empty[st], (r / kStages - 1) & 1)) break;
        unsigned char* base = smem + st * St::kBytes;
        const long long ch = static_cast<long long>(q.slot + c) * p.H + h;
        mbar_arrive_expect_tx(&bar.full[st], (K / 64) * kReg + (4 + regions) * kTile + kGateFloats * 4);
        for (int i = 0; i < K / 64; ++i) {
          tma_load_4d(base + St::oKQ + i * kReg, &mq, &bar.full[st], 64 * i, gr, q.t0 + c * kC, q.b);
          tma_load_4d(base + St::oKQ + i * kReg + kTile, &mk, &bar.full[st], 64 * i, gr, q.t0 + c * kC, q.b);
        }
        for (int i = 0; i < regions; ++i)
          tma_load_4d(base + St::oO + i * kTile, &mo, &bar.full[st], 64 * i, h, q.t0 + c * kC, q.b);
        bulk_g2s(base + St::oT, w.T + ch * 2 * kTile, 2 * kTile, &bar.full[st]);
        bulk_g2s(base + St::oP, w.P + ch * 2 * kTile, 2 * kTile, &bar.full[st]);
        bulk_g2s(base + St::oG, w.gates + ch * kGateFloats, kGateFloats * 4, &bar.full[st]);
      }
      bar.issued = r;
    }
    if (warp == kMma) {  // ---- MMAs
      constexpr uint32_t id64 = tc::idesc_bf16(128, 64, false, false);   // Z
      constexpr uint32_t idY = tc::idesc_bf16(128, 64, true, true);
      constexpr uint32_t idT = tc::idesc_bf16(128, 128, false, true);    // W [T hi | T lo]
      constexpr uint32_t idTl = tc::idesc_bf16(128, 64, false, true);
      constexpr uint32_t idK = tc::idesc_bf16(128, K, false, true);
      auto kstep = [](int s) { return static_cast<uint64_t>(((s >> 2) * kReg + (s & 3) * 32) >> 4); };
      auto nstep = [](int s) { return static_cast<uint64_t>((s * 2048) >> 4); };
      // step r's tiles, and Y from them
      auto begin = [&](int r) {
        const int st = r % kStages;
        unsigned char* base = smem + st * St::kBytes;
        if (!wait(&bar.full[st], (r / kStages) & 1)) return false;
        const int have = q.len - chunk(r) * kC;
        if (have < kC && p.cu != nullptr) {  // rows of the next sequence
          zero_rows(base + St::oKQ, K / 64, kReg, have);
          zero_rows(base + St::oKQ + kTile, K / 64, kReg, have);
          zero_rows(base + St::oO, 2, kTile, have);
          fence_proxy_async_smem();
        }
        __syncwarp();
        const uint32_t sb = smem_u32(base);
        // (headdim <= 64: the second region is not loaded; what it holds only reaches lanes that nothing reads)
        const uint64_t da = tc::smem_desc_sw128(sb + St::oO, kTile, 1024);
        const uint64_t dp = tc::smem_desc_sw128(sb + St::oP, kTile, 1024);
        const uint64_t dpl = tc::smem_desc_sw128(sb + St::oP + kTile, kTile, 1024);
        if (elect_one()) {
#pragma unroll
          for (int s = 0; s < 4; ++s) tc::mma_bf16(tb + cY, da + nstep(s), dp + nstep(s), idY, s > 0);
#pragma unroll
          for (int s = 0; s < 4; ++s) tc::mma_bf16(tb + cY, da + nstep(s), dpl + nstep(s), idY, true);
        }
        __syncwarp();
        return true;
      };
      bool ok = nc == 0 || begin(0);
      for (int r = 0; ok && r < nc; ++r) {
        const uint32_t sb = smem_u32(smem + (r % kStages) * St::kBytes);
        const uint64_t dk = tc::smem_desc_sw128(sb + St::oKQ + kTile, 16, 1024);
        const uint64_t dkn = tc::smem_desc_sw128(sb + St::oKQ + kTile, kReg, 1024);
        const uint64_t dqn = tc::smem_desc_sw128(sb + St::oKQ, kReg, 1024);
        const uint64_t dt = tc::smem_desc_sw128(sb + St::oT, kTile, 1024);
        ok = wait(&bar.s, r & 1);
        if (!ok) break;
        tc::fence_after_sync();
        if (elect_one()) {
#pragma unroll
          for (int s = 0; s < K / 16; ++s) mma_ts(tb + cZ, tb + cDh + 8 * s, dk + kstep(s), id64, s > 0);
#pragma unroll
          for (int s = 0; s < K / 16; ++s) mma_ts(tb + cZ, tb + cDl + 8 * s, dk + kstep(s), id64, true);
          tc::mma_commit(&bar.z);
        }
        __syncwarp();
        ok = wait(&bar.w, r & 1);
        if (!ok) break;
        tc::fence_after_sync();
        if (elect_one()) {
#pragma unroll
          for (int s = 0; s < 4; ++s) mma_ts(tb + cZ, tb + cW + 8 * s, dt + nstep(s), idT, s > 0);
#pragma unroll
          for (int s = 0; s < 4; ++s) mma_ts(tb + cZ, tb + cW + 32 + 8 * s, dt + nstep(s), idTl, true);
          tc::mma_commit(&bar.dx);
        }
        __syncwarp();
        ok = wait(&bar.dot, r & 1);
        if (!ok) break;
        tc::fence_after_sync();
        if (elect_one()) {
#pragma unroll
          for (int s = 0; s < 4; ++s) mma_ts(tb + cDS, tb + cO + 8 * s, dqn + nstep(s), idK, s > 0);
#pragma unroll
          for (int s = 0; s < 4; ++s) mma_ts(tb + cDS, tb + cO + 32 + 8 * s, dqn + nstep(s), idK, true);
#pragma unroll
          for (int s = 0; s < 4; ++s) mma_ts(tb + cDS, tb + cO + 64 + 8 * s, dqn + nstep(s), idK, true);
        }
        __syncwarp();
        ok = wait(&bar.wx, r & 1);
        if (!ok) break;
        tc::fence_after_sync();
        if (elect_one()) {
#pragma unroll
          for (int s = 0; s < 4; ++s) mma_ts(tb + cDS, tb + cW + 8 * s, dkn + nstep(s), idK, true);
#pragma unroll
          for (int s = 0; s < 4; ++s) mma_ts(tb + cDS, tb + cW + 32 + 8 * s, dkn + nstep(s), idK, true);
          tc::mma_commit(&bar.ds);
        }
        __syncwarp();
        if (r + 1 < nc) ok = begin(r + 1);
      }
      if (*fail != 0u && elect_one()) {
        tc::mma_commit(&bar.drain);
        mbar_wait_bounded(&bar.drain, 0, status);
      }
      __syncwarp();
    }
  } else if (warp >= kEpi) {  // ---- dO~, and dv to its rows
    set_regs_down<kRegAux>();
    const int row = 32 * (warp & 3) + lane;
    const uint32_t tl = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const bool live = row < p.V;
    const int pieces = p.V / 8;  // 16-byte pieces of a row
    for (int r = 0; r < nc; ++r) {
      const int st = r % kStages, c = chunk(r);
      unsigned char* base = smem + st * St::kBytes;
      const float* gate = reinterpret_cast<const float*>(base + St::oG);
      const int have = min(kC, q.len - c * kC);
      if (!wait(&bar.full[st], (r / kStages) & 1)) break;
      if (!wait(&bar.z, r & 1)) break;
      tc::fence_after_sync();
      const unsigned char* src = base + St::oO + (row >> 6) * kTile;
      const uint32_t col = (row & 63) * 2;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        uint32_t hi[16], mid[16], lo[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int t = 32 * g + 2 * i;
          const float2 e = *reinterpret_cast<const float2*>(gate + kGateE + t);  // -exp(b)
          float2 v;
          v.x = to_f32(*reinterpret_cast<const __nv_bfloat16*>(src + t * 128 + (col ^ ((t & 7) << 4))));
          v.y = to_f32(*reinterpret_cast<const __nv_bfloat16*>(src + (t + 1) * 128 + (col ^ (((t + 1) & 7) << 4))));
          v.x = (live && t < have) ? v.x * (-p.scale * e.x) : 0.f;
          v.y = (live && t + 1 < have) ? v.y * (-p.scale * e.y) : 0.f;
          split3(v, hi[i], mid[i], lo[i]);
        }
        tmem_st16u(tb + tl + cO + 16 * g, hi);
        tmem_st16u(tb + tl + cO + 32 + 16 * g, mid);
        tmem_st16u(tb + tl + cO + 64 + 16 * g, lo);
      }
      tc::tmem_wait_st();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.dot);
      if (!wait(&bar.dv, r & 1)) break;
      {
        const int pc = lane & 15, t0 = 2 * (warp - kEpi) + (lane >> 4);
        const uint4* from = reinterpret_cast<const uint4*>(base + St::oO);
        __nv_bfloat16* dst = row_of<__nv_bfloat16>(p.dv, p.vdv, q.b, q.t0 + c * kC, h) + 8 * pc;
        if (pc < pieces) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int t = t0 + 8 * i;
            if (t < have) *(reinterpret_cast<uint4*>(dst + t * p.vdv.t)) = from[t * pieces + pc];
          }
        }
      }
      fence_proxy_async_smem();  // the stage's next load overwrites what was written here
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.empty[st]);
    }
  } else {  // ---- the chain's epilogues
    set_regs_up<kRegEpi>();
    constexpr int KC = K / 2;  // state columns of a thread
    const int row = 32 * (warp & 3) + lane, hf = warp >> 2;
    const uint32_t tl = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const bool live = row < p.V;
    float2 D[KC / 2];
    const long long srow = ((static_cast<long long>(n) * p.H + h) * p.V + row) * K + hf * KC;
#pragma unroll
    for (int i = 0; i < KC; i += 4) {
      const float4 f = (live && p.ds1 != nullptr) ? *reinterpret_cast<const float4*>(p.ds1 + srow + i)
                                                   : make_float4(0, 0, 0, 0);
      D[i / 2] = make_float2(f.x, f.y), D[i / 2 + 1] = make_float2(f.z, f.w);
    }
    auto arrive = [&](uint64_t* b) {
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(b);
    };
    for (int r = 0; r < nc; ++r) {
      const int st = r % kStages, c = chunk(r);
      unsigned char* base = smem + st * St::kBytes;
      const float* gate = reinterpret_cast<const float*>(base + St::oG);
      const long long ch = static_cast<long long>(q.slot + c) * p.H + h;
      {  // dS as hi / lo operand columns
#pragma unroll
        for (int g = 0; g < KC / 32; ++g) {
          uint32_t hi[16], lo[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) split2(D[16 * g + i], hi[i], lo[i]);
          tmem_st16u(tb + tl + cDh + hf * (KC / 2) + 16 * g, hi);
          tmem_st16u(tb + tl + cDl + hf * (KC / 2) + 16 * g, lo);
        }
        tc::tmem_wait_st();
      }
      arrive(&bar.s);
      // dS's image in parts
      auto keep_state = [&](int from, int to) {
        if (row < VP) {
          float* img = w.dS + ch * state_image(p.V, K);
#pragma unroll
          for (int i = 0; i < KC / 4; ++i)
            if (i >= from && i < to)
              *reinterpret_cast<float4*>(img + image_at(VP, row, hf * KC / 4 + i)) =
                  make_float4(D[2 * i].x, D[2 * i].y, D[2 * i + 1].x, D[2 * i + 1].y);
        }
      };
      keep_state(0, 3 * KC / 32);
      if (!wait(&bar.full[st], (r / kStages) & 1) || !wait(&bar.z, r & 1)) break;
      tc::fence_after_sync();
      float2 x[16];  // W, then dX
      {  // W = beta Y + (beta w) Z
        float a[2][16], b[2][16];
        uint32_t hi[16], lo[16];
        tc::tmem_ld16(tb + tl + cZ + 32 * hf, a[0]);
        tc::tmem_ld16(tb + tl + cZ + 32 * hf + 16, a[1]);
        tc::tmem_ld16(tb + tl + cY + 32 * hf, b[0]);
        tc::tmem_ld16(tb + tl + cY + 32 * hf + 16, b[1]);
        tc::tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float2 be = *reinterpret_cast<const float2*>(gate + kGateBeta + 32 * hf + 2 * i);
          const float2 bw = *reinterpret_cast<const float2*>(gate + kGateW + 32 * hf + 2 * i);
          x[i] = f2_fma(bw, pair(a, i), f2_mul(be, pair(b, i)));
          split2(x[i], hi[i], lo[i]);
        }
        tmem_st16u(tb + tl + cW + 16 * hf, hi);
        tmem_st16u(tb + tl + cW + 32 + 16 * hf, lo);
        tc::tmem_wait_st();
      }
      arrive(&bar.w);
      keep_state(3 * KC / 32, 3 * KC / 16);
      if (!wait(&bar.dx, r & 1)) break;
      tc::fence_after_sync();
      {
        uint32_t hi[16], lo[16];
        {
          float a[2][16], b[2][16];
          tc::tmem_ld16(tb + tl + cZ + 32 * hf, a[0]);
          tc::tmem_ld16(tb + tl + cZ + 32 * hf + 16, a[1]);
          tc::tmem_ld16(tb + tl + cY + 32 * hf, b[0]);
          tc::tmem_ld16(tb + tl + cY + 32 * hf + 16, b[1]);
          tc::tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            x[i] = f2_add(x[i], f2_add(pair(a, i), pair(b, i)));
            split2(f2_mul(*reinterpret_cast<const float2*>(gate + kGateE + 32 * hf + 2 * i), x[i]), hi[i], lo[i]);
          }
        }
        tmem_st16u(tb + tl + cW + 16 * hf, hi);
        tmem_st16u(tb + tl + cW + 32 + 16 * hf, lo);
        tc::tmem_wait_st();
        arrive(&bar.wx);
        // while the state product runs: dX's low piece, dv over dO's tile
        if (!wait(&bar.dot, r & 1)) break;
#pragma unroll
        for (int i = 0; i < 16; ++i) split2(x[i], hi[i], lo[i]);
        if (row < VP) {
          char* img = w.dX + ch * token_piece(p.V);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<uint4*>(img + tc::chunk_off(row, 4 * hf + i)) =
                make_uint4(lo[4 * i], lo[4 * i + 1], lo[4 * i + 2], lo[4 * i + 3]);
        }
        if (live) {
          uint16_t* so = reinterpret_cast<uint16_t*>(base + St::oO) + 32 * hf * p.V + row;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            so[2 * i * p.V] = static_cast<uint16_t>(hi[i]);
            so[(2 * i + 1) * p.V] = static_cast<uint16_t>(hi[i] >> 16);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar.dv);
      }
      keep_state(3 * KC / 16, KC / 4);
      if (!wait(&bar.ds, r & 1)) break;
      tc::fence_after_sync();
      const float dec = gate[kGateEnd];
#pragma unroll
      for (int g = 0; g < KC / 32; ++g) {
        float a[2][16];
        tc::tmem_ld16(tb + tl + cDS + hf * KC + 32 * g, a[0]);
        tc::tmem_ld16(tb + tl + cDS + hf * KC + 32 * g + 16, a[1]);
        tc::tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) D[16 * g + i] = f2_fma(f2_bcast(dec), D[16 * g + i], pair(a, i));
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.empty[st]);
    }
    if (live && p.ds0 != nullptr) {
#pragma unroll
      for (int i = 0; i < KC; i += 4)
        *reinterpret_cast<float4*>(p.ds0 + srow + i) =
            make_float4(D[i / 2].x, D[i / 2].y, D[i / 2 + 1].x, D[i / 2 + 1].y);
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (*fail != 0u && tid == 0)  // the copies in flight land before the block ends
    for (int i = max(0, bar.issued - kStages); i < bar.issued; ++i)
      mbar_wait_bounded(&bar.full[i % kStages], (i / kStages) & 1, status);
  if (warp == kMma) {
    tc::tmem_relinquish();
    tc::tmem_dealloc(bar.taddr, 512);
  }
}

template <int K>
cudaError_t launch(const CUtensorMap& mk, const CUtensorMap& mq, const CUtensorMap& mo, const Params& p,
                   const TcBuffers& w, uint32_t* status, cudaStream_t st) {
  static unsigned long long mask = 0;
  const int bytes = kStages * Stage<K>::kBytes + static_cast<int>(sizeof(Bars));
  const cudaError_t e = static_cast<cudaError_t>(
      ensure_smem_attr(reinterpret_cast<const void*>(bwd_tc_kernel<K>), bytes, &mask));
  if (e != cudaSuccess) return e;
  bwd_tc_kernel<K><<<dim3(p.H, p.nseq), kThreads, bytes, st>>>(mk, mq, mo, p, w, status);
  return cudaGetLastError();
}

}  // namespace

cudaError_t tc_bwd_walk(const CUtensorMap& mk, const CUtensorMap& mq, const CUtensorMap& mo, const Params& p,
                        const TcBuffers& w, uint32_t* status, cudaStream_t st) {
  return p.K == 64 ? launch<64>(mk, mq, mo, p, w, status, st) : launch<128>(mk, mq, mo, p, w, status, st);
}

}  // namespace delta
}  // namespace emab
