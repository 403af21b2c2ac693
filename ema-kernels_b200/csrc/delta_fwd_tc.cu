// Gated delta rule, tensor-core family: the forward walk over a sequence's chunks.
//
// One block per (sequence, head) carries the state through the chunks.  Everything is held transposed: a
// tensor-memory lane is a value channel, so the chain of products
//
//   KS = S K^t  ->  X = V^t - exp(b) KS  ->  E = X + X (T - I)^t  ->  U = beta E  ->  S = exp(b_end) S + (w U) K
//
// is a chain of M = 128 MMAs whose left operand (S, X, U) the epilogue threads write straight back to tensor memory
// -- no shared-memory round trip and no transpose -- and whose right operands K, Q, T, P are the tiles as
// loaded.  Operands that are not bf16 by nature are hi + lo pairs (delta_tc.cuh): 2 products for S K^t and S Q^t, 3
// for E and U P^t; w U, whose rounding stays in the state, is three pieces.  (o = scale exp(b) S Q^t
// + U P^t ends in bf16, but where keys repeat its two terms cancel: hi parts alone left it 1e-2 off there.)
//
// Bound: the chain's latency, 6000 cycles a chunk at dstate 128 (16384 tokens of 32 heads of 128: 856 us, 3 % more with the
// state product in one piece; 40 sequences, 8111 tokens of 16 heads: 117): three
// dependent MMA groups (about 1000, 640 and 950 cycles) with an epilogue after each (600, 750 and 980) and the hand-overs
// between them; the products for o run in their shadow.  A training forward with a block on most SMs is near its bytes
// instead: it writes S, E and o, 128 KB a chunk and head, and reads 96 (4 x 4096 x 32: 320 us, 5.8 TB/s; 250 without S).
// Roles: warps 0-7 the chain's epilogues (warp w: lanes 32 (w % 4), 32 (w / 4) .. of every 64 columns; the fp32 state lives
// in their registers), warps 8-11 the output, warp 12 issues the MMAs, warp 13 the loads (TMA for K, Q, V; bulk copies for
// the images), two stages deep, warp 14 E's copies to memory.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "delta_host.h"
#include "delta_tc.cuh"
#include "ema_scan_dispatch.h"

namespace emab {
namespace delta {
namespace {

constexpr int kEpi = 8;                      // epilogue warps
constexpr int kOut = 4;                      // output warps
constexpr int kMma = 12, kLoad = 13, kStore = 14;  // (15 only fills its warpgroup)
constexpr int kThreads = 16 * 32;
// registers a thread, by warpgroup: 2 epilogue, output, MMA and loads; 4 x 128 at launch
constexpr int kRegEpi = 160, kRegOut = 120, kRegCtl = 72;
static_assert(2 * kRegEpi + kRegOut + kRegCtl == 4 * 128, "register split");
constexpr int kStages = 2;
constexpr int kKeep = 3 * 2 * kTile;
constexpr int kReg = 128 * 128;              // 64 query rows, then 64 key rows of 64 columns

// tensor-memory columns.  An MMA step with its left operand in tensor memory takes about 32 + N / 2 cycles here, so what
// can share one runs as N = 128: X [T hi; T lo]^t.
constexpr uint32_t cX = 0;     // X hi, lo; then w U hi, mid, lo (32 columns each)
constexpr uint32_t cKS = 128;  // K S; then X (T hi)^t; then U: hi and lo of tokens 0-31, hi and lo of 32-63 (16 columns each)
constexpr uint32_t cPU = 192;  // X (T lo)^t; then U P^t
constexpr uint32_t cDS = 256;  // Q S (64 columns), read before the state's product needs the place
constexpr uint32_t cSh = 384;  // S hi (K / 2 columns)
constexpr uint32_t cSl = 448;  // S lo

struct Bars {
  uint64_t full[kStages], empty[kStages];
  uint64_t ks, qs, e, ds[2], pu;  // MMA groups done (ds: 64 state columns each)
  uint64_t s[2], x, wu, u;  // epilogues done: state (64 columns each), X, w U and U ready
  uint64_t q, o;           // Q S, U P read
  uint64_t ek, ekfree;     // E's pieces staged, and on their way to memory
  uint64_t out_sync;       // meeting of the output warps (bounded, unlike a barrier instruction)
  uint64_t drain;          // MMAs still in flight after a failed wait
  uint32_t taddr, fail;
  int issued;  // chunks whose loads were issued
};

__device__ __forceinline__ float2 pair(const float (&a)[2][16], int i) {
  return make_float2(a[i / 8][(2 * i) % 16], a[i / 8][(2 * i) % 16 + 1]);
}

template <int K>
struct Stage {
  static constexpr int oKQ = 0;                     // per 64 columns: 64 rows of Q, 64 of K
  static constexpr int oT = oKQ + (K / 64) * kReg;  // T hi, lo
  static constexpr int oP = oT + 2 * kTile;         // P hi, lo
  static constexpr int oV = oP + 2 * kTile;         // V: 64 rows of V channels, as they are; later o in the same places
  static constexpr int oG = oV + 64 * 128 * 2;
  static constexpr int kBytes = (oG + kGateFloats * 4 + 1023) / 1024 * 1024;
};

template <int K, bool KEEP>
__global__ void __launch_bounds__(kThreads, 1)
    fwd_tc_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mq,
                  const __grid_constant__ CUtensorMap mv, const Params p, const TcBuffers w, uint32_t* status) {
  using St = Stage<K>;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* keep = smem + kStages * St::kBytes;  // KEEP: E's pieces, up to three of 16 KB
  Bars& bar = *reinterpret_cast<Bars*>(keep + (KEEP ? kKeep : 0));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int h = blockIdx.x, n = blockIdx.y, gr = h / (p.H / p.G);
  const Seq q = seq_at(p, n);
  const int nc = (q.len + kC - 1) / kC;
  const int VP = pad_channels(p.V);
  volatile uint32_t* fail = &bar.fail;

  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bar.full[i], 1);
      mbar_init(&bar.empty[i], kEpi + kOut);
    }
    mbar_init(&bar.ks, 1);
    mbar_init(&bar.e, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.ds[i], 1);
      mbar_init(&bar.s[i], kEpi);
    }
    mbar_init(&bar.x, kEpi);
    mbar_init(&bar.wu, kEpi);
    mbar_init(&bar.u, kEpi);
    mbar_init(&bar.q, kOut);
    mbar_init(&bar.o, kOut);
    mbar_init(&bar.qs, 1);
    mbar_init(&bar.pu, 1);
    mbar_init(&bar.out_sync, kOut);
    mbar_init(&bar.ek, kEpi);
    mbar_init(&bar.ekfree, 1);
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
  // a wait that runs out marks the block as failed; every role then leaves its loop at the next wait, warps as a whole
  auto wait1 = [&](uint64_t* b, uint32_t parity) { return chain_wait(b, parity, status, fail); };
  auto wait = [&](uint64_t* b, uint32_t parity) { return chain_wait_warp(b, parity, status, fail); };

  if (warp >= kMma) {
    set_regs_down<kRegCtl>();
    if (warp == kLoad && lane == 0) {  // ---- loads
      int c = 0;
      for (; c < nc; ++c) {
        const int st = c % kStages;
        if (c >= kStages && !wait1(&bar.empty[st], (c / kStages - 1) & 1)) break;
        unsigned char* base = smem + st * St::kBytes;
        const long long ch = static_cast<long long>(q.slot + c) * p.H + h;
        const uint32_t vbytes = 64u * p.V * 2u;
        mbar_arrive_expect_tx(&bar.full[st], (K / 64) * kReg + 4 * kTile + vbytes + kGateFloats * 4);
        for (int r = 0; r < K / 64; ++r) {
          tma_load_4d(base + St::oKQ + r * kReg, &mq, &bar.full[st], 64 * r, gr, q.t0 + c * kC, q.b);
          tma_load_4d(base + St::oKQ + r * kReg + kTile, &mk, &bar.full[st], 64 * r, gr, q.t0 + c * kC, q.b);
        }
        bulk_g2s(base + St::oT, w.T + ch * 2 * kTile, 2 * kTile, &bar.full[st]);
        bulk_g2s(base + St::oP, w.P + ch * 2 * kTile, 2 * kTile, &bar.full[st]);
        tma_load_4d(base + St::oV, &mv, &bar.full[st], 0, h, q.t0 + c * kC, q.b);
        bulk_g2s(base + St::oG, w.gates + ch * kGateFloats, kGateFloats * 4, &bar.full[st]);
      }
      bar.issued = c;
    }
    if (KEEP && warp == kStore && lane == 0) {  // ---- E's pieces
      for (int c = 0; c < nc && wait1(&bar.ek, c & 1); ++c) {
        bulk_s2g(w.E + (static_cast<long long>(q.slot + c) * p.H + h) * 3 * token_piece(p.V), keep, 3 * VP * 128);
        bulk_commit();
        bulk_wait_read_all();
        mbar_arrive(&bar.ekfree);
      }
      bulk_wait_all();
    }
    if (warp == kMma) {  // ---- MMAs
      constexpr uint32_t id64 = tc::idesc_bf16(128, 64, false, false);
      constexpr uint32_t id128 = tc::idesc_bf16(128, 128, false, false);
      constexpr uint32_t idK = tc::idesc_bf16(128, 64, false, true);
      for (int c = 0; c < nc; ++c) {
        const int st = c % kStages;
        unsigned char* base = smem + st * St::kBytes;
        const uint32_t sb = smem_u32(base);
        bool ok = wait(&bar.full[st], (c / kStages) & 1);
        const int have = q.len - c * kC;
        if (ok && have < kC && p.cu != nullptr) {  // rows of the next sequence
          zero_rows(base + St::oKQ, K / 64, kReg, have);
          zero_rows(base + St::oKQ + kTile, K / 64, kReg, have);
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (ok && c > 0) ok = wait(&bar.pu, (c - 1) & 1);  // U has been read where K S lands
        if (!ok) break;
        const uint64_t dq = tc::smem_desc_sw128(sb + St::oKQ, 16, 1024);
        const uint64_t dk = tc::smem_desc_sw128(sb + St::oKQ + kTile, 16, 1024);
        const uint64_t dkn = tc::smem_desc_sw128(sb + St::oKQ + kTile, kReg, 1024);
        const uint64_t dt = tc::smem_desc_sw128(sb + St::oT, 16, 1024);  // 64 rows hi, 64 rows lo
        const uint64_t dp = tc::smem_desc_sw128(sb + St::oP, 16, 1024);
        const uint64_t dpl = tc::smem_desc_sw128(sb + St::oP + kTile, 16, 1024);
        auto kstep = [](int s) { return static_cast<uint64_t>(((s >> 2) * kReg + (s & 3) * 32) >> 4); };
        auto jstep = [](int s) { return static_cast<uint64_t>((s * 32) >> 4); };
        auto nstep = [](int s) { return static_cast<uint64_t>((s * 2048) >> 4); };
        auto ucol = [](int s) { return static_cast<uint32_t>((s >> 1) * 32 + (s & 1) * 8); };
#pragma unroll
        for (int g = 0; g < K / 64; ++g) {
          ok = ok && wait(&bar.s[g], c & 1);
          if (!ok) break;
          tc::fence_after_sync();
          if (elect_one()) {
#pragma unroll
            for (int s = 4 * g; s < 4 * g + 4; ++s) mma_ts(tb + cKS, tb + cSh + 8 * s, dk + kstep(s), id64, s > 0);
#pragma unroll
            for (int s = 4 * g; s < 4 * g + 4; ++s) mma_ts(tb + cKS, tb + cSl + 8 * s, dk + kstep(s), id64, true);
            if (g == K / 64 - 1) tc::mma_commit(&bar.ks);
          }
          __syncwarp();
        }
        if (!ok) break;
        if (elect_one()) {
#pragma unroll
          for (int s = 0; s < K / 16; ++s) mma_ts(tb + cDS, tb + cSh + 8 * s, dq + kstep(s), id64, s > 0);
#pragma unroll
          for (int s = 0; s < K / 16; ++s) mma_ts(tb + cDS, tb + cSl + 8 * s, dq + kstep(s), id64, true);
          tc::mma_commit(&bar.qs);
        }
        __syncwarp();
        if (c > 0 && !wait(&bar.o, (c - 1) & 1)) break;  // U P has been read where X (T lo)^t goes
        if (!wait(&bar.x, c & 1)) break;
        tc::fence_after_sync();
        if (elect_one()) {
#pragma unroll
          for (int s = 0; s < 4; ++s) mma_ts(tb + cKS, tb + cX + 8 * s, dt + jstep(s), id128, s > 0);
#pragma unroll
          for (int s = 0; s < 4; ++s) mma_ts(tb + cKS, tb + cX + 32 + 8 * s, dt + jstep(s), id64, true);
          tc::mma_commit(&bar.e);
        }
        __syncwarp();
        if (!wait(&bar.q, c & 1) || !wait(&bar.wu, c & 1)) break;
        tc::fence_after_sync();
        if (elect_one()) {
#pragma unroll
          for (int g = 0; g < K / 64; ++g) {  // a tile of K each, so that the first columns' epilogue starts earlier
            const uint64_t kg = dkn + ((g * kReg) >> 4);
#pragma unroll
            for (int s = 0; s < 4; ++s) mma_ts(tb + cDS + 64 * g, tb + cX + 8 * s, kg + nstep(s), idK, s > 0);
#pragma unroll
            for (int s = 0; s < 4; ++s) mma_ts(tb + cDS + 64 * g, tb + cX + 32 + 8 * s, kg + nstep(s), idK, true);
#pragma unroll
            for (int s = 0; s < 4; ++s) mma_ts(tb + cDS + 64 * g, tb + cX + 64 + 8 * s, kg + nstep(s), idK, true);
            tc::mma_commit(&bar.ds[g]);
          }
        }
        __syncwarp();
        if (!wait(&bar.u, c & 1)) break;
        tc::fence_after_sync();
        if (elect_one()) {
#pragma unroll
          for (int s = 0; s < 4; ++s) mma_ts(tb + cPU, tb + cKS + ucol(s), dp + jstep(s), id64, s > 0);
#pragma unroll
          for (int s = 0; s < 4; ++s) mma_ts(tb + cPU, tb + cKS + 16 + ucol(s), dp + jstep(s), id64, true);
#pragma unroll
          for (int s = 0; s < 4; ++s) mma_ts(tb + cPU, tb + cKS + ucol(s), dpl + jstep(s), id64, true);
          tc::mma_commit(&bar.pu);
        }
        __syncwarp();
      }
      if (*fail != 0u && elect_one()) {
        tc::mma_commit(&bar.drain);
        mbar_wait_bounded(&bar.drain, 0, status);
      }
      __syncwarp();
    }
  } else if (warp >= kEpi) {  // ---- o = scale exp(b) Q S + P U
    set_regs_down<kRegOut>();
    const int row = 32 * (warp & 3) + lane;
    const uint32_t tl = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const bool live = row < p.V;
    const int pieces = p.V / 8;  // 16-byte pieces of a row
    for (int c = 0; c < nc; ++c) {
      const int st = c % kStages;
      unsigned char* base = smem + st * St::kBytes;
      const float* gate = reinterpret_cast<const float*>(base + St::oG);
      const int have = min(kC, q.len - c * kC);
      if (!wait(&bar.full[st], (c / kStages) & 1) || !wait(&bar.qs, c & 1)) break;
      tc::fence_after_sync();
      float2 f[32];  // token pairs
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        float a[2][16];
        tc::tmem_ld16(tb + tl + cDS + 32 * g, a[0]);
        tc::tmem_ld16(tb + tl + cDS + 32 * g + 16, a[1]);
        tc::tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i)
          f[16 * g + i] = f2_mul(f2_mul(f2_bcast(-p.scale), *reinterpret_cast<const float2*>(gate + kGateE + 32 * g + 2 * i)),
                                 pair(a, i));
      }
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.q);
      if (!wait(&bar.pu, c & 1)) break;
      tc::fence_after_sync();
      uint32_t o[32];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float a[16];
        tc::tmem_ld16(tb + tl + cPU + 16 * g, a);
        tc::tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 8; ++i)
          o[8 * g + i] = pack_pair<__nv_bfloat16>(f2_add(f[8 * g + i], make_float2(a[2 * i], a[2 * i + 1])));
      }
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.o);
      // over V's tile, which X has consumed; then out in whole pieces
      if (live) {
        uint16_t* so = reinterpret_cast<uint16_t*>(base + St::oV) + row;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          so[2 * i * p.V] = static_cast<uint16_t>(o[i]);
          so[(2 * i + 1) * p.V] = static_cast<uint16_t>(o[i] >> 16);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.out_sync);
      if (!wait(&bar.out_sync, c & 1)) break;
      {
        const int pc = lane & 15, t0 = 2 * (warp - kEpi) + (lane >> 4);
        const uint4* src = reinterpret_cast<const uint4*>(base + St::oV);
        __nv_bfloat16* dst = row_of<__nv_bfloat16>(p.o, p.vo, q.b, q.t0 + c * kC, h) + 8 * pc;
        if (pc < pieces) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int t = t0 + 8 * i;
            if (t < have) __stcs(reinterpret_cast<uint4*>(dst + t * p.vo.t), src[t * pieces + pc]);
          }
        }
      }
      fence_proxy_async_smem();  // the stage's next load overwrites what was written here
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.empty[st]);
    }
  } else {  // ---- the chain's epilogues
    set_regs_up<kRegEpi>();
    constexpr int KC = K / 2;  // state columns of a thread: 32 hf .. of each 64
    const int row = 32 * (warp & 3) + lane, hf = warp >> 2;
    const uint32_t tl = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const bool live = row < p.V;
    float2 S[KC / 2];
    const long long srow = ((static_cast<long long>(n) * p.H + h) * p.V + row) * K + 32 * hf;
#pragma unroll
    for (int i = 0; i < KC; i += 4) {
      const float4 f = (live && p.s0 != nullptr) ? *reinterpret_cast<const float4*>(p.s0 + srow + i + (i & 32))
                                                  : make_float4(0, 0, 0, 0);
      S[i / 2] = make_float2(f.x, f.y), S[i / 2 + 1] = make_float2(f.z, f.w);
    }
    auto arrive = [&](uint64_t* b) {
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(b);
    };
    // 32 columns of the state as hi / lo operand columns
    auto publish = [&](int g) {
      uint32_t hi[16], lo[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) split2(S[16 * g + i], hi[i], lo[i]);
      tmem_st16u(tb + tl + cSh + 32 * g + 16 * hf, hi);
      tmem_st16u(tb + tl + cSl + 32 * g + 16 * hf, lo);
      tc::tmem_wait_st();
      arrive(&bar.s[g]);
    };
#pragma unroll
    for (int g = 0; g < KC / 32; ++g) publish(g);
    for (int c = 0; c < nc; ++c) {
      // KEEP: the state's image, a part in every gap of the chain (all at once the stores hold up the loads behind them)
      auto keep_state = [&](int from, int to) {
        if (KEEP && row < VP) {
          float* img = w.S + (static_cast<long long>(q.slot + c) * p.H + h) * state_image(p.V, K);
#pragma unroll
          for (int i = 0; i < KC / 4; ++i)
            if (i >= from && i < to)
              *reinterpret_cast<float4*>(img + image_at(VP, row, 8 * hf + i + (i & 8))) =
                  make_float4(S[2 * i].x, S[2 * i].y, S[2 * i + 1].x, S[2 * i + 1].y);
        }
      };
      const int st = c % kStages;
      const unsigned char* base = smem + st * St::kBytes;
      const float* gate = reinterpret_cast<const float*>(base + St::oG);
      const __nv_bfloat16* sv = reinterpret_cast<const __nv_bfloat16*>(base + St::oV) + 32 * hf * p.V + (live ? row : 0);
      const int have = min(kC, q.len - c * kC);
      if (!wait(&bar.full[st], (c / kStages) & 1)) break;
      // X = V - exp(b) K S, tokens 32 hf ..
      float v[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = to_f32(sv[i * p.V]);
      if (!live || have < kC) {  // lanes past headdim, rows past the sequence
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = (live && 32 * hf + i < have) ? v[i] : 0.f;
      }
      keep_state(0, KC / 16);
      if (!wait(&bar.ks, c & 1)) break;
      tc::fence_after_sync();
      float2 x[16];
      {
        float a[2][16];
        tc::tmem_ld16(tb + tl + cKS + 32 * hf, a[0]);
        tc::tmem_ld16(tb + tl + cKS + 32 * hf + 16, a[1]);
        tc::tmem_wait_ld();
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float2 e = *reinterpret_cast<const float2*>(gate + kGateE + 32 * hf + 2 * i);  // -exp(b)
          x[i] = f2_fma(e, pair(a, i), make_float2(v[2 * i], v[2 * i + 1]));
          split2(x[i], hi[i], lo[i]);
        }
        tmem_st16u(tb + tl + cX + 16 * hf, hi);
        tmem_st16u(tb + tl + cX + 32 + 16 * hf, lo);
        tc::tmem_wait_st();
      }
      arrive(&bar.x);
      keep_state(KC / 16, 3 * KC / 16);
      // U = beta E; first w U, which the state waits for
      if (!wait(&bar.e, c & 1)) break;
      tc::fence_after_sync();
      {
        float2 e[16];
        uint32_t hi[16], lo[16];
        {
          float a[2][16], b[2][16];
          tc::tmem_ld16(tb + tl + cKS + 32 * hf, a[0]);
          tc::tmem_ld16(tb + tl + cKS + 32 * hf + 16, a[1]);
          tc::tmem_ld16(tb + tl + cPU + 32 * hf, b[0]);
          tc::tmem_ld16(tb + tl + cPU + 32 * hf + 16, b[1]);
          tc::tmem_wait_ld();
          uint32_t mid[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            e[i] = f2_add(x[i], f2_add(pair(a, i), pair(b, i)));
            split3(f2_mul(e[i], *reinterpret_cast<const float2*>(gate + kGateW + 32 * hf + 2 * i)), hi[i], mid[i], lo[i]);
          }
          tmem_st16u(tb + tl + cX + 16 * hf, hi);
          tmem_st16u(tb + tl + cX + 32 + 16 * hf, mid);
          tmem_st16u(tb + tl + cX + 64 + 16 * hf, lo);
          tc::tmem_wait_st();
        }
        arrive(&bar.wu);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          split2(f2_mul(e[i], *reinterpret_cast<const float2*>(gate + kGateBeta + 32 * hf + 2 * i)), hi[i], lo[i]);
        }
        tmem_st16u(tb + tl + cKS + 32 * hf, hi);
        tmem_st16u(tb + tl + cKS + 32 * hf + 16, lo);
        tc::tmem_wait_st();
        arrive(&bar.u);
        if (KEEP) {  // E's pieces, while the state product runs: staged, then out in one copy
          if (c > 0 && !wait(&bar.ekfree, (c - 1) & 1)) break;
          if (row < VP) {
            const int pc = VP * 128;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t m[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) split3(e[4 * i + k], hi[k], m[k], lo[k]);
              unsigned char* to = keep + tc::chunk_off(row, 4 * hf + i);
              *reinterpret_cast<uint4*>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
              *reinterpret_cast<uint4*>(to + pc) = make_uint4(m[0], m[1], m[2], m[3]);
              *reinterpret_cast<uint4*>(to + 2 * pc) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar.ek);
        }
      }
      // S = exp(b_end) S + (w U) K
      keep_state(3 * KC / 16, KC / 4);
      const float dec = gate[kGateEnd];
      bool ok = true;
#pragma unroll
      for (int g = 0; g < KC / 32; ++g) {
        ok = ok && wait(&bar.ds[g], c & 1);
        if (!ok) break;
        tc::fence_after_sync();
        float a[2][16];
        tc::tmem_ld16(tb + tl + cDS + 64 * g + 32 * hf, a[0]);
        tc::tmem_ld16(tb + tl + cDS + 64 * g + 32 * hf + 16, a[1]);
        tc::tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) S[16 * g + i] = f2_fma(f2_bcast(dec), S[16 * g + i], pair(a, i));
        publish(g);
      }
      if (!ok) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.empty[st]);
    }
    if (live && p.s1 != nullptr) {
#pragma unroll
      for (int i = 0; i < KC; i += 4)
        *reinterpret_cast<float4*>(p.s1 + srow + i + (i & 32)) =
            make_float4(S[i / 2].x, S[i / 2].y, S[i / 2 + 1].x, S[i / 2 + 1].y);
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

template <int K, bool KEEP>
cudaError_t launch(const CUtensorMap& mk, const CUtensorMap& mq, const CUtensorMap& mv, const Params& p,
                   const TcBuffers& w, uint32_t* status, cudaStream_t st) {
  static unsigned long long mask = 0;
  constexpr int bytes = kStages * Stage<K>::kBytes + (KEEP ? kKeep : 0) + static_cast<int>(sizeof(Bars));
  static_assert(bytes <= kMaxDynSmem, "shared memory");
  const cudaError_t e = static_cast<cudaError_t>(
      ensure_smem_attr(reinterpret_cast<const void*>(fwd_tc_kernel<K, KEEP>), bytes, &mask));
  if (e != cudaSuccess) return e;
  fwd_tc_kernel<K, KEEP><<<dim3(p.H, p.nseq), kThreads, bytes, st>>>(mk, mq, mv, p, w, status);
  return cudaGetLastError();
}

}  // namespace

cudaError_t tc_fwd_walk(const CUtensorMap& mk, const CUtensorMap& mq, const CUtensorMap& mv, const Params& p,
                        const TcBuffers& w, uint32_t* status, cudaStream_t st) {
  const bool keep = w.S != nullptr;
  if (p.K == 64)
    return keep ? launch<64, true>(mk, mq, mv, p, w, status, st) : launch<64, false>(mk, mq, mv, p, w, status, st);
  return keep ? launch<128, true>(mk, mq, mv, p, w, status, st) : launch<128, false>(mk, mq, mv, p, w, status, st);
}

}  // namespace delta
}  // namespace emab
