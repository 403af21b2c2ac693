// Shared pieces of the tensor-core (tcgen05) kernels of the gated delta rule: the buffers between them as
// operand images, and 32-bit precision out of bf16 products.
//
// Precision.  States, gate gradients and every other fp32 output have to be good to fp32's own order, so a product's
// operand that is not bf16 by nature enters as two bf16 pieces, hi = bf16(x), lo = bf16(x - hi), x = hi + lo to
// 2^-16, or as three (2^-24) where the sums that follow cancel: what the gate gradients are summed from (E, dX, S0 and
// dS1 in the gradient kernel).  A bf16 tensor times a pair is two MMAs, a pair times a pair three (lo lo is dropped), three
// pieces times three six.  T enters without its unit diagonal, which is added in fp32 from the operand itself.
//
// Images.  T and P lie in global memory as the 128-byte swizzled bf16 tiles that shared memory wants (rows of 64 bf16,
// 16-byte chunk c of row r at c ^ (r % 8)), so that a plain bulk copy stages them: 64 x 64, row = token i, column =
// token j, hi then lo (8 KB each); E and dX likewise, row = value channel, column = token, one piece after another.
// S and dS are fp32, for a thread that owns the row of a value channel: four columns after four columns, each with all
// the rows, so that a warp stores 512 bytes at a time.
#pragma once

#include "delta_common.cuh"
#include "tc_common.cuh"

namespace emab {
namespace delta {

constexpr int kTile = kC * 128;  // bytes of a 64-row, 128-byte-row region
// gate record of a (chunk, head), 64 each: -exp(b_i), beta_i w_i, beta_i, b_i hi, key_j = exp(b_r - b_j), w_j = exp(b_end -
// b_j), b_i lo; then exp(b_end) and, as bits 0, 8, 16, 24 of a word, the wide groups.  exp(b_i - b_j) = exp(b_i - b_r) key_j, r
// the first token of j's 16-token group, except where a group is wide (its gates sum to more than kWideSpan, a reset
// among them): there it is taken as it is.
constexpr float kWideSpan = 60.f;
constexpr int kGateFloats = 464;
constexpr uint32_t kStatusTmem = 0x200u;  // device status: a block that owns all of tensor memory did not get base 0
constexpr int kGateE = 0, kGateW = 64, kGateBeta = 128, kGateB = 192, kGateKey = 256, kGateTail = 320, kGateBLo = 384,
              kGateEnd = 448, kGateWide = 449;

struct TcBuffers {
  float* gates;      // kGateFloats per (slot, head)
  char* T;           // T - I: hi, lo
  char* P;           // hi, lo
  float* S;          // state entering the chunk (null: not kept)
  char* E;           // hi, mid, lo (null: not kept)
  float* dS;         // gradient of the state at the chunk's end
  char* dX;          // lo alone: dv is its hi
};

__host__ __device__ inline int pad_channels(int V) { return V <= 64 ? 64 : 128; }
// Floats of an image, and the place of columns 4 piece .. 4 piece + 3 of a row in it.
__host__ __device__ inline size_t state_image(int V, int K) { return static_cast<size_t>(pad_channels(V)) * K; }
// Bytes of one piece of E or dX.
__host__ __device__ inline size_t token_piece(int V) { return static_cast<size_t>(pad_channels(V)) * kC * 2; }
__device__ __forceinline__ int image_at(int VP, int row, int piece) { return (piece * VP + row) * 4; }

// bf16 pair (x, y) -> packed hi and packed lo.
__device__ __forceinline__ void split2(float2 v, uint32_t& hi, uint32_t& lo) {
  hi = pack_pair<__nv_bfloat16>(v);
  lo = pack_pair<__nv_bfloat16>(f2_fma(cvt_pair<__nv_bfloat16>(hi), make_float2(-1.f, -1.f), v));
}

// Three pieces.
__device__ __forceinline__ void split3(float2 v, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  hi = pack_pair<__nv_bfloat16>(v);
  const float2 r = f2_fma(cvt_pair<__nv_bfloat16>(hi), make_float2(-1.f, -1.f), v);
  mid = pack_pair<__nv_bfloat16>(r);
  lo = pack_pair<__nv_bfloat16>(f2_fma(cvt_pair<__nv_bfloat16>(mid), make_float2(-1.f, -1.f), r));
}

// D[tmem] (+)= A[tmem] B^T for one K = 16 step: A's 16 columns are 8 packed 32-bit tensor-memory columns.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b_desc), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
      : "memory");
}

// One lane of a converged warp.  MMA issue stands under this and takes warp-uniform operands (descriptors from the loop
// counter and the shared-memory base, tensor-memory addresses from a base of zero): operands the compiler cannot
// prove uniform cost a few tens of cycles each, more than the MMA they feed.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0u;
}

// Shared-memory descriptors of 128-byte swizzled tiles with 1024 bytes from one 8-row group to the next differ only in
// their low word (address and leading offset, both in 16 bytes); the high one is a constant.
__device__ __forceinline__ uint32_t desc_lo(uint32_t smem_addr, uint32_t lbo_bytes) {
  return ((smem_addr >> 4) & 0x3fffu) | (((lbo_bytes >> 4) & 0x3fffu) << 16);
}
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}\n" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(static_cast<uint32_t>(accumulate)), "r"(kDescHi)
      : "memory");
}

__device__ __forceinline__ void mma_ts_lo(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(idesc), "r"(static_cast<uint32_t>(accumulate)), "r"(kDescHi)
      : "memory");
}

// 32 lanes x 8 and x 16 columns of raw 32-bit words.
__device__ __forceinline__ void tmem_st8u(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st16u(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// A tile on its way to the L2 cache.
__device__ __forceinline__ void tma_prefetch_4d(const void* map, int x, int y, int z, int w) {
  asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global.tile [%0, {%1, %2, %3, %4}];" ::"l"(map), "r"(x), "r"(y), "r"(z),
               "r"(w)
               : "memory");
}
// Shared to global memory; the caller commits and waits.
__device__ __forceinline__ void bulk_s2g(void* dst, const void* src_smem, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(src_smem)), "r"(bytes)
               : "memory");
}

// A warpgroup's share of the registers the block was launched with; all its warps call it.  N is at least (up), at
// most (down) what it has: the other way round is an illegal instruction.
template <int N>
__device__ __forceinline__ void set_regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void set_regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Bounded wait of the chain's roles: plain polls, without suspending the thread (3 % of the gradient kernel against
// try_wait).  The first poll stands alone: a phase that is complete already (most are) costs that and a vote, no clock and
// no look at the block's failure word.
__device__ __forceinline__ bool mbar_test_wait(uint64_t* bar, uint32_t phase) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(phase)
      : "memory");
  return ok != 0;
}
constexpr long long kWaitLimitCycles = 2000000000ll;  // about a second
__device__ __forceinline__ bool chain_wait_slow(uint64_t* bar, uint32_t phase, uint32_t* status, volatile uint32_t* fail) {
  const long long t0 = clock64();
  while (!mbar_test_wait(bar, phase)) {
    if (*fail != 0u) return false;
    if (clock64() - t0 > kWaitLimitCycles) {
      atomicOr(status, kStatusTmaTimeout);
      *fail = 1u;
      return false;
    }
  }
  return true;
}
// By one thread.
__device__ __forceinline__ bool chain_wait(uint64_t* bar, uint32_t phase, uint32_t* status, volatile uint32_t* fail) {
  return mbar_test_wait(bar, phase) || chain_wait_slow(bar, phase, status, fail);
}
// By a whole warp, with one answer.
__device__ __forceinline__ bool chain_wait_warp(uint64_t* bar, uint32_t phase, uint32_t* status, volatile uint32_t* fail) {
  if (__all_sync(0xffffffffu, mbar_test_wait(bar, phase))) return true;
  return __all_sync(0xffffffffu, chain_wait_slow(bar, phase, status, fail)) != 0;
}

// Zero rows [from, 64) of `regions` 64-row regions `stride` bytes apart (one warp).
__device__ __forceinline__ void zero_rows(unsigned char* base, int regions, int stride, int from) {
  const int n = (kC - from) * 8;
  for (int r = 0; r < regions; ++r)
    for (int i = threadIdx.x & 31; i < n; i += 32)
      *reinterpret_cast<uint4*>(base + r * stride + from * 128 + i * 16) = make_uint4(0, 0, 0, 0);
}

}  // namespace delta
}  // namespace emab
