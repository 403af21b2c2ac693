// The gated delta rule, recurrent form: a few tokens of every row on a cache of fp32 states, in place.
//
//   S <- a S + beta (v - a S k) k^T,   o = scale S q,   a = exp(g)
//
// Every row of S (one value channel, dstate numbers) evolves by itself given k, q: with sk = S_row . k and
// sq = S_row . q taken from the state before the token,
//   u = beta (v - a sk),   S_row <- a S_row + u k,   o = scale (a sq + u (k . q)),
// so one pass over the registers gives both sums and the update needs no second one.
//
// Bound: HBM, 8 bytes per state element and call (read + write); the products are 6 flops per element
// (256 rows of 32 heads of 128 x 128: 163 us, 6.6 TB/s, the copy's rate; one row 2.6 us, a launch's latency).
// A warp owns kRows rows of one (batch row, head) in registers, a lane dstate / 32 consecutive elements of each
// (512-byte row reads), so all of a warp's state is in flight at once and the tokens of a call run on
// it without touching memory.  The 2 kRows sums of a token are reduced together by a transposed butterfly:
// 16 values over 32 lanes in 16 shuffles instead of 80.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdio>

#include "delta_b200.h"
#include "ema_common.cuh"
#include "ema_scan_dispatch.h"

namespace emab {
void set_last_error(const char* msg);

namespace dstep {

constexpr int kRows = 8;   // state rows of a warp
constexpr int kWarps = 4;  // warps of a block
constexpr unsigned kAll = 0xffffffffu;

struct Params {
  int T, H, G, V, slots;
  float scale;
  const void* q;  long long qb, qt, qg;
  const void* k;  long long kb, kt, kg;
  const void* v;  long long vb, vt, vh;
  const float* g;
  const float* beta;
  float* s;       long long ss, sh;
  const int32_t* index;
  void* o;        long long ob, ot, oh;
};

// Sums of 16 values over the warp: lane l gets the total of value l / 2.
__device__ __forceinline__ float sum16(float (&x)[16], int lane) {
#pragma unroll
  for (int o = 16, n = 8; n >= 1; o >>= 1, n >>= 1) {
    const bool up = (lane & o) != 0;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float give = up ? x[i] : x[i + n];
      x[i] = (up ? x[i + n] : x[i]) + __shfl_xor_sync(kAll, give, o);
    }
  }
  return x[0] + __shfl_xor_sync(kAll, x[0], 1);
}

template <class T, int KPL>  // dstate = 32 KPL
__global__ void __launch_bounds__(kWarps * 32) step_kernel(const Params p) {
  constexpr int K = 32 * KPL;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = blockIdx.y, b = blockIdx.z, gr = h / (p.H / p.G);
  const int r0 = (blockIdx.x * kWarps + warp) * kRows;
  grid_dep_wait();
  grid_dep_release();
  if (r0 >= p.V) return;
  T* o = static_cast<T*>(p.o) + b * p.ob + h * p.oh;
  const int slot = p.index != nullptr ? p.index[b] : b;
  if (slot < 0 || slot >= p.slots) {  // a row without a state
    if (lane < kRows && r0 + lane < p.V)
      for (int t = 0; t < p.T; ++t) o[t * p.ot + r0 + lane] = from_f32<T>(0.f);
    return;
  }
  float* s = p.s + slot * p.ss + h * p.sh + static_cast<long long>(r0) * K + lane * KPL;
  const T* q = static_cast<const T*>(p.q) + b * p.qb + gr * p.qg + lane * KPL;
  const T* k = static_cast<const T*>(p.k) + b * p.kb + gr * p.kg + lane * KPL;
  const T* v = static_cast<const T*>(p.v) + b * p.vb + h * p.vh;
  float S[kRows][KPL];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    if (r0 + r < p.V) load_pack<float, KPL>(s + r * K, S[r]);
    else
#pragma unroll
      for (int i = 0; i < KPL; ++i) S[r][i] = 0.f;
  }
  const int mine = lane >> 1;                // the sum this lane holds: S_r . k of row r (< 8), S_r . q of row r - 8
  const int row = r0 + (mine & (kRows - 1));  // its state row
  for (int t = 0; t < p.T; ++t) {
    float kv[KPL], qv[KPL];
    load_pack<T, KPL>(k + t * p.kt, kv);
    load_pack<T, KPL>(q + t * p.qt, qv);
    const float vr = row < p.V ? to_f32(v[t * p.vt + row]) : 0.f;
    const long long gi = (static_cast<long long>(b) * p.T + t) * p.H + h;
    const float a = expf(p.g[gi]), be = p.beta[gi];
    float x[16], kq = 0.f;
#pragma unroll
    for (int i = 0; i < KPL; ++i) kq = fmaf(kv[i], qv[i], kq);
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) kq += __shfl_xor_sync(kAll, kq, w);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      x[r] = x[kRows + r] = 0.f;
#pragma unroll
      for (int i = 0; i < KPL; ++i) {
        x[r] = fmaf(S[r][i], kv[i], x[r]);
        x[kRows + r] = fmaf(S[r][i], qv[i], x[kRows + r]);
      }
    }
    const float got = a * sum16(x, lane);
    const float u = be * (vr - got);  // meaningful in lanes of the S . k sums
    const float ur = __shfl_sync(kAll, u, lane & 15);
    if (lane >= 16 && (lane & 1) == 0 && row < p.V) o[t * p.ot + row] = from_f32<T>(p.scale * fmaf(ur, kq, got));
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const float w = __shfl_sync(kAll, u, 2 * r);
#pragma unroll
      for (int i = 0; i < KPL; ++i) S[r][i] = fmaf(w, kv[i], a * S[r][i]);
    }
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r)
    if (r0 + r < p.V) store_pack<float, KPL>(s + r * K, S[r]);
}

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  set_last_error(buf);
  return code;
}

template <class T>
int launch(const Params& p, int64_t batch, int64_t dstate, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>((p.V + kRows * kWarps - 1) / (kRows * kWarps)), static_cast<unsigned>(p.H),
                  static_cast<unsigned>(batch));
  const cudaError_t e = dstate == 128 ? launch_programmatic(step_kernel<T, 4>, grid, dim3(kWarps * 32), 0, st, p)
                                      : launch_programmatic(step_kernel<T, 2>, grid, dim3(kWarps * 32), 0, st, p);
  if (e != cudaSuccess) return fail(EMA_ERR_CUDA, "delta_step launch failed: %s", cudaGetErrorString(e));
  return EMA_OK;
}

}  // namespace dstep
}  // namespace emab

extern "C" EMA_API int delta_step_launch(const DeltaStepArgs* a, void* stream) {
  using namespace emab;
  using namespace emab::dstep;
  if (a == nullptr) return fail(EMA_ERR_INVALID_ARGUMENT, "delta_step: args is NULL");
  if (a->batch < 0 || a->tokens < 0 || a->nheads <= 0 || a->ngroups <= 0 || a->headdim <= 0 || a->dstate <= 0 ||
      a->slots < 0 || a->nheads % a->ngroups != 0)
    return fail(EMA_ERR_INVALID_ARGUMENT, "delta_step: bad shape");
  if (a->dtype != EMA_DTYPE_F32 && a->dtype != EMA_DTYPE_BF16 && a->dtype != EMA_DTYPE_F16)
    return fail(EMA_ERR_INVALID_ARGUMENT, "delta_step: unknown dtype %d", a->dtype);
  if ((a->dstate != 64 && a->dstate != 128) || a->headdim % 8 != 0 || a->headdim > 256)
    return fail(EMA_ERR_UNSUPPORTED, "delta_step: dstate 64 or 128, headdim a multiple of 8 up to 256");
  if (a->batch > 65535 || a->nheads > 65535 || a->tokens > 1048576 || a->slots > 2147483647)
    return fail(EMA_ERR_UNSUPPORTED, "delta_step: shape too large");
  if (a->batch == 0 || a->tokens == 0) return EMA_OK;
  if (a->q == nullptr || a->k == nullptr || a->v == nullptr || a->g == nullptr || a->beta == nullptr ||
      a->states == nullptr || a->out == nullptr)
    return fail(EMA_ERR_INVALID_ARGUMENT, "delta_step: NULL tensor");
  if (a->state_indices == nullptr && a->slots < a->batch)
    return fail(EMA_ERR_INVALID_ARGUMENT, "delta_step: %lld rows on %lld slots", static_cast<long long>(a->batch),
                static_cast<long long>(a->slots));
  const int es = a->dtype == EMA_DTYPE_F32 ? 4 : 2;
  auto aligned = [](const void* p, const int64_t* s, int n, int e) {
    bool ok = reinterpret_cast<uintptr_t>(p) % 16 == 0;
    for (int i = 0; i < n; ++i) ok = ok && (s[i] * e) % 16 == 0;
    return ok;
  };
  if (!aligned(a->q, a->q_stride, 3, es) || !aligned(a->k, a->k_stride, 3, es) ||
      !aligned(a->states, a->state_stride, 2, 4))
    return fail(EMA_ERR_INVALID_ARGUMENT, "delta_step: q, k and states need 16-byte aligned rows");
  Params p{};
  p.T = static_cast<int>(a->tokens), p.H = static_cast<int>(a->nheads), p.G = static_cast<int>(a->ngroups);
  p.V = static_cast<int>(a->headdim), p.slots = static_cast<int>(a->slots), p.scale = a->scale;
  p.q = a->q, p.qb = a->q_stride[0], p.qt = a->q_stride[1], p.qg = a->q_stride[2];
  p.k = a->k, p.kb = a->k_stride[0], p.kt = a->k_stride[1], p.kg = a->k_stride[2];
  p.v = a->v, p.vb = a->v_stride[0], p.vt = a->v_stride[1], p.vh = a->v_stride[2];
  p.o = a->out, p.ob = a->out_stride[0], p.ot = a->out_stride[1], p.oh = a->out_stride[2];
  p.g = a->g, p.beta = a->beta, p.s = a->states, p.ss = a->state_stride[0], p.sh = a->state_stride[1];
  p.index = a->state_indices;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->dtype == EMA_DTYPE_F32) return launch<float>(p, a->batch, a->dstate, st);
  if (a->dtype == EMA_DTYPE_BF16) return launch<__nv_bfloat16>(p, a->batch, a->dstate, st);
  return launch<__half>(p, a->batch, a->dstate, st);
}
