// C entry points of the chunked gated delta rule: argument checks, buffer layout, choice of the kernels.
#include "delta_host.h"

#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdio>

#include "delta_b200.h"
#include "ema_scan_dispatch.h"

namespace emab {
void set_last_error(const char* msg);

namespace delta {
namespace {

__device__ uint32_t g_status;  // error word of the tensor-core kernels

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  set_last_error(buf);
  return code;
}

struct Shape {
  int64_t batch, seqlen, nseq, H, V, K, G;
  bool packed;
};

int64_t chunks(int64_t seqlen) { return (seqlen + kC - 1) / kC; }
// (a packed call's slots bound a plain batch of one too)
int64_t slots_of(const Shape& s) { return s.packed ? s.seqlen / kC + s.nseq : s.batch * chunks(s.seqlen); }
int64_t slots_bound(int64_t batch, int64_t seqlen, int64_t nseq) {
  const int64_t a = batch * chunks(seqlen), b = seqlen / kC + nseq;
  return batch == 1 && b > a ? b : a;
}

struct Carver {
  char* base;
  size_t at = 0;
  char* bytes(size_t n) {
    char* p = base != nullptr ? base + at : nullptr;
    at += (n + 255) / 256 * 256;
    return p;
  }
  float* take(size_t n) { return reinterpret_cast<float*>(bytes(n * 4)); }
};

size_t carve_tc_fwd(TcBuffers* w, char* base, int64_t slots, int64_t H, int64_t V, int64_t K, bool keep) {
  Carver c{base};
  const size_t n = static_cast<size_t>(slots) * H;
  w->gates = c.take(n * kGateFloats);
  w->T = c.bytes(n * 2 * kTile);
  w->P = c.bytes(n * 2 * kTile);
  w->S = keep ? c.take(n * state_image(static_cast<int>(V), static_cast<int>(K))) : nullptr;
  w->E = keep ? c.bytes(n * 3 * token_piece(static_cast<int>(V))) : nullptr;
  return c.at;
}
size_t carve_tc_bwd(TcBuffers* w, char* base, int64_t slots, int64_t H, int64_t V, int64_t K) {
  Carver c{base};
  const size_t n = static_cast<size_t>(slots) * H;
  w->dS = c.take(n * state_image(static_cast<int>(V), static_cast<int>(K)));
  w->dX = c.bytes(n * token_piece(static_cast<int>(V)));
  return c.at;
}
// The tensor-core kernels take bf16 (every dstate and headdim of the entry points); a call without tokens, whose
// tiles no tensor map can describe, goes to the fp32 family, which then only copies the states.
bool on_tensor_cores(int dtype, int64_t seqlen, int flags) {
  return dtype == EMA_DTYPE_BF16 && seqlen > 0 && (flags & DELTA_FP32_PRODUCTS) == 0;
}

// Tiles of 64 tokens of one head of a (batch, token, head, channel) tensor: `box` channels, swizzled or as they are.
int tile_map(CUtensorMap* m, const void* t, const int64_t (&st)[3], int64_t channels, int64_t heads, int64_t seqlen,
             int64_t batch, int64_t box, bool swizzle) {
  const uint64_t d[4] = {static_cast<uint64_t>(channels), static_cast<uint64_t>(heads), static_cast<uint64_t>(seqlen),
                         static_cast<uint64_t>(batch)};
  const uint64_t s[3] = {static_cast<uint64_t>(st[2]) * 2, static_cast<uint64_t>(st[1]) * 2,
                         static_cast<uint64_t>(st[0]) * 2};
  const uint32_t b[4] = {static_cast<uint32_t>(box), 1, static_cast<uint32_t>(kC), 1};
  return encode_map(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, t, d, s, b, swizzle);
}

// What the forward keeps for a backward (T, P, S0, E); without one only T and P, in the workspace.
size_t carve_fwd(Buffers* w, char* base, int64_t slots, int64_t H, int64_t V, int64_t K, bool keep) {
  Carver c{base};
  const size_t n = static_cast<size_t>(slots) * H;
  w->T = c.take(n * kC * kC);
  w->P = c.take(n * kC * kC);
  w->S0 = keep ? c.take(n * V * K) : nullptr;
  w->E = keep ? c.take(n * kC * V) : nullptr;
  return c.at;
}
size_t carve_bwd(Buffers* w, char* base, int64_t slots, int64_t H, int64_t V, int64_t K) {
  Carver c{base};
  const size_t n = static_cast<size_t>(slots) * H;
  w->dU = c.take(n * kC * V);
  w->dX = c.take(n * kC * V);
  w->dS1 = c.take(n * V * K);
  return c.at;
}

template <class A>
int check(const A* a, const char* what, Shape* s) {
  if (a == nullptr) return fail(EMA_ERR_INVALID_ARGUMENT, "%s: args is NULL", what);
  *s = Shape{a->batch, a->seqlen, a->nseq, a->nheads, a->headdim, a->dstate, a->ngroups, a->cu_seqlens != nullptr};
  if (s->batch < 0 || s->seqlen < 0 || s->nseq < 0 || s->H <= 0 || s->V <= 0 || s->K <= 0 || s->G <= 0 ||
      s->H % s->G != 0)
    return fail(EMA_ERR_INVALID_ARGUMENT, "%s: bad shape", what);
  if (s->packed ? s->batch != 1 : s->nseq != s->batch)
    return fail(EMA_ERR_INVALID_ARGUMENT, "%s: %lld sequences in a batch of %lld", what,
                static_cast<long long>(s->nseq), static_cast<long long>(s->batch));
  if (a->dtype != EMA_DTYPE_F32 && a->dtype != EMA_DTYPE_BF16 && a->dtype != EMA_DTYPE_F16)
    return fail(EMA_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d", what, a->dtype);
  if ((a->flags & ~DELTA_FP32_PRODUCTS) != 0) return fail(EMA_ERR_INVALID_ARGUMENT, "%s: unknown flags", what);
  if ((s->K != 64 && s->K != 128) || s->V % 8 != 0 || s->V > 128)
    return fail(EMA_ERR_UNSUPPORTED, "%s: dstate 64 or 128, headdim a multiple of 8 up to 128", what);
  if (s->H > 65535 || s->nseq > 65535 || s->seqlen > 1073741824 || slots_of(*s) > 16777216)
    return fail(EMA_ERR_UNSUPPORTED, "%s: shape too large", what);
  return EMA_OK;
}

bool aligned(const void* p, const int64_t (&s)[3], int es) {
  bool ok = reinterpret_cast<uintptr_t>(p) % 16 == 0;
  for (int i = 0; i < 3; ++i) ok = ok && (s[i] * es) % 16 == 0;
  return ok;
}
View view(const int64_t (&s)[3]) { return View{s[0], s[1], s[2]}; }

template <class A>
Params params(const A* a, const Shape& s) {
  Params p{};
  p.B = static_cast<int>(s.batch), p.L = static_cast<int>(s.seqlen), p.H = static_cast<int>(s.H);
  p.G = static_cast<int>(s.G), p.V = static_cast<int>(s.V), p.K = static_cast<int>(s.K);
  p.nseq = static_cast<int>(s.nseq);
  p.nc = static_cast<int>(chunks(s.seqlen));
  p.slots = static_cast<int>(slots_of(s));
  p.scale = a->scale;
  p.q = a->q, p.vq = view(a->q_stride), p.k = a->k, p.vk = view(a->k_stride), p.v = a->v, p.vv = view(a->v_stride);
  p.g = a->g, p.beta = a->beta, p.cu = a->cu_seqlens;
  return p;
}

}  // namespace
}  // namespace delta
}  // namespace emab

using namespace emab::delta;

extern "C" EMA_API size_t delta_saved_bytes(int64_t batch, int64_t seqlen, int64_t nseq, int64_t nheads, int64_t headdim,
                                            int64_t dstate, int64_t ngroups, int32_t dtype, int32_t flags) {
  if (batch < 0 || seqlen < 0 || nseq < 0 || nheads <= 0 || headdim <= 0 || dstate <= 0) return 0;
  const int64_t n = slots_bound(batch, seqlen, nseq);
  if (on_tensor_cores(dtype, seqlen, flags)) {
    TcBuffers t{};
    return carve_tc_fwd(&t, nullptr, n, nheads, headdim, dstate, true);
  }
  Buffers w{};
  return carve_fwd(&w, nullptr, n, nheads, headdim, dstate, true);
}

extern "C" EMA_API size_t delta_workspace_bytes(int64_t batch, int64_t seqlen, int64_t nseq, int64_t nheads,
                                                int64_t headdim, int64_t dstate, int64_t ngroups, int32_t dtype,
                                                int32_t flags, int32_t backward) {
  if (batch < 0 || seqlen < 0 || nseq < 0 || nheads <= 0 || headdim <= 0 || dstate <= 0) return 0;
  Buffers w{};
  const int64_t n = slots_bound(batch, seqlen, nseq);
  if (on_tensor_cores(dtype, seqlen, flags)) {
    TcBuffers t{};
    return backward ? carve_tc_bwd(&t, nullptr, n, nheads, headdim, dstate)
                    : carve_tc_fwd(&t, nullptr, n, nheads, headdim, dstate, false);
  }
  return backward ? carve_bwd(&w, nullptr, n, nheads, headdim, dstate)
                  : carve_fwd(&w, nullptr, n, nheads, headdim, dstate, false);
}

extern "C" EMA_API int delta_fwd_launch(const DeltaFwdArgs* a, void* stream) {
  Shape s;
  const int r = check(a, "delta_fwd", &s);
  if (r) return r;
  if (s.nseq == 0) return EMA_OK;
  const bool tokens = s.seqlen > 0;
  if (tokens && (a->q == nullptr || a->k == nullptr || a->v == nullptr || a->g == nullptr || a->beta == nullptr ||
                 a->out == nullptr))
    return fail(EMA_ERR_INVALID_ARGUMENT, "delta_fwd: NULL tensor");
  const int es = a->dtype == EMA_DTYPE_F32 ? 4 : 2;
  if (tokens && (!aligned(a->q, a->q_stride, es) || !aligned(a->k, a->k_stride, es) ||
                 !aligned(a->v, a->v_stride, es) || !aligned(a->out, a->out_stride, es)))
    return fail(EMA_ERR_INVALID_ARGUMENT, "delta_fwd: q, k, v and out need 16-byte aligned rows");
  Params p = params(a, s);
  p.s0 = a->initial_states, p.s1 = a->final_states;
  p.o = a->out, p.vo = view(a->out_stride);
  Buffers w{};
  const bool keep = a->saved != nullptr;
  void* base = keep ? a->saved : a->workspace;
  if (on_tensor_cores(a->dtype, s.seqlen, a->flags)) {
    TcBuffers t{};
    const size_t need = carve_tc_fwd(&t, static_cast<char*>(base), p.slots, s.H, s.V, s.K, keep);
    if (base == nullptr || (keep ? a->saved_bytes : a->workspace_bytes) < need ||
        reinterpret_cast<uintptr_t>(base) % 256 != 0)
      return fail(EMA_ERR_WORKSPACE, "delta_fwd: needs %zu bytes, 256-byte aligned, of %s", need,
                  keep ? "saved" : "workspace");
    CUtensorMap mk{}, mq{}, mv{};
    int e = tile_map(&mk, a->k, a->k_stride, s.K, s.G, s.seqlen, s.batch, 64, true);
    if (e == EMA_OK) e = tile_map(&mq, a->q, a->q_stride, s.K, s.G, s.seqlen, s.batch, 64, true);
    if (e == EMA_OK) e = tile_map(&mv, a->v, a->v_stride, s.V, s.H, s.seqlen, s.batch, s.V, false);
    if (e != EMA_OK) return e;
    void* st = nullptr;
    cudaError_t ce = cudaGetSymbolAddress(&st, g_status);
    uint32_t* status = static_cast<uint32_t*>(st);
    if (ce == cudaSuccess) ce = tc_prep(mk, mq, p, t, status, static_cast<cudaStream_t>(stream));
    if (ce == cudaSuccess) ce = tc_fwd_walk(mk, mq, mv, p, t, status, static_cast<cudaStream_t>(stream));
    if (ce != cudaSuccess) return fail(EMA_ERR_CUDA, "delta_fwd launch failed: %s", cudaGetErrorString(ce));
    return EMA_OK;
  }
  const size_t need = carve_fwd(&w, static_cast<char*>(base), p.slots, s.H, s.V, s.K, keep);
  if (tokens && (base == nullptr || (keep ? a->saved_bytes : a->workspace_bytes) < need ||
                 reinterpret_cast<uintptr_t>(base) % 256 != 0))
    return fail(EMA_ERR_WORKSPACE, "delta_fwd: needs %zu bytes, 256-byte aligned, of %s", need,
                keep ? "saved" : "workspace");
  const cudaError_t e = simt_fwd(p, w, a->dtype, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail(EMA_ERR_CUDA, "delta_fwd launch failed: %s", cudaGetErrorString(e));
  return EMA_OK;
}

extern "C" EMA_API int delta_bwd_launch(const DeltaBwdArgs* a, void* stream) {
  Shape s;
  const int r = check(a, "delta_bwd", &s);
  if (r) return r;
  if (s.nseq == 0) return EMA_OK;
  const bool tokens = s.seqlen > 0;
  if (tokens && (a->q == nullptr || a->k == nullptr || a->v == nullptr || a->g == nullptr || a->beta == nullptr ||
                 a->dout == nullptr || a->dq == nullptr || a->dk == nullptr || a->dv == nullptr || a->dg == nullptr ||
                 a->dbeta == nullptr))
    return fail(EMA_ERR_INVALID_ARGUMENT, "delta_bwd: NULL tensor");
  const int es = a->dtype == EMA_DTYPE_F32 ? 4 : 2;
  if (tokens && (!aligned(a->q, a->q_stride, es) || !aligned(a->k, a->k_stride, es) ||
                 !aligned(a->v, a->v_stride, es) || !aligned(a->dout, a->dout_stride, es) ||
                 !aligned(a->dq, a->dq_stride, es) || !aligned(a->dk, a->dk_stride, es) ||
                 !aligned(a->dv, a->dv_stride, es)))
    return fail(EMA_ERR_INVALID_ARGUMENT, "delta_bwd: q, k, v, dout, dq, dk and dv need 16-byte aligned rows");
  Params p = params(a, s);
  p.dout = a->dout, p.vd = view(a->dout_stride);
  p.ds1 = a->d_final_states, p.ds0 = a->d_initial_states;
  p.dq = a->dq, p.vdq = view(a->dq_stride), p.dk = a->dk, p.vdk = view(a->dk_stride);
  p.dv = a->dv, p.vdv = view(a->dv_stride), p.dg = a->dg, p.dbeta = a->dbeta;
  if (on_tensor_cores(a->dtype, s.seqlen, a->flags)) {
    TcBuffers t{};
    const size_t saved = carve_tc_fwd(&t, static_cast<char*>(const_cast<void*>(a->saved)), p.slots, s.H, s.V, s.K, true);
    const size_t need = carve_tc_bwd(&t, static_cast<char*>(a->workspace), p.slots, s.H, s.V, s.K);
    if (a->saved == nullptr || a->saved_bytes < saved || a->workspace == nullptr || a->workspace_bytes < need ||
        reinterpret_cast<uintptr_t>(a->saved) % 256 != 0 || reinterpret_cast<uintptr_t>(a->workspace) % 256 != 0)
      return fail(EMA_ERR_WORKSPACE, "delta_bwd: needs %zu bytes of saved and %zu of workspace, 256-byte aligned", saved,
                  need);
    CUtensorMap mk{}, mq{}, mo{}, mdv{};
    int e = tile_map(&mk, a->k, a->k_stride, s.K, s.G, s.seqlen, s.batch, 64, true);
    if (e == EMA_OK) e = tile_map(&mq, a->q, a->q_stride, s.K, s.G, s.seqlen, s.batch, 64, true);
    if (e == EMA_OK) e = tile_map(&mo, a->dout, a->dout_stride, s.V, s.H, s.seqlen, s.batch, 64, true);
    if (e == EMA_OK) e = tile_map(&mdv, a->dv, a->dv_stride, s.V, s.H, s.seqlen, s.batch, 64, true);
    if (e != EMA_OK) return e;
    cudaStream_t stm = static_cast<cudaStream_t>(stream);
    void* st = nullptr;
    cudaError_t ce = cudaGetSymbolAddress(&st, g_status);
    uint32_t* status = static_cast<uint32_t*>(st);
    if (ce == cudaSuccess) ce = tc_bwd_walk(mk, mq, mo, p, t, status, stm);
    if (ce == cudaSuccess) ce = tc_grads(mk, mq, mo, mdv, p, t, status, stm);
    if (ce != cudaSuccess) return fail(EMA_ERR_CUDA, "delta_bwd launch failed: %s", cudaGetErrorString(ce));
    return EMA_OK;
  }
  Buffers w{};
  const size_t saved = carve_fwd(&w, static_cast<char*>(const_cast<void*>(a->saved)), p.slots, s.H, s.V, s.K, true);
  const size_t need = carve_bwd(&w, static_cast<char*>(a->workspace), p.slots, s.H, s.V, s.K);
  if (tokens && (a->saved == nullptr || a->saved_bytes < saved || a->workspace == nullptr ||
                 a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->saved) % 256 != 0 ||
                 reinterpret_cast<uintptr_t>(a->workspace) % 256 != 0))
    return fail(EMA_ERR_WORKSPACE, "delta_bwd: needs %zu bytes of saved and %zu of workspace, 256-byte aligned", saved,
                need);
  const cudaError_t e = simt_bwd(p, w, a->dtype, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return fail(EMA_ERR_CUDA, "delta_bwd launch failed: %s", cudaGetErrorString(e));
  return EMA_OK;
}

extern "C" EMA_API int delta_device_status(uint32_t* status, int clear, void* stream) {
  if (status == nullptr) return fail(EMA_ERR_INVALID_ARGUMENT, "delta_device_status: NULL");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint32_t v = 0, z = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(&v, g_status, 4, 0, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && clear) e = cudaMemcpyToSymbolAsync(g_status, &z, 4, 0, cudaMemcpyHostToDevice, st);
  if (e == cudaSuccess && clear) e = cudaStreamSynchronize(st);
  if (e != cudaSuccess) return fail(EMA_ERR_CUDA, "delta_device_status: %s", cudaGetErrorString(e));
  *status = v;
  return EMA_OK;
}
