// Norms around a block: the gated RMS norm behind it and the residual RMS norm before the next one, with
// their gradients.  All fp32 arithmetic on bf16 / fp16 / fp32 tensors, every tensor read and written once.
//
//   gated, norm first:  y = t r w s,  t = x,      r = (mean t^2 + eps)^-1/2,  s = silu(z)
//   gated, gate first:  y = t r w,    t = x s
//   residual:           h = residual + scale x (rounded to h's type),  y = h r w
//
// Gradients, with t^ = t r, dn = dy (times s when the norm comes first), d^ = dn w, c = mean(d^ t^):
//   dt = r (d^ - t^ c),  dw = sum over rows of dn t^
//   norm first: dx = dt, dz = dy t^ w silu'(z);  gate first: dx = dt s, dz = dt x silu'(z)
//   residual: dh_total = dh + dt, d_residual = dh_total, dx = scale dh_total
//
// Bound: HBM.  A group of TG threads owns one norm row at a time and keeps all of it in registers (NV
// vectors of VEC = 8 elements a thread), so the two sums a row needs (t^2 and d^ t) come from one
// reduction and nothing is read twice; a thread keeps its columns over all its rows, so the weight is
// read once and dw is a register sum, joined over the block's groups in shared memory and over the
// blocks by a second kernel in a fixed order (bitwise reproducible).  TG is the smallest of 8, 16, 32 and
// 256 threads that hold a row: a row per warp or less needs shuffles only.  The layout goes by the width alone:
// rows that do not start on 16 bytes are read element by element in the same places, so results do not
// depend on strides.  Widths that are no multiple of 8 take VEC = 1 with 256 threads, rows beyond 8192 (those: 2048)
// columns a form that reads the row twice from L1 / L2.  Where a row does not fit its threads well the bytes in flight are
// fewer (64 Mi bf16 elements, gated forward and backward: 4.9 and 4.6 TB/s at 128 columns, 4.5 and 4.0 at 2048, 2.8 and 2.6
// at 1024, where half of the threads hold nothing, 3.1 and 2.1 at 8192, whose backward spills 360 bytes a thread with the gate
// first and 48 without, 1.6 and 1.6 at 777, two bytes a load).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdio>
#include <type_traits>

#include "block_norm_b200.h"
#include "ema_common.cuh"
#include "ema_scan_dispatch.h"

namespace emab {
void set_last_error(const char* msg);

namespace bnorm {

constexpr int kThreads = 256;

struct Params {
  long long rows;
  int D, m;          // channels, channels of a norm row
  int wtype, before;
  bool aligned;      // rows of every tensor start on 16 bytes
  float eps, scale;
  const void* x;   long long sx;
  const void* z;   long long sz;   // gate, or the residual
  const void* w;
  void* y;         long long sy;
  void* h;         long long sh;
  const void* dy;  long long sdy;
  const void* dh;  long long sdh;
  void* dx;        long long sdx;
  void* dz;        long long sdz;  // d gate, or d residual
  float* partial;  // (blocks, m) of this group's weight gradient, group-major
};

// The approximate reciprocal is within 2 ulp, and 0 where exp(-v) overflows.  16-bit calls take the approximate exponential too
// (2 + 1.2 |v| ulp of fp32, far below their rounding); in fp32 calls it would show (1.9e-6 of y at gates down to -30).
template <class T>
__device__ __forceinline__ float sigmoid(float v) {
  const float e = std::is_same_v<T, float> ? expf(-v) : __expf(-v);
  return __fdividef(1.f, 1.f + e);
}

__device__ __forceinline__ float load_weight(const void* w, int type, int i) {
  if (type == EMA_DTYPE_F32) return static_cast<const float*>(w)[i];
  if (type == EMA_DTYPE_BF16) return to_f32(static_cast<const __nv_bfloat16*>(w)[i]);
  return to_f32(static_cast<const __half*>(w)[i]);
}

// VEC consecutive elements as they lie in memory; `al`: all rows of the call start on 16 bytes (uniform over the grid).
template <class T, int VEC>
struct alignas(sizeof(T) * VEC >= 16 ? 16 : sizeof(T) * VEC) Raw {
  T e[VEC];
};
template <class T, int VEC>
__device__ __forceinline__ void load_raw(const void* base, long long at, bool al, Raw<T, VEC>& r) {
  const T* p = static_cast<const T*>(base) + at;
  if (VEC == 1 || !al) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) r.e[k] = p[k];
  } else {
    uint4* to = reinterpret_cast<uint4*>(&r);
#pragma unroll
    for (int k = 0; k < static_cast<int>(sizeof(r) / 16); ++k) to[k] = __ldcs(reinterpret_cast<const uint4*>(p) + k);
  }
}
template <class T, int VEC>
__device__ __forceinline__ void store_v(T* p, bool al, const float (&f)[VEC]) {
  if (VEC == 1 || !al) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) p[k] = from_f32<T>(f[k]);
  } else if constexpr (VEC == 8) {
    float2 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = make_float2(f[2 * k], f[2 * k + 1]);
    store8_cs<T>(p, v, 8);
  }
}

// Sums of a and b over a group of TG consecutive threads (a sub-warp, a warp or the block); every thread
// gets them.  Block form: two buffers in turn, so one barrier a call.
template <int TG>
__device__ __forceinline__ float2 group_sum(float a, float b, float2 (*buf)[kThreads / 32], int& turn) {
  constexpr int W = TG < 32 ? TG : 32;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if constexpr (TG > 32) {
    if ((threadIdx.x & 31) == 0) buf[turn][threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int i = 0; i < TG / 32; ++i) {
      a += buf[turn][i].x;
      b += buf[turn][i].y;
    }
    turn ^= 1;
  }
  return make_float2(a, b);
}

// Adds the groups' column sums of one block and writes them to partial[blockIdx.x][0 .. m).
template <int TG, int VEC, int NV>
__device__ __forceinline__ void write_partial(const Params& p, const float (&dw)[NV][VEC], int lane, int grp) {
  constexpr int NG = kThreads / TG;
  float* out = p.partial + (static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x) * p.m;
  if constexpr (NG == 1) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const int c = (j * TG + lane) * VEC + k;
        if (c < p.m) out[c] = dw[j][k];
      }
  } else {
    __shared__ float s[NG][TG * VEC];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) s[grp][lane * VEC + k] = dw[j][k];
      __syncthreads();
      for (int i = threadIdx.x; i < TG * VEC; i += kThreads) {
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < NG; ++q) v += s[q][i];
        if (j * TG * VEC + i < p.m) out[j * TG * VEC + i] = v;
      }
      __syncthreads();
    }
  }
}

// grid: (row blocks, groups of a row).  One norm row per group of TG threads at a time; the loads of the next two rows
// (of the next one where a row is longer) are issued before a row's arithmetic, raw, so that a 16-bit tensor costs four
// registers a vector: the bytes in flight are what bounds it.  The gated pair at 8192 x 32 heads of 128: 202 and 396 us
// without, 156 and 261 one row ahead, 146 and 251 two (5.5 and 5.3 TB/s; packed arithmetic, two channels an instruction,
// made no difference); the residual pair at 32768 x 2048: 134 and 179 (6.0 TB/s).
// FIRST: the norm comes before the gate.
template <class T, class R, int TG, int VEC, int NV, bool RES, bool BWD, bool FIRST>
__global__ void __launch_bounds__(kThreads, (NV * VEC <= 8 && sizeof(T) == 2) ? (BWD ? 2 : 3) : 1) norm_kernel(const Params p) {
  __shared__ float2 buf[2][kThreads / 32];
  using TA = std::conditional_t<RES && BWD, R, T>;  // x, or h
  using TB = std::conditional_t<RES, R, T>;         // the gate, the residual, or dh
  const int lane = threadIdx.x % TG, grp = threadIdx.x / TG;
  const int g0 = blockIdx.y * p.m;
  const float inv_m = 1.f / static_cast<float>(p.m);
  const void* pa = RES && BWD ? p.h : p.x;
  const void* pb = RES && BWD ? p.dh : p.z;
  const long long sa = RES && BWD ? p.sh : p.sx, sb = RES && BWD ? p.sdh : p.sz;
  int turn = 0;
  float w[NV][VEC], dw[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const int c = (j * TG + lane) * VEC + k;
      w[j][k] = c < p.m ? load_weight(p.w, p.wtype, g0 + c) : 0.f;
      dw[j][k] = 0.f;
    }
  constexpr int NG = kThreads / TG;
  // rows loaded ahead (long rows have enough bytes in flight by themselves, and no registers for more)
  constexpr int kBytes = NV * VEC * static_cast<int>(sizeof(T)), kAhead = kBytes <= 16 && VEC > 1 ? 2 : kBytes <= 32 ? 1 : 0;
  const long long step = static_cast<long long>(gridDim.x) * NG;
  struct Row {
    Raw<TA, VEC> a[NV];
    Raw<TB, VEC> b[NV];
    Raw<T, VEC> d[NV];
  };
  auto fetch = [&](long long row, Row& in) {
    auto &a = in.a;
    auto &b = in.b;
    auto &d = in.d;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * TG + lane) * VEC;
      if (row < p.rows && c < p.m) {
        load_raw<TA, VEC>(pa, row * sa + g0 + c, p.aligned, a[j]);
        if (!RES || pb != nullptr) load_raw<TB, VEC>(pb, row * sb + g0 + c, p.aligned, b[j]);
        if (BWD) load_raw<T, VEC>(p.dy, row * p.sdy + g0 + c, p.aligned, d[j]);
      } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) a[j].e[k] = from_f32<TA>(0.f), b[j].e[k] = from_f32<TB>(0.f), d[j].e[k] = from_f32<T>(0.f);
      }
      if (RES && pb == nullptr)
#pragma unroll
        for (int k = 0; k < VEC; ++k) b[j].e[k] = from_f32<TB>(0.f);
    }
  };
  // every thread of a warp takes part in the shuffles of every row: a group without one (past the end) adds zeros
  auto work = [&](long long row, const Row& in) {
    const auto &ra = in.a;
    const auto &rb = in.b;
    const auto &rc = in.d;
    const bool live = row < p.rows;
    float t[NV][VEC], sg[NV][VEC];  // the normed value, the gate's sigmoid
    float sum = 0.f, dot = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const float a = to_f32(ra[j].e[k]), z = to_f32(rb[j].e[k]), d = BWD ? to_f32(rc[j].e[k]) : 0.f;
        if (RES) {
          t[j][k] = BWD ? a : to_f32(from_f32<R>(fmaf(p.scale, a, z)));
          sum = fmaf(t[j][k], t[j][k], sum);
          if (BWD) dot = fmaf(d * w[j][k], t[j][k], dot);
        } else {
          sg[j][k] = sigmoid<T>(z);
          const float s = z * sg[j][k];
          t[j][k] = FIRST ? a : a * s;
          sum = fmaf(t[j][k], t[j][k], sum);
          if (BWD) dot = fmaf((FIRST ? d * s : d) * w[j][k], t[j][k], dot);
        }
      }
    const float2 sums = group_sum<TG>(sum, dot, buf, turn);
    // (past the end: 0, so that with eps = 0, whose rstd of an empty row is infinite, dw gets nothing from there either)
    const float rstd = BWD && !live ? 0.f : rsqrtf(fmaf(sums.x, inv_m, p.eps));
    const float c1 = sums.y * rstd * inv_m;  // mean of d^ t^
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * TG + lane) * VEC;
      float a[VEC], b[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const float z = to_f32(rb[j].e[k]), d = BWD ? to_f32(rc[j].e[k]) : 0.f;
        const float th = t[j][k] * rstd;
        if (RES) {
          if (!BWD) {
            a[k] = th * w[j][k];
          } else {
            b[k] = fmaf(rstd, fmaf(-th, c1, d * w[j][k]), z);
            a[k] = p.scale * b[k];
            dw[j][k] = fmaf(d, th, dw[j][k]);
          }
        } else {
          const float s = z * sg[j][k];
          if (!BWD) {
            a[k] = th * w[j][k] * (FIRST ? s : 1.f);
          } else {
            const float ds = sg[j][k] * (1.f + z * (1.f - sg[j][k]));
            const float dn = FIRST ? d * s : d;
            const float dt = rstd * fmaf(-th, c1, dn * w[j][k]);
            a[k] = FIRST ? dt : dt * s;
            b[k] = FIRST ? d * th * w[j][k] * ds : dt * to_f32(ra[j].e[k]) * ds;
            dw[j][k] = fmaf(dn, th, dw[j][k]);
          }
        }
      }
      if (live && c < p.m) {
        if (!BWD) {
          store_v<T, VEC>(static_cast<T*>(p.y) + row * p.sy + g0 + c, p.aligned, a);
          if (RES) store_v<R, VEC>(static_cast<R*>(p.h) + row * p.sh + g0 + c, p.aligned, t[j]);
        } else {
          store_v<T, VEC>(static_cast<T*>(p.dx) + row * p.sdx + g0 + c, p.aligned, a);
          if (!RES) store_v<T, VEC>(static_cast<T*>(p.dz) + row * p.sdz + g0 + c, p.aligned, b);
          if (RES && p.dz != nullptr) store_v<R, VEC>(static_cast<R*>(p.dz) + row * p.sdz + g0 + c, p.aligned, b);
        }
      }
    }
  };
  long long row = static_cast<long long>(blockIdx.x) * NG + grp;
  if constexpr (kAhead == 2) {
    Row r0, r1, r2;
    fetch(row, r0);
    fetch(row + step, r1);
    for (; row - grp < p.rows; row += 3 * step) {
      fetch(row + 2 * step, r2);
      work(row, r0);
      fetch(row + 3 * step, r0);
      work(row + step, r1);
      fetch(row + 4 * step, r1);
      work(row + 2 * step, r2);
    }
  } else if constexpr (kAhead == 1) {
    Row r0, r1;
    fetch(row, r0);
    for (; row - grp < p.rows; row += 2 * step) {
      fetch(row + step, r1);
      work(row, r0);
      fetch(row + 2 * step, r0);
      work(row + step, r1);
    }
  } else {
    for (; row - grp < p.rows; row += step) {
      Row r0;
      fetch(row, r0);
      work(row, r0);
    }
  }
  if constexpr (BWD) write_partial<TG, VEC, NV>(p, dw, lane, grp);
}

// Any width: the row is read again for the second pass, the weight gradient is summed in the block's own
// row of `partial` (each column by one thread).
template <class T, class R, bool RES, bool BWD>
__global__ void __launch_bounds__(kThreads) norm_wide_kernel(const Params p) {
  __shared__ float2 buf[2][kThreads / 32];
  const int g0 = blockIdx.y * p.m;
  int turn = 0;
  float* part = BWD ? p.partial + (static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x) * p.m : nullptr;
  if (BWD)
    for (int c = threadIdx.x; c < p.m; c += kThreads) part[c] = 0.f;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    auto at = [&](int c, float& t, float& z, float& d) {
      d = BWD ? to_f32(static_cast<const T*>(p.dy)[row * p.sdy + g0 + c]) : 0.f;
      if (RES) {
        if (BWD) {
          t = to_f32(static_cast<const R*>(p.h)[row * p.sh + g0 + c]);
          z = p.dh != nullptr ? to_f32(static_cast<const R*>(p.dh)[row * p.sdh + g0 + c]) : 0.f;
        } else {
          const float r = p.z != nullptr ? to_f32(static_cast<const R*>(p.z)[row * p.sz + g0 + c]) : 0.f;
          t = to_f32(from_f32<R>(fmaf(p.scale, to_f32(static_cast<const T*>(p.x)[row * p.sx + g0 + c]), r)));
          z = 0.f;
        }
      } else {
        t = to_f32(static_cast<const T*>(p.x)[row * p.sx + g0 + c]);
        z = to_f32(static_cast<const T*>(p.z)[row * p.sz + g0 + c]);
      }
    };
    float sum = 0.f, dot = 0.f;
    for (int c = threadIdx.x; c < p.m; c += kThreads) {
      float t, z, d;
      at(c, t, z, d);
      const float s = RES ? 1.f : z * sigmoid<T>(z);
      const float v = (RES || p.before) ? t : t * s;
      sum = fmaf(v, v, sum);
      if (BWD) dot = fmaf((p.before ? d * s : d) * load_weight(p.w, p.wtype, g0 + c), v, dot);
    }
    const float2 sums = group_sum<kThreads>(sum, dot, buf, turn);
    const float rstd = rsqrtf(sums.x / static_cast<float>(p.m) + p.eps);
    const float c1 = sums.y * rstd / static_cast<float>(p.m);
    for (int c = threadIdx.x; c < p.m; c += kThreads) {
      float t, z, d;
      at(c, t, z, d);
      const float w = load_weight(p.w, p.wtype, g0 + c);
      if (RES) {
        const float th = t * rstd;
        if (!BWD) {
          static_cast<T*>(p.y)[row * p.sy + g0 + c] = from_f32<T>(th * w);
          static_cast<R*>(p.h)[row * p.sh + g0 + c] = from_f32<R>(t);
        } else {
          const float b = fmaf(rstd, fmaf(-th, c1, d * w), z);
          static_cast<T*>(p.dx)[row * p.sdx + g0 + c] = from_f32<T>(p.scale * b);
          if (p.dz != nullptr) static_cast<R*>(p.dz)[row * p.sdz + g0 + c] = from_f32<R>(b);
          part[c] = fmaf(d, th, part[c]);
        }
      } else {
        const float sg = sigmoid<T>(z), s = z * sg;
        const float th = (p.before ? t : t * s) * rstd;
        if (!BWD) {
          static_cast<T*>(p.y)[row * p.sy + g0 + c] = from_f32<T>(th * w * (p.before ? s : 1.f));
        } else {
          const float ds = sg * (1.f + z * (1.f - sg)), dn = p.before ? d * s : d;
          const float dt = rstd * fmaf(-th, c1, dn * w);
          static_cast<T*>(p.dx)[row * p.sdx + g0 + c] = from_f32<T>(p.before ? dt : dt * s);
          static_cast<T*>(p.dz)[row * p.sdz + g0 + c] = from_f32<T>(p.before ? d * th * w * ds : dt * t * ds);
          part[c] = fmaf(dn, th, part[c]);
        }
      }
    }
  }
}

// dweight[group][c] = sum over the blocks of partial[group][block][c].  A block owns 32 columns; its 32 warps take
// every 32nd row of partials, eight in flight, and are joined in shared memory in warp order.
__global__ void __launch_bounds__(1024) weight_grad_kernel(const float* partial, float* dw, int m, int blocks) {
  __shared__ float s[32][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  const float* src = partial + static_cast<long long>(blockIdx.y) * blocks * m;
  float v = 0.f;
  if (c < m) {
#pragma unroll 8
    for (int b = warp; b < blocks; b += 32) v += src[static_cast<long long>(b) * m + c];
  }
  s[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && c < m) {
#pragma unroll
    for (int i = 1; i < 32; ++i) v += s[i][lane];
    dw[static_cast<long long>(blockIdx.y) * m + c] = v;
  }
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

int esize(int dtype) { return dtype == EMA_DTYPE_F32 ? 4 : 2; }
bool known(int dtype) { return dtype == EMA_DTYPE_F32 || dtype == EMA_DTYPE_BF16 || dtype == EMA_DTYPE_F16; }
bool vec_ok(const void* p, int64_t stride, int es) {
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && (stride * es) % 16 == 0);
}

// The threads of a norm row: the smallest of 8, 16, 32 that hold it with one to four vectors, else 256.
struct Layout {
  int tg, nv;
  bool vec, wide;
};
Layout layout(int64_t m) {
  if (m % 8 != 0) return Layout{256, 8, false, m > 2048};
  if (m <= 64) return Layout{8, 1, true, false};
  if (m <= 128) return Layout{16, 1, true, false};
  if (m <= 256) return Layout{32, 1, true, false};
  if (m <= 512) return Layout{32, 2, true, false};
  if (m <= 2048) return Layout{256, 1, true, false};
  if (m <= 4096) return Layout{256, 2, true, false};
  return Layout{256, 4, true, m > 8192};
}
// Blocks over the rows of one group: enough for every SM to hold several, no more than there are rows.
int64_t row_blocks(int64_t rows, int64_t groups, int per_block) {
  constexpr int64_t kTarget = 148 * 6;
  int64_t want = (kTarget + groups - 1) / groups;
  const int64_t have = (rows + per_block - 1) / per_block;
  if (want > have) want = have;
  return want < 1 ? 1 : want;
}

template <class T, class R, bool RES, bool BWD, bool FIRST>
void run_rows(const Params& p, const Layout& l, dim3 grid, cudaStream_t st) {
  if (!l.vec) norm_kernel<T, R, 256, 1, 8, RES, BWD, FIRST><<<grid, kThreads, 0, st>>>(p);
  else if (l.tg == 8) norm_kernel<T, R, 8, 8, 1, RES, BWD, FIRST><<<grid, kThreads, 0, st>>>(p);
  else if (l.tg == 16) norm_kernel<T, R, 16, 8, 1, RES, BWD, FIRST><<<grid, kThreads, 0, st>>>(p);
  else if (l.tg == 32 && l.nv == 1) norm_kernel<T, R, 32, 8, 1, RES, BWD, FIRST><<<grid, kThreads, 0, st>>>(p);
  else if (l.tg == 32) norm_kernel<T, R, 32, 8, 2, RES, BWD, FIRST><<<grid, kThreads, 0, st>>>(p);
  else if (l.nv == 1) norm_kernel<T, R, 256, 8, 1, RES, BWD, FIRST><<<grid, kThreads, 0, st>>>(p);
  else if (l.nv == 2) norm_kernel<T, R, 256, 8, 2, RES, BWD, FIRST><<<grid, kThreads, 0, st>>>(p);
  else norm_kernel<T, R, 256, 8, 4, RES, BWD, FIRST><<<grid, kThreads, 0, st>>>(p);
}
template <class T, class R, bool RES, bool BWD>
void run(const Params& p, const Layout& l, dim3 grid, cudaStream_t st) {
  if (l.wide) norm_wide_kernel<T, R, RES, BWD><<<grid, kThreads, 0, st>>>(p);
  else if (!RES && p.before) run_rows<T, R, RES, BWD, !RES>(p, l, grid, st);
  else run_rows<T, R, RES, BWD, false>(p, l, grid, st);
}

template <bool RES, bool BWD>
int launch(Params& p, int dtype, int rtype, bool vec, float* dweight, void* ws, size_t ws_bytes, const char* what,
           cudaStream_t st) {
  const int64_t groups = p.D / p.m;
  if (groups > 65535) return fail(EMA_ERR_UNSUPPORTED, "%s: more than 65535 groups", what);
  if (BWD && p.rows == 0) {
    const cudaError_t e = cudaMemsetAsync(dweight, 0, sizeof(float) * p.D, st);
    return e == cudaSuccess ? EMA_OK : fail(EMA_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  }
  if (p.rows == 0) return EMA_OK;
  p.aligned = vec;
  const Layout l = layout(p.m);
  const int64_t blocks = row_blocks(p.rows, groups, l.wide ? 1 : kThreads / l.tg);
  if (BWD) {
    if (ws == nullptr || ws_bytes < static_cast<size_t>(blocks) * p.D * 4)
      return fail(EMA_ERR_WORKSPACE, "%s: workspace of %zu bytes is too small", what, ws_bytes);
    p.partial = static_cast<float*>(ws);
  }
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(groups));
  const bool wide_res = RES && rtype == EMA_DTYPE_F32;
  if (dtype == EMA_DTYPE_F32) run<float, float, RES, BWD>(p, l, grid, st);
  else if (dtype == EMA_DTYPE_BF16 && !wide_res) run<__nv_bfloat16, __nv_bfloat16, RES, BWD>(p, l, grid, st);
  else if (dtype == EMA_DTYPE_F16 && !wide_res) run<__half, __half, RES, BWD>(p, l, grid, st);
  else if constexpr (RES) {
    if (dtype == EMA_DTYPE_BF16) run<__nv_bfloat16, float, RES, BWD>(p, l, grid, st);
    else run<__half, float, RES, BWD>(p, l, grid, st);
  }
  if (BWD)
    weight_grad_kernel<<<dim3(static_cast<unsigned>((p.m + 31) / 32), static_cast<unsigned>(groups)), 1024, 0, st>>>(
        p.partial, dweight, p.m, static_cast<int>(blocks));
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(EMA_ERR_CUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
  return EMA_OK;
}

int check_shape(int64_t rows, int64_t dim, int64_t m, int dtype, int wtype, float eps, const char* what) {
  if (rows < 0 || dim <= 0 || m <= 0 || dim % m != 0) return fail(EMA_ERR_INVALID_ARGUMENT, "%s: bad shape", what);
  if (dim > 1073741824) return fail(EMA_ERR_UNSUPPORTED, "%s: row too long", what);
  if (!known(dtype) || !known(wtype)) return fail(EMA_ERR_INVALID_ARGUMENT, "%s: unknown dtype", what);
  if (!(eps >= 0.f)) return fail(EMA_ERR_INVALID_ARGUMENT, "%s: eps must not be negative", what);
  return EMA_OK;
}

template <bool BWD>
int gated(const GatedNormArgs* a, cudaStream_t st) {
  const char* what = BWD ? "gated_norm_bwd" : "gated_norm_fwd";
  if (a == nullptr) return fail(EMA_ERR_INVALID_ARGUMENT, "%s: args is NULL", what);
  const int r = check_shape(a->rows, a->dim, a->group_size, a->dtype, a->weight_dtype, a->eps, what);
  if (r) return r;
  if (a->weight == nullptr || (BWD && a->dweight == nullptr))
    return fail(EMA_ERR_INVALID_ARGUMENT, "%s: NULL tensor", what);
  if (a->rows > 0 && (a->x == nullptr || a->z == nullptr ||
                      (BWD ? (a->dy == nullptr || a->dx == nullptr || a->dz == nullptr) : a->y == nullptr)))
    return fail(EMA_ERR_INVALID_ARGUMENT, "%s: NULL tensor", what);
  Params p{};
  p.rows = a->rows;
  p.D = static_cast<int>(a->dim);
  p.m = static_cast<int>(a->group_size);
  p.wtype = a->weight_dtype;
  p.before = a->norm_before_gate != 0;
  p.eps = a->eps;
  p.x = a->x, p.sx = a->x_stride, p.z = a->z, p.sz = a->z_stride, p.w = a->weight;
  const int es = esize(a->dtype);
  bool vec = vec_ok(a->x, a->x_stride, es) && vec_ok(a->z, a->z_stride, es);
  if (BWD) {
    p.dy = a->dy, p.sdy = a->dy_stride, p.dx = a->dx, p.sdx = a->dx_stride, p.dz = a->dz, p.sdz = a->dz_stride;
    vec = vec && vec_ok(a->dy, a->dy_stride, es) && vec_ok(a->dx, a->dx_stride, es) && vec_ok(a->dz, a->dz_stride, es);
  } else {
    p.y = a->y, p.sy = a->y_stride;
    vec = vec && vec_ok(a->y, a->y_stride, es);
  }
  return launch<false, BWD>(p, a->dtype, a->dtype, vec, a->dweight, a->workspace, a->workspace_bytes, what, st);
}

template <bool BWD>
int residual(const ResidualNormArgs* a, cudaStream_t st) {
  const char* what = BWD ? "residual_norm_bwd" : "residual_norm_fwd";
  if (a == nullptr) return fail(EMA_ERR_INVALID_ARGUMENT, "%s: args is NULL", what);
  const int r = check_shape(a->rows, a->dim, a->dim, a->dtype, a->weight_dtype, a->eps, what);
  if (r) return r;
  if (a->residual_dtype != a->dtype && a->residual_dtype != EMA_DTYPE_F32)
    return fail(EMA_ERR_UNSUPPORTED, "%s: the residual has x's type or fp32", what);
  if (a->weight == nullptr || (BWD && a->dweight == nullptr))
    return fail(EMA_ERR_INVALID_ARGUMENT, "%s: NULL tensor", what);
  if (a->rows > 0 && (a->h == nullptr || (BWD ? (a->dy == nullptr || a->dx == nullptr)
                                              : (a->x == nullptr || a->y == nullptr))))
    return fail(EMA_ERR_INVALID_ARGUMENT, "%s: NULL tensor", what);
  Params p{};
  p.rows = a->rows;
  p.D = p.m = static_cast<int>(a->dim);
  p.wtype = a->weight_dtype;
  p.eps = a->eps;
  p.scale = a->scale;
  p.w = a->weight;
  p.h = a->h, p.sh = a->h_stride;
  const int es = esize(a->dtype), rs = esize(a->residual_dtype);
  bool vec = vec_ok(a->h, a->h_stride, rs);
  if (BWD) {
    p.dy = a->dy, p.sdy = a->dy_stride, p.dh = a->dh, p.sdh = a->dh_stride;
    p.dx = a->dx, p.sdx = a->dx_stride, p.dz = a->d_residual, p.sdz = a->d_residual_stride;
    vec = vec && vec_ok(a->dy, a->dy_stride, es) && vec_ok(a->dh, a->dh_stride, rs) &&
          vec_ok(a->dx, a->dx_stride, es) && vec_ok(a->d_residual, a->d_residual_stride, rs);
  } else {
    p.x = a->x, p.sx = a->x_stride, p.z = a->residual, p.sz = a->residual_stride, p.y = a->y, p.sy = a->y_stride;
    vec = vec && vec_ok(a->x, a->x_stride, es) && vec_ok(a->residual, a->residual_stride, rs) &&
          vec_ok(a->y, a->y_stride, es);
  }
  return launch<true, BWD>(p, a->dtype, a->residual_dtype, vec, a->dweight, a->workspace, a->workspace_bytes, what, st);
}

}  // namespace bnorm
}  // namespace emab

extern "C" EMA_API size_t block_norm_workspace_bytes(int64_t rows, int64_t dim, int64_t group_size) {
  if (rows <= 0 || dim <= 0 || group_size <= 0) return 0;
  // a block per row is the most any layout asks for
  return static_cast<size_t>(emab::bnorm::row_blocks(rows, dim / group_size > 0 ? dim / group_size : 1, 1)) * dim * 4;
}
extern "C" EMA_API int gated_norm_fwd_launch(const GatedNormArgs* args, void* stream) {
  return emab::bnorm::gated<false>(args, static_cast<cudaStream_t>(stream));
}
extern "C" EMA_API int gated_norm_bwd_launch(const GatedNormArgs* args, void* stream) {
  return emab::bnorm::gated<true>(args, static_cast<cudaStream_t>(stream));
}
extern "C" EMA_API int residual_norm_fwd_launch(const ResidualNormArgs* args, void* stream) {
  return emab::bnorm::residual<false>(args, static_cast<cudaStream_t>(stream));
}
extern "C" EMA_API int residual_norm_bwd_launch(const ResidualNormArgs* args, void* stream) {
  return emab::bnorm::residual<true>(args, static_cast<cudaStream_t>(stream));
}
