/*
 * delta_b200.h -- C ABI of the gated delta rule in libema_ssd_b200.so (sm_100a).
 *
 * Per sequence and head, with a state S (headdim x dstate), a_t = exp(g_t):
 *   S_t = a_t S_{t-1} + beta_t (v_t - a_t S_{t-1} k_t) k_t^T,   o_t = scale S_t q_t
 *
 *   q, k, dq, dk        (batch, seqlen, ngroups, dstate)   dstate stride 1; head h reads group h / (nheads / ngroups)
 *   v, out, dout, dv    (batch, seqlen, nheads, headdim)   headdim stride 1
 *   g, beta, dg, dbeta  (batch, seqlen, nheads)            fp32 contiguous; g <= -100 is a full reset (e^-100 = 0)
 *   states              (sequences, nheads, headdim, dstate) fp32 contiguous
 *   cu_seqlens          (nseq + 1,) int32 on the device, or NULL: sequence n is tokens
 *                       [cu[n], cu[n + 1]) of a batch of one.  Values outside [0, seqlen] and falling
 *                       ones are clamped on the device, never followed out of range.
 *
 * dstate is 64 or 128, headdim a multiple of 8 up to 128 (up to 256 for the step), nheads a multiple of
 * ngroups; q, k, v, out and their gradients share one type.  Base addresses are 16-byte aligned and
 * strides multiples of 16 bytes.  Launchers are asynchronous on the given stream, allocate nothing and
 * return an EMA_* code (ema_ssd_b200.h) with the text in ema_last_error().
 */
#ifndef DELTA_B200_H_
#define DELTA_B200_H_

#include "ema_ssd_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* bf16 calls run on the tensor cores, their 32-bit operands as two or three bf16 pieces (2^-16 of each); with this flag
 * their products are fp32 on the CUDA cores, as those of fp16 and fp32 calls always are. */
#define DELTA_FP32_PRODUCTS 1

typedef struct DeltaFwdArgs {
  int64_t batch, seqlen, nheads, headdim, dstate, ngroups;
  int64_t nseq;                  /* sequences: batch without cu_seqlens */
  int32_t dtype;                 /* EMA_DTYPE_* of q, k, v, out */
  float scale;
  const void* q; int64_t q_stride[3];  /* element strides of batch, token, group */
  const void* k; int64_t k_stride[3];
  const void* v; int64_t v_stride[3];  /* of batch, token, head */
  const float* g;
  const float* beta;
  const int32_t* cu_seqlens;
  const float* initial_states;   /* or NULL: zero */
  void* out; int64_t out_stride[3];
  float* final_states;           /* or NULL */
  void* workspace; size_t workspace_bytes;  /* delta_workspace_bytes(.., 0) */
  void* saved; size_t saved_bytes;          /* delta_saved_bytes(): kept for the backward; NULL without one */
  int32_t flags;                 /* DELTA_FP32_PRODUCTS or 0; the same for the sizes, the forward and the backward */
  int32_t reserved;
} DeltaFwdArgs;

typedef struct DeltaBwdArgs {
  int64_t batch, seqlen, nheads, headdim, dstate, ngroups;
  int64_t nseq;
  int32_t dtype;
  float scale;
  const void* q; int64_t q_stride[3];
  const void* k; int64_t k_stride[3];
  const void* v; int64_t v_stride[3];
  const float* g;
  const float* beta;
  const int32_t* cu_seqlens;
  const void* saved; size_t saved_bytes;    /* from the forward of the same inputs */
  const void* dout; int64_t dout_stride[3];
  const float* d_final_states;   /* or NULL: zero */
  void* dq; int64_t dq_stride[3];
  void* dk; int64_t dk_stride[3];
  void* dv; int64_t dv_stride[3];
  float* dg;
  float* dbeta;
  float* d_initial_states;       /* or NULL */
  void* workspace; size_t workspace_bytes;  /* delta_workspace_bytes(.., 1) */
  int32_t flags;
  int32_t reserved;
} DeltaBwdArgs;

/* The recurrent form: `tokens` tokens of every row on a cache of states, updated in place.  Row b works on
 * slot state_indices[b] (b itself when NULL); a negative or too large index leaves every state as it is
 * and writes zeros to that row of out.  Two rows of one call must not share a slot. */
typedef struct DeltaStepArgs {
  int64_t batch, tokens, nheads, headdim, dstate, ngroups, slots;
  int32_t dtype;
  float scale;
  const void* q; int64_t q_stride[3];
  const void* k; int64_t k_stride[3];
  const void* v; int64_t v_stride[3];
  const float* g;                /* (batch, tokens, nheads) contiguous */
  const float* beta;
  float* states; int64_t state_stride[2];   /* (slots, nheads, headdim, dstate): element strides of slot, head */
  const int32_t* state_indices;
  void* out; int64_t out_stride[3];
} DeltaStepArgs;

/* Bytes of scratch (contents need not be initialised) and of what the forward keeps for the backward. */
EMA_API size_t delta_workspace_bytes(int64_t batch, int64_t seqlen, int64_t nseq, int64_t nheads, int64_t headdim,
                                     int64_t dstate, int64_t ngroups, int32_t dtype, int32_t flags, int32_t backward);
EMA_API size_t delta_saved_bytes(int64_t batch, int64_t seqlen, int64_t nseq, int64_t nheads, int64_t headdim,
                                 int64_t dstate, int64_t ngroups, int32_t dtype, int32_t flags);
EMA_API int delta_fwd_launch(const DeltaFwdArgs* args, void* stream);
EMA_API int delta_bwd_launch(const DeltaBwdArgs* args, void* stream);
EMA_API int delta_step_launch(const DeltaStepArgs* args, void* stream);
/* Error word of the chunked kernels (0: none; 2: a bounded wait on the device timed out and results are
 * invalid), read on `stream` after the work queued before it; zeroed afterwards when `clear` is non-zero. */
EMA_API int delta_device_status(uint32_t* status, int clear, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DELTA_B200_H_ */
