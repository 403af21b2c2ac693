"""The gated delta rule on the B200 kernels: whole sequences (autograd) and the recurrent step.

Per sequence and head, a state S (headdim x dstate, fp32) with the decay a_t = exp(g_t):

    S_t = a_t S_{t-1} + beta_t (v_t - a_t S_{t-1} k_t) k_t^T,    o_t = scale S_t q_t

Layouts are those of the SSD scan (kernels.ssd_combined): v and o (batch, seqlen, nheads, headdim), q and k
(batch, seqlen, ngroups, dstate) shared by the nheads / ngroups heads of a group, g and beta (batch,
seqlen, nheads), states (sequences, nheads, headdim, dstate).  The keys are taken as given: a model that
wants unit keys normalises them first.  The reference has no delta rule; no reference file stands behind this.

* :func:`gated_delta_rule` -- training and prefill, chunks of 64 tokens, forward and backward, plain
  batches or sequences packed end to end (``cu_seqlens``).
* :func:`gated_delta_step` -- decoding: one or a few tokens per row on a cache of states, updated in place.

bf16 / fp16 / fp32 q, k, v; dstate 64 or 128; headdim a multiple of 8 up to 128 (256 for the step).
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib

__all__ = ["gated_delta_rule", "gated_delta_step"]

_T = "P3q"  # a tensor with three strides
_fwd_launch = _lib.Launcher("delta_fwd_launch", _lib.DeltaFwdArgs, "7qif" + _T * 3 + "4P" + _T + "PPNPN2i")
_bwd_launch = _lib.Launcher("delta_bwd_launch", _lib.DeltaBwdArgs,
                            "7qif" + _T * 3 + "3PPN" + _T + "P" + _T * 3 + "3PPN2i")
_step_launch = _lib.Launcher("delta_step_launch", _lib.DeltaStepArgs, "7qif" + _T * 3 + "3P2qP" + _T)

_DSTATES = (64, 128)


def _check(q, k, v, g, beta, what):
    if not v.is_cuda:
        raise ValueError(f"{what}: q, k, v, g and beta must be on CUDA")
    if not (q.get_device() == k.get_device() == v.get_device() == g.get_device() == beta.get_device()):
        raise ValueError(f"{what}: q, k, v, g and beta must be on one device")
    if v.ndim != 4 or q.ndim != 4:
        raise ValueError(f"{what}: q, k (batch, seqlen, ngroups, dstate), v (batch, seqlen, nheads, headdim)")
    b, length, H, V = v.shape
    G, K = q.shape[2], q.shape[3]
    if q.shape != (b, length, G, K) or k.shape != q.shape:
        raise ValueError(f"{what}: q and k must be (batch, seqlen, ngroups, dstate), got {tuple(q.shape)} and "
                         f"{tuple(k.shape)} for v {tuple(v.shape)}")
    if g.shape != (b, length, H) or beta.shape != (b, length, H):
        raise ValueError(f"{what}: g and beta must be (batch, seqlen, nheads)")
    if G == 0 or H == 0 or H % G:
        raise ValueError(f"{what}: nheads {H} must be a multiple of ngroups {G}")
    if v.dtype not in _lib.DTYPE_CODES or q.dtype != v.dtype or k.dtype != v.dtype:
        raise ValueError(f"{what}: q, k and v must share one of bf16, fp16, fp32")
    if K not in _DSTATES:
        raise ValueError(f"{what}: dstate must be 64 or 128, got {K}")
    return b, length, H, V, G, K


def _check_headdim(V, most, what):
    if V == 0 or V % 8 or V > most:
        raise ValueError(f"{what}: headdim must be a multiple of 8 up to {most}, got {V}")


def _rows(t, most=15):
    """t itself where its rows can be addressed as they are: unit last stride, steps of 16 bytes, a base on 16."""
    es = t.element_size()
    a, b, c, d = t.stride()
    if d == 1 and not t.data_ptr() & most:
        n = t.shape
        if not any(m > 1 and (s <= 0 or (s * es) & 15) for s, m in ((a, n[0]), (b, n[1]), (c, n[2]))):
            return t
    return t.clone(memory_format=torch.contiguous_format)


def _strides3(t):
    """Element strides of the three outer axes; an axis of one element, whatever its stride, takes a row's step."""
    a, b, c, _ = t.stride()
    n = t.shape
    return (a if n[0] > 1 else n[3], b if n[1] > 1 else n[3], c if n[2] > 1 else n[3])


def _f32(t):
    return t if t.dtype == torch.float32 and t.is_contiguous() else t.to(torch.float32).contiguous()


def _saved_bytes(b, length, nseq, packed, H, V, K, code, flags):
    """Bytes that a forward keeps for a backward: those of one (chunk, head), which the library knows, times their
    number in plain arithmetic, so that a traced length stays a symbol."""
    slots = length // 64 + nseq if packed else b * ((length + 63) // 64)
    return slots * H * _lib.lib.delta_saved_bytes(1, 1, 0, 1, int(V), int(K), 1, code, flags)


def _delta_fwd(q, k, v, g, beta, initial_states, cu_seqlens, scale, flags, want_final, save):
    """One forward launch: (o, final states or None, what a backward needs or None)."""
    b, length, H, V = v.shape
    G, K = q.shape[2], q.shape[3]
    nseq = b if cu_seqlens is None else cu_seqlens.numel() - 1
    # (the limits stand here: in the traced part they would bound a symbolic size)
    if max(nseq, H) > 65535 or length > 1 << 30 or max(b * ((length + 63) // 64), length // 64 + nseq) > 1 << 24:
        raise ValueError(f"gated_delta_rule: q, k and v of {nseq} sequences, {length} tokens and {H} heads: at most 65535 "
                         "sequences and heads, 2^30 tokens and 2^24 chunks of 64")
    dev, code = v.device, _lib.DTYPE_CODES[v.dtype]
    q, k, v, g, beta = _rows(q), _rows(k), _rows(v), _f32(g), _f32(beta)
    # a packed call's tokens outside every sequence get zeros
    o = (torch.empty if cu_seqlens is None else torch.zeros)(b, length, H, V, dtype=v.dtype, device=dev)
    final = torch.empty(nseq, H, V, K, dtype=torch.float32, device=dev) if want_final else None
    s0 = None if initial_states is None else _f32(initial_states)
    n = (_saved_bytes(b, length, nseq, cu_seqlens is not None, H, V, K, code, flags) if save else
         _lib.lib.delta_workspace_bytes(b, length, nseq, H, V, K, G, code, flags, 0))
    buf = torch.empty(n, dtype=torch.uint8, device=dev)
    at = buf.data_ptr()
    _fwd_launch(v.get_device(), b, length, H, V, K, G, nseq, code, scale, q.data_ptr(), *_strides3(q), k.data_ptr(),
                *_strides3(k), v.data_ptr(), *_strides3(v), g.data_ptr(), beta.data_ptr(), _lib.ptr(cu_seqlens),
                _lib.ptr(s0), o.data_ptr(), *_strides3(o), _lib.ptr(final), *((0, 0, at, n) if save else (at, n, 0, 0)),
                flags, 0)
    return o, final, buf if save else None


def _delta_bwd(q, k, v, g, beta, cu_seqlens, saved, do, d_final, scale, flags, want_d_initial):
    """One backward launch: (dq, dk, dv, dg, dbeta, d initial states or None); dg, dbeta fp32."""
    b, length, H, V = v.shape
    G, K = q.shape[2], q.shape[3]
    nseq = b if cu_seqlens is None else cu_seqlens.numel() - 1
    dev, code = v.device, _lib.DTYPE_CODES[v.dtype]
    q, k, v, g, beta, do = _rows(q), _rows(k), _rows(v), _f32(g), _f32(beta), _rows(do.to(v.dtype))
    new = torch.empty if cu_seqlens is None else torch.zeros
    dq, dk = (new(b, length, G, K, dtype=v.dtype, device=dev) for _ in range(2))
    dv = new(b, length, H, V, dtype=v.dtype, device=dev)
    dg, dbeta = (new(b, length, H, dtype=torch.float32, device=dev) for _ in range(2))
    ds0 = torch.empty(nseq, H, V, K, dtype=torch.float32, device=dev) if want_d_initial else None
    n = _lib.lib.delta_workspace_bytes(b, length, nseq, H, V, K, G, code, flags, 1)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    ds1 = None if d_final is None else _f32(d_final)
    qk, vo = _strides3(dq), _strides3(dv)
    _bwd_launch(v.get_device(), b, length, H, V, K, G, nseq, code, scale, q.data_ptr(), *_strides3(q), k.data_ptr(),
                *_strides3(k), v.data_ptr(), *_strides3(v), g.data_ptr(), beta.data_ptr(), _lib.ptr(cu_seqlens),
                saved.data_ptr(), saved.numel(), do.data_ptr(), *_strides3(do), _lib.ptr(ds1), dq.data_ptr(), *qk,
                dk.data_ptr(), *qk, dv.data_ptr(), *vo, dg.data_ptr(), dbeta.data_ptr(), _lib.ptr(ds0), ws.data_ptr(),
                n, flags, 0)
    return dq, dk, dv, dg, dbeta, ds0


# ---- dispatcher operators: torch.compile traces them, autograd through register_autograd ----
def _empty0(like):
    return like.new_empty((0,), dtype=torch.float32)


@torch.library.custom_op("ema_b200::delta_fwd", mutates_args=(), device_types="cuda")
def _delta_fwd_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                  initial_states: Optional[torch.Tensor], cu_seqlens: Optional[torch.Tensor], scale: float,
                  flags: int = 0) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(o, the final states, what the backward reads)."""
    return _delta_fwd(q, k, v, g, beta, initial_states, cu_seqlens, scale, flags, True, True)


@_delta_fwd_op.register_fake
def _(q, k, v, g, beta, initial_states, cu_seqlens, scale, flags=0):
    b, length, H, V = v.shape
    G, K = q.shape[2], q.shape[3]
    nseq = b if cu_seqlens is None else cu_seqlens.shape[0] - 1
    nbytes = _saved_bytes(b, length, nseq, cu_seqlens is not None, H, V, K, _lib.DTYPE_CODES[v.dtype], flags)
    return (v.new_empty((b, length, H, V)), v.new_empty((nseq, H, V, K), dtype=torch.float32),
            v.new_empty((nbytes,), dtype=torch.uint8))


@torch.library.custom_op("ema_b200::delta_infer", mutates_args=(), device_types="cuda")
def _delta_infer_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                    initial_states: Optional[torch.Tensor], cu_seqlens: Optional[torch.Tensor], scale: float,
                    flags: int, want_final: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """The forward that keeps nothing for a backward: (o, the final states, empty when not wanted)."""
    o, final, _ = _delta_fwd(q, k, v, g, beta, initial_states, cu_seqlens, scale, flags, want_final, False)
    return o, final if want_final else _empty0(v)


@_delta_infer_op.register_fake
def _(q, k, v, g, beta, initial_states, cu_seqlens, scale, flags, want_final):
    b, _, H, V = v.shape
    nseq = b if cu_seqlens is None else cu_seqlens.shape[0] - 1
    return (v.new_empty(v.shape), v.new_empty((nseq, H, V, k.shape[3]), dtype=torch.float32) if want_final
            else _empty0(v))


@torch.library.custom_op("ema_b200::delta_bwd", mutates_args=(), device_types="cuda")
def _delta_bwd_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                  cu_seqlens: Optional[torch.Tensor], saved: torch.Tensor, do: torch.Tensor,
                  d_final: Optional[torch.Tensor], scale: float, flags: int,
                  want_d_initial: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor,
                                                 torch.Tensor]:
    """(dq, dk, dv, dg, dbeta, d initial states), the last empty when not wanted."""
    *grads, ds0 = _delta_bwd(q, k, v, g, beta, cu_seqlens, saved, do, d_final, scale, flags, want_d_initial)
    return (*grads, ds0 if ds0 is not None else _empty0(v))


@_delta_bwd_op.register_fake
def _(q, k, v, g, beta, cu_seqlens, saved, do, d_final, scale, flags, want_d_initial):
    b, length, H, V = v.shape
    G, K = q.shape[2], q.shape[3]
    nseq = b if cu_seqlens is None else cu_seqlens.shape[0] - 1
    f32 = torch.float32
    return (q.new_empty((b, length, G, K)), q.new_empty((b, length, G, K)), v.new_empty((b, length, H, V)),
            v.new_empty((b, length, H), dtype=f32), v.new_empty((b, length, H), dtype=f32),
            v.new_empty((nseq, H, V, K), dtype=f32) if want_d_initial else _empty0(v))


def _setup(ctx, inputs, output):
    q, k, v, g, beta, initial_states, cu_seqlens, scale, flags = inputs
    ctx.save_for_backward(q, k, v, g, beta, cu_seqlens, output[2])
    ctx.scale, ctx.flags = scale, flags
    ctx.d_initial = initial_states is not None and ctx.needs_input_grad[5]
    ctx.initial_dtype = None if initial_states is None else initial_states.dtype
    ctx.set_materialize_grads(False)


def _backward(ctx, do, d_final, _d_saved):
    q, k, v, g, beta, cu, saved = ctx.saved_tensors
    if do is None and d_final is None:
        return (None,) * 9
    if do is None:
        do = torch.zeros_like(v)
    dq, dk, dv, dg, dbeta, ds0 = torch.ops.ema_b200.delta_bwd(q, k, v, g, beta, cu, saved, do, d_final, ctx.scale,
                                                              ctx.flags, ctx.d_initial)
    return (dq, dk, dv, dg.to(g.dtype), dbeta.to(beta.dtype), ds0.to(ctx.initial_dtype) if ctx.d_initial else None,
            None, None, None)


torch.library.register_autograd("ema_b200::delta_fwd", _backward, setup_context=_setup)


class _Rule(torch.autograd.Function):
    """The eager form of the operators above (torch.compile traces the operators)."""

    @staticmethod
    def forward(ctx, q, k, v, g, beta, initial_states, cu_seqlens, scale, flags, want_final):
        o, final, saved = _delta_fwd(q, k, v, g, beta, initial_states, cu_seqlens, scale, flags, want_final, True)
        ctx.save_for_backward(q, k, v, g, beta, cu_seqlens, saved)
        ctx.scale, ctx.flags = scale, flags
        ctx.initial_dtype = None if initial_states is None else initial_states.dtype
        ctx.set_materialize_grads(False)
        return o, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do, d_final):
        q, k, v, g, beta, cu, saved = ctx.saved_tensors
        if do is None and d_final is None:
            return (None,) * 10
        if do is None:
            do = torch.zeros_like(v)
        want = ctx.initial_dtype is not None and ctx.needs_input_grad[5]
        dq, dk, dv, dg, dbeta, ds0 = _delta_bwd(q, k, v, g, beta, cu, saved, do, d_final, ctx.scale, ctx.flags, want)
        return (dq, dk, dv, dg.to(g.dtype), dbeta.to(beta.dtype), ds0.to(ctx.initial_dtype) if want else None,
                None, None, None, None)


def gated_delta_rule(q, k, v, g, beta, scale=None, initial_states=None, return_final_states=False, cu_seqlens=None,
                     fp32_products=False):
    """o (batch, seqlen, nheads, headdim), or (o, final states) with ``return_final_states``.

    g is the log decay (not positive in a decaying layer; at or below -100 the state is dropped; a NaN makes NaN of
    its head's results from its token on and of those before it in its chunk of 64), beta the write strength, ``scale``
    defaults to dstate ** -0.5.  ``initial_states`` (sequences, nheads, headdim, dstate) is the state before the first
    token.  ``cu_seqlens`` (nseq + 1, int32 or int64, on the device) packs sequences into a batch of one: sequence n is
    tokens [cu[n], cu[n + 1]), of any length, zero too (its final state is its initial one); tokens outside every
    sequence give zeros.

    Gradients: q, k, v, g, beta and initial_states; those of a group's q and k sum over its heads.  The states,
    all sums and both gate gradients are fp32.  bf16 calls run on the tensor cores with their 32-bit operands as
    pairs or threes of bf16: 2^-16 of each, 2e-6 to 4e-6 of a state or gate gradient (a plain fp32 form: 2e-7 to 4e-7).
    Where keys repeat and beta is near one, the gate gradients are small differences of large terms and keep fewer
    digits (130 equal keys at beta 0.98: 0.8 % of dg and 1.5e-4 of dbeta; at beta 0.9, 6e-4 and 5e-5);
    ``fp32_products`` then gives those of fp32 arithmetic (0.06 % and 1.5e-6; 5e-5 and 1.2e-6), at about seventeen times
    the time.  fp16 and fp32 calls are always fp32 products."""
    b, length, H, V, G, K = _check(q, k, v, g, beta, "gated_delta_rule")
    _check_headdim(V, 128, "gated_delta_rule")
    nseq = b
    if cu_seqlens is not None:
        if b != 1:
            raise ValueError("gated_delta_rule: packed sequences come as a batch of one")
        if cu_seqlens.ndim != 1 or cu_seqlens.numel() < 1 or cu_seqlens.dtype not in (torch.int32, torch.int64):
            raise ValueError("gated_delta_rule: cu_seqlens must be (nseq + 1,) int32 or int64")
        if cu_seqlens.device != v.device:
            raise ValueError("gated_delta_rule: cu_seqlens must be on v's device")
        nseq = cu_seqlens.numel() - 1
        if cu_seqlens.dtype == torch.int64:
            # clamped before the narrowing, as the kernels clamp: past 32 bits an offset is still the call's end
            cu_seqlens = cu_seqlens.clamp(0, length).to(torch.int32)
        cu_seqlens = cu_seqlens.contiguous()
    if initial_states is not None:
        if initial_states.shape != (nseq, H, V, K) or initial_states.device != v.device:
            raise ValueError(f"gated_delta_rule: initial_states must be {(nseq, H, V, K)} on v's device, got "
                             f"{tuple(initial_states.shape)}")
    scale = K ** -0.5 if scale is None else float(scale)
    flags = _lib.DELTA_FP32_PRODUCTS if fp32_products else 0
    train = torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in (q, k, v, g, beta, initial_states))
    if torch.compiler.is_compiling():
        if train:
            o, final, _ = torch.ops.ema_b200.delta_fwd(q, k, v, g, beta, initial_states, cu_seqlens, scale, flags)
        else:
            o, final = torch.ops.ema_b200.delta_infer(q, k, v, g, beta, initial_states, cu_seqlens, scale, flags,
                                                      return_final_states)
    elif train:
        o, final = _Rule.apply(q, k, v, g, beta, initial_states, cu_seqlens, scale, flags, return_final_states)
    else:
        o, final, _ = _delta_fwd(q, k, v, g, beta, initial_states, cu_seqlens, scale, flags, return_final_states,
                                 False)
    return (o, final) if return_final_states else o


_BLOCKS = "gated_delta_step: the (headdim, dstate) block of a state must be contiguous, 16-byte aligned and its own"


def _overlap(n, s0, m, s1, size):
    """Whether two of n x m blocks of ``size`` elements, s0 and s1 apart, share one (a step writes all of them at once)."""
    if (n > 1 and s0 < size) or (m > 1 and s1 < size):
        return True
    if n <= 1 or m <= 1 or s0 >= (m - 1) * s1 + size or s1 >= (n - 1) * s0 + size:
        return False
    for j in range(1, m):  # neither axis steps over the whole of the other: j s1 against the multiples of s0 beside it
        i, rest = divmod(j * s1, s0)
        if (i < n and rest < size) or (i + 1 < n and s0 - rest < size):
            return True
    return False


def _delta_step(q, k, v, g, beta, states, state_indices, scale):
    b, T, H, V = v.shape
    if b > 65535 or H > 65535 or T > 1048576:
        raise ValueError(f"gated_delta_step: v of {b} rows, {T} tokens and {H} heads: at most 65535 rows and heads and 2^20 "
                         "tokens")
    if states.data_ptr() & 15:  # (here: an address is nothing that a trace has)
        raise ValueError(_BLOCKS)
    o = torch.empty(b, T, H, V, dtype=v.dtype, device=v.device)
    q, k, g, beta = _rows(q), _rows(k), _f32(g), _f32(beta)
    if v.stride(3) != 1:
        v = v.clone(memory_format=torch.contiguous_format)
    ss = states.stride()
    _step_launch(v.get_device(), b, T, H, V, q.shape[3], q.shape[2], states.shape[0], _lib.DTYPE_CODES[v.dtype], scale,
                 q.data_ptr(), *_strides3(q), k.data_ptr(), *_strides3(k), v.data_ptr(), *_strides3(v), g.data_ptr(),
                 beta.data_ptr(), states.data_ptr(), ss[0], ss[1], _lib.ptr(state_indices), o.data_ptr(), T * H * V,
                 H * V, V)
    return o


@torch.library.custom_op("ema_b200::delta_step", mutates_args=("states",), device_types="cuda")
def _delta_step_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                   states: torch.Tensor, state_indices: Optional[torch.Tensor], scale: float) -> torch.Tensor:
    return _delta_step(q, k, v, g, beta, states, state_indices, scale)


@_delta_step_op.register_fake
def _(q, k, v, g, beta, states, state_indices, scale):
    return torch.empty_like(v, memory_format=torch.contiguous_format)


def gated_delta_step(q, k, v, g, beta, states, scale=None, state_indices=None):
    """The recurrent form for decoding: o (batch, tokens, nheads, headdim), ``states`` updated in place.

    q, k (batch, tokens, ngroups, dstate), v (batch, tokens, nheads, headdim), g, beta (batch, tokens,
    nheads), tokens usually one; the token axis may be left out of all of them (and is then left out of o).  ``states``
    (slots, nheads, headdim, dstate) fp32 is the cache; row b works on slot ``state_indices[b]`` (int32 or
    int64 on the device; b itself when None).  An index outside the cache marks an idle row: its output is zero and no
    state changes.  Rows of one call must not share a slot.  No gradient."""
    squeeze = v.ndim == 3
    if squeeze:
        q, k, v, g, beta = (t.unsqueeze(1) for t in (q, k, v, g, beta))
    b, _, H, V, _, K = _check(q, k, v, g, beta, "gated_delta_step")
    _check_headdim(V, 256, "gated_delta_step")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or g.requires_grad
                                    or beta.requires_grad or states.requires_grad):
        raise ValueError("gated_delta_step has no gradient: call it under torch.no_grad() or use gated_delta_rule")
    if states.shape[1:] != (H, V, K) or states.dtype != torch.float32:
        raise ValueError(f"gated_delta_step: states must be (slots, {H}, {V}, {K}) fp32, got {tuple(states.shape)} "
                         f"{states.dtype}")
    if states.get_device() != v.get_device():
        raise ValueError("gated_delta_step: states must be on v's device")
    s0, s1, s2, s3 = states.stride()
    if s3 != 1 or s2 != K or s0 % 4 or s1 % 4 or _overlap(states.shape[0], s0, H, s1, V * K):
        raise ValueError(_BLOCKS)
    if state_indices is None:
        if states.shape[0] < b:
            raise ValueError(f"gated_delta_step: {b} rows on {states.shape[0]} slots")
    else:
        if state_indices.shape != (b,) or state_indices.dtype not in (torch.int32, torch.int64):
            raise ValueError("gated_delta_step: state_indices must be (batch,) int32 or int64")
        if state_indices.get_device() != v.get_device():
            raise ValueError("gated_delta_step: state_indices must be on v's device")
        if state_indices.dtype == torch.int64:
            # clamped before the narrowing, so that a huge index stays outside the cache
            state_indices = state_indices.clamp(-1, states.shape[0]).to(torch.int32)
        state_indices = state_indices.contiguous()
    scale = K ** -0.5 if scale is None else float(scale)
    if torch.compiler.is_compiling():
        o = torch.ops.ema_b200.delta_step(q, k, v, g, beta, states, state_indices, scale)
    else:
        o = _delta_step(q, k, v, g, beta, states, state_indices, scale)
        torch.autograd.graph.increment_version(states)  # written in place: a backward that saved them has to know
    return o.squeeze(1) if squeeze else o
