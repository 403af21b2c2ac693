"""Norms around a block, fused with its gate and its residual scale, on the B200 kernels (autograd).

* :func:`rms_norm_gated` -- behind a scan: the RMS norm of its output over groups of channels with the
  gate silu(z), in either order (per-head norms first, Mamba-2's gate first).
* :func:`residual_rms_norm` -- before the next block: h = residual + scale x and the RMS norm of h, one pass.

One element type per call (bf16 / fp16 / fp32; the residual stream may be fp32 beside 16-bit blocks),
fp32 arithmetic, each result rounded once; the weight in any of the three types.  The reference has no norms; no
reference file stands behind this.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib

__all__ = ["rms_norm_gated", "residual_rms_norm"]


_GATED = "3q3if" + "Pq" * 2 + "P" + "Pq" * 4 + "2PN"
_RESIDUAL = "2q3i2fi" + "Pq" * 2 + "P" + "Pq" * 6 + "2PN"
_gated_fwd_launch = _lib.Launcher("gated_norm_fwd_launch", _lib.GatedNormArgs, _GATED)
_gated_bwd_launch = _lib.Launcher("gated_norm_bwd_launch", _lib.GatedNormArgs, _GATED)
_residual_fwd_launch = _lib.Launcher("residual_norm_fwd_launch", _lib.ResidualNormArgs, _RESIDUAL)
_residual_bwd_launch = _lib.Launcher("residual_norm_bwd_launch", _lib.ResidualNormArgs, _RESIDUAL)
_CODES = _lib.DTYPE_CODES


def _rows2d(t, dim):
    """t as (rows, dim) with unit channel stride: a view where its strides allow one."""
    if t.ndim != 2:
        t = t.reshape(-1, dim)
    s = t.stride()
    return t if s[1] == 1 and s[0] >= 0 else t.contiguous()


def _workspace(rows, dim, group, dev):
    n = _lib.lib.block_norm_workspace_bytes(rows, dim, group)
    return torch.empty(n, dtype=torch.uint8, device=dev), n


def _gated_fwd(x, z, weight, eps, group_size, before):
    dim = x.shape[-1]
    if dim // group_size > 65535 or dim > 1 << 30:
        raise ValueError(f"rms_norm_gated: x of {dim} channels in groups of {group_size}: at most 65535 groups and 2^30 "
                         "channels")
    x2, z2, w = _rows2d(x, dim), _rows2d(z, dim), weight.contiguous()
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    _gated_fwd_launch(x.get_device(), x2.shape[0], dim, group_size, _CODES[x.dtype], _CODES[w.dtype], before, eps,
                      x2.data_ptr(), x2.stride(0), z2.data_ptr(), z2.stride(0), w.data_ptr(), y.data_ptr(), dim,
                      0, 0, 0, 0, 0, 0, 0, 0, 0)
    return y


def _gated_bwd(x, z, weight, dy, eps, group_size, before):
    dim, dev = x.shape[-1], x.device
    x2, z2, w, d2 = _rows2d(x, dim), _rows2d(z, dim), weight.contiguous(), _rows2d(dy.to(x.dtype), dim)
    dx, dz = (torch.empty(x.shape, dtype=x.dtype, device=dev) for _ in range(2))
    dw = torch.empty(dim, dtype=torch.float32, device=dev)
    ws, n = _workspace(x2.shape[0], dim, group_size, dev)
    _gated_bwd_launch(x.get_device(), x2.shape[0], dim, group_size, _CODES[x.dtype], _CODES[w.dtype], before, eps,
                      x2.data_ptr(), x2.stride(0), z2.data_ptr(), z2.stride(0), w.data_ptr(), 0, 0,
                      d2.data_ptr(), d2.stride(0), dx.data_ptr(), dim, dz.data_ptr(), dim, dw.data_ptr(),
                      ws.data_ptr(), n)
    return dx, dz, dw


@torch.library.custom_op("ema_b200::gated_norm_fwd", mutates_args=(), device_types="cuda")
def _gated_fwd_op(x: torch.Tensor, z: torch.Tensor, weight: torch.Tensor, eps: float, group_size: int,
                  norm_before_gate: bool) -> torch.Tensor:
    return _gated_fwd(x, z, weight, eps, group_size, norm_before_gate)


@_gated_fwd_op.register_fake
def _(x, z, weight, eps, group_size, norm_before_gate):
    return x.new_empty(x.shape)


@torch.library.custom_op("ema_b200::gated_norm_bwd", mutates_args=(), device_types="cuda")
def _gated_bwd_op(x: torch.Tensor, z: torch.Tensor, weight: torch.Tensor, dy: torch.Tensor, eps: float,
                  group_size: int, norm_before_gate: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dz, dweight); dweight fp32."""
    return _gated_bwd(x, z, weight, dy, eps, group_size, norm_before_gate)


@_gated_bwd_op.register_fake
def _(x, z, weight, dy, eps, group_size, norm_before_gate):
    return x.new_empty(x.shape), x.new_empty(x.shape), x.new_empty((x.shape[-1],), dtype=torch.float32)


def _gated_setup(ctx, inputs, output):
    x, z, weight, *ctx.opts = inputs
    ctx.save_for_backward(x, z, weight)


def _gated_backward(ctx, dy):
    x, z, weight = ctx.saved_tensors
    dx, dz, dw = torch.ops.ema_b200.gated_norm_bwd(x, z, weight, dy, *ctx.opts)
    return dx, dz, dw.to(weight.dtype), None, None, None


torch.library.register_autograd("ema_b200::gated_norm_fwd", _gated_backward, setup_context=_gated_setup)


class _Gated(torch.autograd.Function):
    """The eager form of the operators above (torch.compile traces the operators)."""

    @staticmethod
    def forward(ctx, x, z, weight, eps, group_size, before):
        ctx.save_for_backward(x, z, weight)
        ctx.opts = (eps, group_size, before)
        return _gated_fwd(x, z, weight, eps, group_size, before)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, z, weight = ctx.saved_tensors
        dx, dz, dw = _gated_bwd(x, z, weight, dy, *ctx.opts)
        return dx, dz, dw.to(weight.dtype), None, None, None


def _check_weight(x, weight, what):
    if not x.is_cuda or weight.device != x.device:
        raise ValueError(f"{what}: the tensors must be on one CUDA device")
    if x.ndim < 1 or x.shape[-1] == 0 or weight.shape != (x.shape[-1],):
        raise ValueError(f"{what}: weight must be ({x.shape[-1] if x.ndim else 0},), got {tuple(weight.shape)}")
    if x.dtype not in _lib.DTYPE_CODES or weight.dtype not in _lib.DTYPE_CODES:
        raise ValueError(f"{what}: bf16, fp16 or fp32 tensors")


def rms_norm_gated(x, z, weight, eps=1e-5, group_size=None, norm_before_gate=True):
    """x rstd(x) weight silu(z) (``norm_before_gate``), or with t = x silu(z): t rstd(t) weight.

    x and z (..., dim); rstd over each ``group_size`` channels (dim when None), (mean of squares + eps)^-1/2; weight
    (dim,).  z is taken in x's type (its gradient returns in z's own)."""
    _check_weight(x, weight, "rms_norm_gated")
    if z.shape != x.shape or z.device != x.device:
        raise ValueError(f"rms_norm_gated: z must have x's shape and device, got {tuple(z.shape)} for {tuple(x.shape)}")
    dim = x.shape[-1]
    group_size = dim if group_size is None else int(group_size)
    if group_size <= 0 or dim % group_size:
        raise ValueError(f"rms_norm_gated: group_size {group_size} must divide {dim}")
    if not eps >= 0:
        raise ValueError("rms_norm_gated: eps must not be negative")
    if z.dtype != x.dtype:
        z = z.to(x.dtype)
    if torch.compiler.is_compiling():
        return torch.ops.ema_b200.gated_norm_fwd(x, z, weight, float(eps), group_size, bool(norm_before_gate))
    if torch.is_grad_enabled() and (x.requires_grad or z.requires_grad or weight.requires_grad):
        return _Gated.apply(x, z, weight, float(eps), group_size, bool(norm_before_gate))
    return _gated_fwd(x, z, weight, float(eps), group_size, bool(norm_before_gate))


class _Residual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps, scale):
        y, h = _residual_fwd(x, residual, weight, eps, scale)
        ctx.save_for_backward(weight, h)
        ctx.has_residual, ctx.x_dtype, ctx.eps, ctx.scale = residual is not None, x.dtype, eps, scale
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh):
        weight, h = ctx.saved_tensors
        if dy is None and dh is None:
            return (None,) * 5
        dy = torch.zeros(h.shape, dtype=ctx.x_dtype, device=h.device) if dy is None else dy.to(ctx.x_dtype)
        want = ctx.has_residual and ctx.needs_input_grad[1]
        dx, dr, dw = _residual_bwd(h, weight, dy, dh, ctx.eps, ctx.scale, want)
        return dx, dr, dw.to(weight.dtype), None, None


def _residual_fwd(x, residual, weight, eps, scale):
    dim, dev = x.shape[-1], x.device
    if dim > 1 << 30:
        raise ValueError(f"residual_rms_norm: x of {dim} channels: at most 2^30")
    x2, w = _rows2d(x, dim), weight.contiguous()
    if residual is None:
        rdtype, rptr, rstride = x.dtype, 0, 0
    else:
        r2 = _rows2d(residual, dim)
        rdtype, rptr, rstride = residual.dtype, r2.data_ptr(), r2.stride(0)
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    h = torch.empty(x.shape, dtype=rdtype, device=dev)
    _residual_fwd_launch(x.get_device(), x2.shape[0], dim, _CODES[x.dtype], _CODES[rdtype], _CODES[w.dtype], eps, scale,
                         0, x2.data_ptr(), x2.stride(0), rptr, rstride, w.data_ptr(), y.data_ptr(), dim, h.data_ptr(),
                         dim, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
    return y, h


def _residual_bwd(h, weight, dy, dh, eps, scale, want_residual):
    dim, dev = h.shape[-1], h.device
    h2, w, d2 = _rows2d(h, dim), weight.contiguous(), _rows2d(dy, dim)
    dx = torch.empty(h.shape, dtype=dy.dtype, device=dev)
    dr = torch.empty(h.shape, dtype=h.dtype, device=dev) if want_residual else None
    dw = torch.empty(dim, dtype=torch.float32, device=dev)
    if dh is not None:
        dh = _rows2d(dh.to(h.dtype), dim)
    ws, n = _workspace(h2.shape[0], dim, dim, dev)
    _residual_bwd_launch(h.get_device(), h2.shape[0], dim, _CODES[dy.dtype], _CODES[h.dtype], _CODES[w.dtype], eps,
                         scale, 0, 0, 0, 0, 0, w.data_ptr(), 0, 0, h2.data_ptr(), h2.stride(0), d2.data_ptr(),
                         d2.stride(0), *((0, 0) if dh is None else (dh.data_ptr(), dh.stride(0))), dx.data_ptr(), dim,
                         _lib.ptr(dr), dim, dw.data_ptr(), ws.data_ptr(), n)
    return dx, dr, dw


@torch.library.custom_op("ema_b200::residual_norm_fwd", mutates_args=(), device_types="cuda")
def _residual_fwd_op(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float,
                     scale: float) -> tuple[torch.Tensor, torch.Tensor]:
    """(y, h)."""
    return _residual_fwd(x, residual, weight, eps, scale)


@_residual_fwd_op.register_fake
def _(x, residual, weight, eps, scale):
    return x.new_empty(x.shape), x.new_empty(x.shape, dtype=x.dtype if residual is None else residual.dtype)


@torch.library.custom_op("ema_b200::residual_norm_bwd", mutates_args=(), device_types="cuda")
def _residual_bwd_op(h: torch.Tensor, weight: torch.Tensor, dy: torch.Tensor, dh: Optional[torch.Tensor], eps: float,
                     scale: float, want_residual: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, d residual (empty when not wanted), dweight); dweight fp32."""
    dx, dr, dw = _residual_bwd(h, weight, dy, dh, eps, scale, want_residual)
    return dx, dr if dr is not None else h.new_empty((0,)), dw


@_residual_bwd_op.register_fake
def _(h, weight, dy, dh, eps, scale, want_residual):
    return (dy.new_empty(h.shape), h.new_empty(h.shape) if want_residual else h.new_empty((0,)),
            h.new_empty((h.shape[-1],), dtype=torch.float32))


def _residual_setup(ctx, inputs, output):
    x, residual, weight, ctx.eps, ctx.scale = inputs
    ctx.save_for_backward(weight, output[1])
    ctx.has_residual, ctx.x_dtype = residual is not None, x.dtype
    ctx.set_materialize_grads(False)


def _residual_backward(ctx, dy, dh):
    weight, h = ctx.saved_tensors
    if dy is None and dh is None:
        return (None,) * 5
    if dy is None:
        dy = torch.zeros(h.shape, dtype=ctx.x_dtype, device=h.device)
    want = ctx.has_residual and ctx.needs_input_grad[1]
    dx, dr, dw = torch.ops.ema_b200.residual_norm_bwd(h, weight, dy.to(ctx.x_dtype), dh, ctx.eps, ctx.scale, want)
    return dx, dr if want else None, dw.to(weight.dtype), None, None


torch.library.register_autograd("ema_b200::residual_norm_fwd", _residual_backward, setup_context=_residual_setup)


def residual_rms_norm(x, residual, weight, eps=1e-5, scale=1.0):
    """(y, h): h = residual + scale x, rounded to the residual's type, and y = h rstd(h) weight in x's type.

    x and residual (..., dim), the residual in x's type or fp32 (None: h = scale x in x's type, a model's
    first block); ``scale`` a number.  y is the norm of h as returned."""
    _check_weight(x, weight, "residual_rms_norm")
    if residual is not None:
        if residual.shape != x.shape or residual.device != x.device:
            raise ValueError(f"residual_rms_norm: residual must have x's shape and device, got "
                             f"{tuple(residual.shape)} for {tuple(x.shape)}")
        if residual.dtype not in (x.dtype, torch.float32):
            raise ValueError("residual_rms_norm: the residual has x's type or fp32")
    if not eps >= 0:
        raise ValueError("residual_rms_norm: eps must not be negative")
    if torch.compiler.is_compiling():
        return torch.ops.ema_b200.residual_norm_fwd(x, residual, weight, float(eps), float(scale))
    if torch.is_grad_enabled() and (
            x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad)):
        return _Residual.apply(x, residual, weight, float(eps), float(scale))
    return _residual_fwd(x, residual, weight, float(eps), float(scale))
