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


def _rows2d(t, dim):
    """t as (rows, dim) with unit channel stride: a view where its strides allow one."""
    if t.ndim != 2:
        t = t.reshape(-1, dim)
    return t if t.stride(1) == 1 and t.stride(0) >= 0 else t.contiguous()


def _workspace(rows, dim, group, dev):
    n = _lib.lib.block_norm_workspace_bytes(rows, dim, group)
    return torch.empty(n, dtype=torch.uint8, device=dev), n


def _gated_args(x, z, weight, eps, group_size, before):
    a = _lib.GatedNormArgs()
    a.rows, a.dim, a.group_size = x.shape[0], x.shape[1], group_size
    a.dtype, a.weight_dtype = _lib.DTYPE_CODES[x.dtype], _lib.DTYPE_CODES[weight.dtype]
    a.norm_before_gate, a.eps = int(before), eps
    a.x, a.x_stride, a.z, a.z_stride = x.data_ptr(), x.stride(0), z.data_ptr(), z.stride(0)
    a.weight = weight.data_ptr()
    return a


def _gated_fwd(x, z, weight, eps, group_size, before):
    dim = x.shape[-1]
    x2, z2, w = _rows2d(x, dim), _rows2d(z, dim), weight.contiguous()
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    a = _gated_args(x2, z2, w, eps, group_size, before)
    a.y, a.y_stride = y.data_ptr(), dim
    with torch.cuda.device(x.device):
        _lib.check(_lib.lib.gated_norm_fwd_launch(a, _lib.stream_ptr(x.device)), "rms_norm_gated")
    return y


def _gated_bwd(x, z, weight, dy, eps, group_size, before):
    dim, dev = x.shape[-1], x.device
    x2, z2, w, d2 = _rows2d(x, dim), _rows2d(z, dim), weight.contiguous(), _rows2d(dy.to(x.dtype), dim)
    dx, dz = (torch.empty(x.shape, dtype=x.dtype, device=dev) for _ in range(2))
    dw = torch.empty(dim, dtype=torch.float32, device=dev)
    a = _gated_args(x2, z2, w, eps, group_size, before)
    a.dy, a.dy_stride = d2.data_ptr(), d2.stride(0)
    a.dx, a.dx_stride, a.dz, a.dz_stride, a.dweight = dx.data_ptr(), dim, dz.data_ptr(), dim, dw.data_ptr()
    ws, n = _workspace(x2.shape[0], dim, group_size, dev)
    a.workspace, a.workspace_bytes = ws.data_ptr(), n
    with torch.cuda.device(dev):
        _lib.check(_lib.lib.gated_norm_bwd_launch(a, _lib.stream_ptr(dev)), "rms_norm_gated backward")
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


def _check_weight(x, weight, what):
    if not x.is_cuda or not weight.is_cuda or weight.device != x.device:
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
    z = z.to(x.dtype)
    if torch.compiler.is_compiling() or (
            torch.is_grad_enabled() and (x.requires_grad or z.requires_grad or weight.requires_grad)):
        return torch.ops.ema_b200.gated_norm_fwd(x, z, weight, float(eps), group_size, bool(norm_before_gate))
    return _gated_fwd(x, z, weight, float(eps), group_size, bool(norm_before_gate))


def _residual_args(rows, dim, dtype, residual_dtype, weight, eps, scale):
    a = _lib.ResidualNormArgs()
    a.rows, a.dim, a.eps, a.scale = rows, dim, eps, scale
    a.dtype, a.residual_dtype = _lib.DTYPE_CODES[dtype], _lib.DTYPE_CODES[residual_dtype]
    a.weight_dtype, a.weight = _lib.DTYPE_CODES[weight.dtype], weight.data_ptr()
    return a


def _residual_fwd(x, residual, weight, eps, scale):
    dim, dev = x.shape[-1], x.device
    rdtype = x.dtype if residual is None else residual.dtype
    x2, r2, w = _rows2d(x, dim), None if residual is None else _rows2d(residual, dim), weight.contiguous()
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    h = torch.empty(x.shape, dtype=rdtype, device=dev)
    a = _residual_args(x2.shape[0], dim, x.dtype, rdtype, w, eps, scale)
    a.x, a.x_stride = x2.data_ptr(), x2.stride(0)
    if r2 is not None:
        a.residual, a.residual_stride = r2.data_ptr(), r2.stride(0)
    a.y, a.y_stride, a.h, a.h_stride = y.data_ptr(), dim, h.data_ptr(), dim
    with torch.cuda.device(dev):
        _lib.check(_lib.lib.residual_norm_fwd_launch(a, _lib.stream_ptr(dev)), "residual_rms_norm")
    return y, h


def _residual_bwd(h, weight, dy, dh, eps, scale, want_residual):
    dim, dev = h.shape[-1], h.device
    h2, w, d2 = _rows2d(h, dim), weight.contiguous(), _rows2d(dy, dim)
    dx = torch.empty(h.shape, dtype=dy.dtype, device=dev)
    dr = torch.empty(h.shape, dtype=h.dtype, device=dev) if want_residual else None
    dw = torch.empty(dim, dtype=torch.float32, device=dev)
    a = _residual_args(h2.shape[0], dim, dy.dtype, h.dtype, w, eps, scale)
    a.h, a.h_stride, a.dy, a.dy_stride = h2.data_ptr(), h2.stride(0), d2.data_ptr(), d2.stride(0)
    if dh is not None:
        dh = _rows2d(dh.to(h.dtype), dim)
        a.dh, a.dh_stride = dh.data_ptr(), dh.stride(0)
    a.dx, a.dx_stride, a.dweight = dx.data_ptr(), dim, dw.data_ptr()
    if dr is not None:
        a.d_residual, a.d_residual_stride = dr.data_ptr(), dim
    ws, n = _workspace(h2.shape[0], dim, dim, dev)
    a.workspace, a.workspace_bytes = ws.data_ptr(), n
    with torch.cuda.device(dev):
        _lib.check(_lib.lib.residual_norm_bwd_launch(a, _lib.stream_ptr(dev)), "residual_rms_norm backward")
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
    if torch.compiler.is_compiling() or (torch.is_grad_enabled() and (
            x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad))):
        return torch.ops.ema_b200.residual_norm_fwd(x, residual, weight, float(eps), float(scale))
    return _residual_fwd(x, residual, weight, float(eps), float(scale))
