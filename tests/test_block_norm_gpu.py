"""The norms around a block on the B200 against float64.

Tolerances: everything is computed in fp32 sums, 1e-5 of the result's root mean square (weight gradients sum over
the rows); a 16-bit output is rounded once on top, by at most 2^-8 (bf16) or 2^-11 (fp16) of the element, or half
the spacing of fp16's subnormals, 2^-25."""

import numpy as np
import pytest
import torch

from oracle import delta_oracle as do_

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
FP32_REL = 1e-5
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _hold(name, got, want):
    assert torch.isfinite(got).all(), name
    a = got.detach().double().cpu().numpy()
    assert a.shape == want.shape, name
    fp32 = FP32_REL * np.maximum(np.sqrt(np.mean(want ** 2)), np.abs(want))
    bad = np.abs(a - want) > fp32 + ROUND[got.dtype] * (np.abs(want) + fp32) + 2.0 ** -25 * (got.dtype == torch.float16)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.size} elements off, worst {np.abs(a - want).max():.2e}"


def _rand(seed, *shapes):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(*s, device=DEV, generator=g) for s in shapes]


def _f64(t):
    return t.detach().double().cpu().numpy()


WIDTHS = [(64, 64), (128, 128), (384, 128), (96, 96), (256, 256), (512, 512), (1000, 1000), (2048, 1024), (4096, 4096),
          (8192, 8192), (9000, 9000), (777, 777), (21, 7), (2100, 2100), (1, 1)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("D,group", WIDTHS)
@pytest.mark.parametrize("before", [True, False])
def test_gated_norm(D, group, before, dt):
    from kernels.block_norm import rms_norm_gated
    rows = 37
    x, z, dy, w = _rand(D, (rows, D), (rows, D), (rows, D), (D,))
    x, z, dy = x.to(dt).requires_grad_(), z.to(dt).requires_grad_(), dy.to(dt)
    w = (1 + 0.2 * w).requires_grad_()
    y = rms_norm_gated(x, z, w, group_size=group, norm_before_gate=before)
    dx, dz, dw = torch.autograd.grad(y, [x, z, w], dy)
    with torch.no_grad():
        assert torch.equal(rms_norm_gated(x, z, w, group_size=group, norm_before_gate=before), y)
    r = do_.gated_norm(_f64(x), _f64(z), _f64(w), 1e-5, group, before, _f64(dy))
    for name, got in (("y", y), ("dx", dx), ("dz", dz), ("dw", dw)):
        _hold(name, got, r[name])


@pytest.mark.parametrize("dt,rdt", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                    (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                    (torch.float16, torch.float32)])
@pytest.mark.parametrize("D", [64, 128, 256, 512, 1000, 2048, 4096, 8192, 9000, 777, 3])
def test_residual_norm(D, dt, rdt):
    from kernels.block_norm import residual_rms_norm
    rows, scale = 29, 0.7
    x, r, dy, dh, w = _rand(D, (rows, D), (rows, D), (rows, D), (rows, D), (D,))
    x, r, dy, dh = x.to(dt).requires_grad_(), r.to(rdt).requires_grad_(), dy.to(dt), dh.to(rdt)
    w = (1 + 0.2 * w).requires_grad_()
    y, h = residual_rms_norm(x, r, w, scale=scale)
    dx, dr, dw = torch.autograd.grad([y, h], [x, r, w], [dy, dh])
    with torch.no_grad():
        y2, h2 = residual_rms_norm(x, r, w, scale=scale)
    assert torch.equal(y, y2) and torch.equal(h, h2)
    e = do_.residual_norm(_f64(x), _f64(r), _f64(w), 1e-5, scale, _f64(h), _f64(dy), _f64(dh))
    for name, got, want in (("h", h, e["h"]), ("y", y, e["y"]), ("dx", dx, e["dx"]), ("dr", dr, e["dh_total"]),
                            ("dw", dw, e["dw"])):
        _hold(name, got, want)


def test_residual_norm_without_a_residual_and_with_one_gradient():
    from kernels.block_norm import residual_rms_norm
    x, w, dy = _rand(1, (5, 64), (64,), (5, 64))
    x.requires_grad_()
    y, h = residual_rms_norm(x, None, w, scale=0.5)
    e = do_.residual_norm(_f64(x), None, _f64(w), 1e-5, 0.5, None, _f64(dy))
    _hold("y", y, e["y"])
    _hold("h", h, e["h"])
    _hold("dx", torch.autograd.grad(y, x, dy, retain_graph=True)[0], e["dx"])
    _hold("dx from h", torch.autograd.grad(h, x, dy)[0], 0.5 * _f64(dy))


@pytest.mark.parametrize("dt", TYPES)
def test_shapes_strides_and_weights(dt):
    """Leading axes, a slice of a fused projection (its rows off 16 bytes), a 16-bit weight, a gate of another type."""
    from kernels.block_norm import rms_norm_gated
    fused, w = _rand(2, (2, 9, 3 * 64 + 1), (64,))
    fused = fused.to(dt)
    x, z = fused[..., 1:65], fused[..., 65:129]
    for wt in TYPES:
        a = rms_norm_gated(x, z, w.to(wt))
        b = rms_norm_gated(x.contiguous(), z.contiguous(), w.to(wt).float())
        assert torch.equal(a, b) and a.shape == x.shape
    assert torch.equal(rms_norm_gated(x, z.double(), w), rms_norm_gated(x, z, w))
    one = rms_norm_gated(x[0, 0], z[0, 0], w)
    assert torch.equal(one, rms_norm_gated(x, z, w)[0, 0])


def test_zero_rows_and_zero_values():
    from kernels.block_norm import residual_rms_norm, rms_norm_gated
    w = torch.ones(64, device=DEV, requires_grad=True)
    x = torch.empty(0, 64, device=DEV, requires_grad=True)
    y = rms_norm_gated(x, x, w)
    assert y.shape == (0, 64) and (torch.autograd.grad(y.sum(), w)[0] == 0).all()
    zero = torch.zeros(3, 64, device=DEV, requires_grad=True)
    y, h = residual_rms_norm(zero, zero, w)
    d = torch.autograd.grad(y.sum(), zero)[0]
    assert (y == 0).all() and (h == 0).all() and torch.isfinite(d).all()


def test_weight_gradient_is_the_same_every_run():
    from kernels.block_norm import rms_norm_gated
    x, z, dy, w = _rand(3, (5000, 128), (5000, 128), (5000, 128), (128,))
    for t in (x, z, w):
        t.requires_grad_()
    runs = [torch.autograd.grad(rms_norm_gated(x, z, w), [x, z, w], dy) for _ in range(3)]
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


def test_refusals():
    from kernels.block_norm import residual_rms_norm, rms_norm_gated
    x, w = torch.zeros(3, 64, device=DEV), torch.ones(64, device=DEV)
    for bad in (lambda: rms_norm_gated(x, x[:2], w), lambda: rms_norm_gated(x, x, w[:32]),
                lambda: rms_norm_gated(x, x, w, group_size=48), lambda: rms_norm_gated(x, x, w, eps=-1.0),
                lambda: rms_norm_gated(x.cpu(), x.cpu(), w.cpu()), lambda: rms_norm_gated(x.double(), x, w),
                lambda: residual_rms_norm(x, x.half(), w), lambda: residual_rms_norm(x, x[:2], w),
                lambda: residual_rms_norm(x, x, w, eps=float("nan"))):
        with pytest.raises(ValueError):
            bad()
