"""The block norms where a thread group works on several rows, or on none, against float64; and gates far
from zero in fp32.  Tolerances as in test_block_norm_gpu."""

import pytest
import torch

from oracle import delta_oracle as do_
from test_block_norm_gpu import DEV, _f64, _hold, _rand

pytestmark = pytest.mark.gpu

# one width for each layout: 8, 16, 32 (one and two vectors) and 256 threads (one, two, four; element by element), wide
LAYOUTS = [64, 128, 256, 512, 1000, 4096, 8192, 777, 9000]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", LAYOUTS)
def test_eps_of_zero(D, dt):
    """No row is zero, so every result is finite: a group without a row must add nothing to the weight gradient."""
    from kernels.block_norm import residual_rms_norm, rms_norm_gated
    x, z, dy, w = _rand(D + 7, (5, D), (5, D), (5, D), (D,))
    x, z, dy = x.to(dt).requires_grad_(), z.to(dt).requires_grad_(), dy.to(dt)
    w = (1 + 0.2 * w).requires_grad_()
    for before in (True, False):
        y = rms_norm_gated(x, z, w, eps=0.0, norm_before_gate=before)
        r = do_.gated_norm(_f64(x), _f64(z), _f64(w), 0.0, D, before, _f64(dy))
        for name, got in zip(("y", "dx", "dz", "dw"), (y, *torch.autograd.grad(y, [x, z, w], dy))):
            _hold(name, got, r[name])
    y, h = residual_rms_norm(x, z, w, eps=0.0, scale=0.7)
    e = do_.residual_norm(_f64(x), _f64(z), _f64(w), 0.0, 0.7, _f64(h), _f64(dy))
    for name, got in zip(("y", "dx", "dh_total", "dw"), (y, *torch.autograd.grad(y, [x, z, w], dy))):
        _hold(name, got, e[name])


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,D,group", [(888 * 32 * 3 + 5, 64, 64), (888 * 16 * 3 + 5, 128, 128), (888 * 8 * 3 + 5, 512, 256),
                                          (888 * 8 * 2 + 3, 512, 512), (888 * 4 + 3, 1000, 1000), (888 * 4 + 3, 777, 777),
                                          (888 * 3 + 2, 4096, 4096), (888 * 2 + 5, 8192, 8192), (888 + 3, 9000, 9000)])
def test_several_rows_for_each_thread_group(rows, D, group, dt):
    """More rows than the grid takes at once, and an uneven rest: rows ahead, the sums' turns, dw over a group's rows."""
    from kernels.block_norm import residual_rms_norm, rms_norm_gated
    x, z, dy, w = _rand(D + rows, (rows, D), (rows, D), (rows, D), (D,))
    x, z, dy = x.to(dt).requires_grad_(), z.to(dt).requires_grad_(), dy.to(dt)
    w = (1 + 0.2 * w).requires_grad_()
    y = rms_norm_gated(x, z, w, group_size=group)
    r = do_.gated_norm(_f64(x), _f64(z), _f64(w), 1e-5, group, True, _f64(dy))
    for name, got in zip(("y", "dx", "dz", "dw"), (y, *torch.autograd.grad(y, [x, z, w], dy))):
        _hold(name, got, r[name])
    if group == D:
        y, h = residual_rms_norm(x, z, w, scale=0.7)
        e = do_.residual_norm(_f64(x), _f64(z), _f64(w), 1e-5, 0.7, _f64(h), _f64(dy), _f64(dy))
        for name, got in zip(("y", "dx", "dh_total", "dw"), (y, *torch.autograd.grad([y, h], [x, z, w], [dy, dy]))):
            _hold(name, got, e[name])


@pytest.mark.parametrize("before", [True, False])
def test_fp32_gates_far_from_zero(before):
    """sigmoid(z) down to e^-30 keeps fp32's digits (the norm first: y carries it as a factor).  Each element is a
    chain of some ten roundings and three functions of at most 2 ulp: 16 ulp."""
    from kernels.block_norm import rms_norm_gated
    x, z, w = _rand(11, (64, 128), (64, 128), (128,))
    z = -30 * torch.sigmoid(z) - 1
    x = torch.where(x.abs() < 0.1, torch.ones_like(x), x)
    w = 1 + 0.2 * w.abs()
    want = do_.gated_norm(_f64(x), _f64(z), _f64(w), 1e-30, 128, before)["y"]
    got = _f64(rms_norm_gated(x, z, w, eps=1e-30, norm_before_gate=before))
    rel = abs(got - want) / abs(want)
    assert rel.max() <= 16 * 2.0 ** -24, rel.max()
