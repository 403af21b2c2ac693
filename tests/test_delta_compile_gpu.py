"""The delta rule and the block norms under torch.compile on the GPU: one graph (fullgraph=True, the aot_eager backend:
the library's kernels are its operators), results equal to those of eager calls bit by bit."""

import numpy as np
import pytest
import torch

from oracle import delta_oracle as do_

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _inputs(B, L, G=2, H=4, K=64, V=64, dt=torch.bfloat16, seed=0):
    per = [do_.make_delta_inputs(L, G, H, K, V, seed + i) for i in range(B)]
    t = [torch.from_numpy(np.stack([x[i] for x in per])).to(DEV) for i in range(6)]
    return [t[0].to(dt), t[1].to(dt), t[2].to(dt), t[3], t[4]], t[5].to(dt)


def _compiled(fn):
    torch._dynamo.reset()
    return torch.compile(fn, backend="aot_eager", fullgraph=True)


@pytest.mark.parametrize("axis", [True, False])
def test_compiled_step(axis):
    from kernels.gated_delta import gated_delta_step
    args, _ = _inputs(3, 1)
    args = args if axis else [t[:, 0] for t in args]
    states = torch.randn(5, 4, 64, 64, device=DEV)
    at = torch.tensor([4, 9, 0], device=DEV)
    ref, got = states.clone(), states.clone()
    fn = lambda *a: gated_delta_step(*a[:-1], state_indices=a[-1])  # noqa: E731
    want = fn(*args, ref, at)
    o = _compiled(fn)(*args, got, at)
    assert torch.equal(o, want) and torch.equal(got, ref) and not torch.equal(got, states)


def test_step_refuses_states_off_16_bytes():
    from kernels.gated_delta import gated_delta_step
    args, _ = _inputs(2, 1)
    off = torch.zeros(2 * 4 * 64 * 64 + 1, device=DEV)[1:].view(2, 4, 64, 64)
    with pytest.raises(ValueError):
        gated_delta_step(*args, off)
    with pytest.raises(ValueError):
        _compiled(lambda *a: gated_delta_step(*a))(*args, off)


def test_compiled_norms():
    from kernels.block_norm import residual_rms_norm, rms_norm_gated

    def fn(x, z, h, w):
        y, h = residual_rms_norm(x, h, w, scale=0.7)
        return rms_norm_gated(y, z, w, group_size=64), h

    leaves = [torch.randn(9, 128, device=DEV) for _ in range(3)] + [torch.ones(128, device=DEV)]
    leaves[:2] = [t.bfloat16() for t in leaves[:2]]
    runs = []
    for f in (fn, _compiled(fn)):
        xs = [t.clone().requires_grad_() for t in leaves]
        y, h = f(*xs)
        runs.append([y, h, *torch.autograd.grad([y, h], xs, [torch.ones_like(y), torch.ones_like(h)])])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("packed", [False, True])
def test_compiled_rule_trains_at_any_length(packed, dt):
    """Forward, gradients and states; one compilation serves the lengths."""
    from kernels.gated_delta import gated_delta_rule

    def fn(q, k, v, g, beta, s0, cu):
        return gated_delta_rule(q, k, v, g, beta, initial_states=s0, return_final_states=True,
                                cu_seqlens=cu if packed else None)

    compiled = _compiled(fn)
    s0 = torch.randn(2, 4, 64, 64, device=DEV)
    for L in (70, 131, 200):
        args, do = _inputs(1 if packed else 2, L, dt=dt, seed=L)
        for t in (*args, do):
            torch._dynamo.mark_dynamic(t, 1)
        cu = torch.tensor([0, 9, 70], device=DEV)
        runs = []
        for f in (fn, compiled):
            xs = [t.detach().clone().requires_grad_() for t in (*args, s0)]
            for t in xs[:5]:
                torch._dynamo.mark_dynamic(t, 1)
            o, fin = f(*xs, cu)
            runs.append([o, fin, *torch.autograd.grad([o, fin], xs, [do, torch.ones_like(fin)])])
        assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("want", [False, True])
def test_compiled_prefill(want):
    from kernels.gated_delta import gated_delta_rule
    args, _ = _inputs(2, 150)
    fn = lambda *a: gated_delta_rule(*a, return_final_states=want)  # noqa: E731
    a, b = fn(*args), _compiled(fn)(*args)
    a, b = (a, b) if want else ([a], [b])
    assert len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_opcheck_operators():
    import kernels.block_norm  # noqa: F401
    import kernels.gated_delta  # noqa: F401
    args, _ = _inputs(2, 70)
    xs = [t.clone().requires_grad_() for t in args]
    torch.library.opcheck(torch.ops.ema_b200.delta_fwd, (*xs, None, None, 1.0, 0),
                          test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))
    torch.library.opcheck(torch.ops.ema_b200.delta_infer, (*args, None, None, 1.0, 0, True))
    one, _ = _inputs(2, 1)
    torch.library.opcheck(torch.ops.ema_b200.delta_step, (*one, torch.randn(3, 4, 64, 64, device=DEV), None, 1.0))
    x, z, w = (torch.randn(*s, device=DEV).requires_grad_() for s in ((5, 64), (5, 64), (64,)))
    torch.library.opcheck(torch.ops.ema_b200.gated_norm_fwd, (x, z, w, 1e-5, 32, True))
    torch.library.opcheck(torch.ops.ema_b200.residual_norm_fwd, (x, z, w, 1e-5, 0.7))
