"""The public functions of the delta rule and the block norms under torch.compile, without a GPU: each traces in one
graph on fake CUDA tensors and reaches its dispatcher operator."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.symbolic_shapes import ShapeEnv


def _trace(fn, make, dynamic=None):
    """The operators of this library in fn's graph, and its outputs; ``dynamic``: an axis of every tensor."""
    torch._dynamo.reset()
    ops = []

    def backend(gm, _):
        ops.extend(str(n.target) for n in gm.graph.nodes if n.op == "call_function" and "ema_b200" in str(n.target))
        return gm.forward

    with FakeTensorMode(shape_env=ShapeEnv()):
        args = make(lambda *s, dt=torch.bfloat16: torch.empty(*s, dtype=dt, device="cuda"))
        if dynamic is not None:
            for t in args:
                torch._dynamo.mark_dynamic(t, dynamic)
        out = torch.compile(fn, backend=backend, fullgraph=True)(*args)
    return ops, out


def _rule(mk, b=2, length=70):
    f = lambda *s: mk(*s, dt=torch.float32)  # noqa: E731
    return [mk(b, length, 2, 64), mk(b, length, 2, 64), mk(b, length, 4, 64), f(b, length, 4), f(b, length, 4)]


@pytest.mark.parametrize("dynamic", [None, 0])
@pytest.mark.parametrize("itype", [None, torch.int32, torch.int64])
def test_step_traces(itype, dynamic):
    from kernels.gated_delta import gated_delta_step

    def make(mk):
        more = [] if itype is None else [mk(2, dt=itype)]
        return _rule(mk, length=1) + [mk(5, 4, 64, 64, dt=torch.float32)] + more

    ops, o = _trace(lambda q, k, v, g, b, s, i=None: gated_delta_step(q, k, v, g, b, s, state_indices=i), make, dynamic)
    assert len(ops) == 1 and "delta_step" in ops[0] and o.shape[1:] == (1, 4, 64)


def test_step_without_a_token_axis_traces():
    from kernels.gated_delta import gated_delta_step
    make = lambda mk: [t[:, 0] for t in _rule(mk, length=1)] + [mk(2, 4, 64, 64, dt=torch.float32)]  # noqa: E731
    ops, o = _trace(lambda *a: gated_delta_step(*a), make)
    assert len(ops) == 1 and o.shape == (2, 4, 64)


@pytest.mark.parametrize("dynamic", [None, 0])
def test_norms_trace(dynamic):
    from kernels.block_norm import residual_rms_norm, rms_norm_gated
    make = lambda mk: [mk(6, 64), mk(6, 64)]  # noqa: E731

    def fn(x, z):
        w = torch.ones(64, device="cuda")
        return rms_norm_gated(x, z, w, group_size=32), *residual_rms_norm(x, z, w, scale=0.7)

    ops, out = _trace(fn, make, dynamic)
    assert len(ops) == 2 and all(t.shape[1:] == (64,) for t in out)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_rule_traces_with_a_length_of_any_size(packed, dt):
    """A length marked dynamic stays a symbol (marking it fails where the code makes a constant of it)."""
    from kernels.gated_delta import gated_delta_rule

    def make(mk):
        a = _rule(mk, 1 if packed else 2, 70)
        return [t.to(dt).requires_grad_() for t in a[:3]] + a[3:]

    def fn(*a):
        cu = torch.tensor([0, 9, 64], device="cuda") if packed else None
        return gated_delta_rule(*a, return_final_states=True, cu_seqlens=cu)

    ops, (o, fin) = _trace(fn, make, dynamic=1)
    assert len(ops) == 1 and o.shape[2:] == (4, 64) and fin.shape == (2, 4, 64, 64)


@pytest.mark.parametrize("want", [False, True])
def test_traced_inference_keeps_nothing_for_a_backward(want):
    """147 KB a chunk and head otherwise, of a call that has no backward."""
    from kernels.gated_delta import gated_delta_rule
    fn = lambda *a: gated_delta_rule(*a, return_final_states=want)  # noqa: E731
    ops, out = _trace(fn, _rule, dynamic=1)
    assert len(ops) == 1 and "delta_infer" in ops[0]
    if want:
        assert out[1].shape == (2, 4, 64, 64)

    def leaf(mk):
        a = _rule(mk)
        a[3].requires_grad_()
        return a

    assert "delta_fwd" in _trace(fn, leaf)[0][0]
    with torch.no_grad():
        assert "delta_infer" in _trace(fn, leaf)[0][0]


def test_bytes_kept_cover_what_the_library_needs():
    """Python's number of bytes against the library's for the same chunk slots, and what it may exceed them by."""
    from kernels import _lib
    from kernels.gated_delta import _saved_bytes
    for code in (0, 1, 2):
        for H, V, K in ((1, 8, 64), (3, 72, 128), (4, 128, 128)):
            for L in (1, 64, 65, 130, 4096):
                got = _saved_bytes(2, L, 2, False, H, V, K, code, 0)
                need = _lib.lib.delta_saved_bytes(2, L, 2, H, V, K, 1, code, 0)
                assert need <= got <= 1.02 * need + 2048
                for n in (1, 2, 9):
                    got = _saved_bytes(1, L, n, True, H, V, K, code, 0)
                    need = _lib.lib.delta_saved_bytes(1, L, n, H, V, K, 1, code, 0)
                    assert need <= got <= 1.02 * need + 2048
