"""What the delta rule and the block norms refuse before anything is launched, on fake CUDA tensors (no GPU)."""

import itertools

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode


def _mk(*shape, dt=torch.float32):
    return torch.empty(*shape, dtype=dt, device="cuda")


def _rule(b, length, H=2, V=64):
    return [_mk(b, length, 1, 64), _mk(b, length, 1, 64), _mk(b, length, H, V), _mk(b, length, H), _mk(b, length, H)]


@pytest.mark.parametrize("stride", [(64 * 64, 64 * 64), (2 * 64 * 64, 64 * 64 + 4), (64 * 64, 2 * 64 * 64)])
def test_step_refuses_states_that_overlap(stride):
    """Blocks of (headdim, dstate) apart from each other along either axis alone, but not along both."""
    from kernels.gated_delta import gated_delta_step
    with FakeTensorMode():
        states = _mk(100 * 64 * 64).as_strided((4, 2, 64, 64), (*stride, 64, 1))
        with pytest.raises(ValueError, match="its own"):
            gated_delta_step(*_rule(2, 1), states)


def test_overlap_against_counting():
    from kernels.gated_delta import _overlap
    seen = set()
    for n, m, s0, s1, size in itertools.product((1, 2, 4), (1, 2, 3), range(1, 14), range(1, 14), (2, 3)):
        cells = [i * s0 + j * s1 + e for i in range(n) for j in range(m) for e in range(size)]
        want = len(set(cells)) < len(cells)
        assert _overlap(n, s0, m, s1, size) == want, (n, m, s0, s1, size)
        seen.add(want)
    assert seen == {True, False}


def test_sizes_past_the_limits_are_value_errors():
    """As every other refusal of the public functions, with the argument named; a limit itself passes the checks."""
    from kernels import _lib
    from kernels.block_norm import residual_rms_norm, rms_norm_gated
    from kernels.gated_delta import gated_delta_rule, gated_delta_step
    with FakeTensorMode():
        states = _mk(70000, 2, 64, 64)
        for call, name in ((lambda: gated_delta_rule(*_rule(65536, 1)), "65536 sequences"),
                           (lambda: gated_delta_rule(*_rule(1, 4), cu_seqlens=_mk(65538, dt=torch.int32)), "sequences"),
                           (lambda: gated_delta_rule(*_rule(1, 4, 65536, 8)), "65536 heads"),
                           (lambda: gated_delta_rule(*_rule(1, 2 ** 30 + 1, 1, 8)), "tokens"),
                           (lambda: gated_delta_rule(*_rule(65535, 64 * 257, 1, 8)), "chunks"),
                           (lambda: gated_delta_step(*_rule(65536, 1), states), "65536 rows"),
                           (lambda: gated_delta_step(*_rule(1, 2 ** 20 + 1), states), "tokens"),
                           (lambda: rms_norm_gated(_mk(2, 65536), _mk(2, 65536), _mk(65536), group_size=1), "groups"),
                           (lambda: residual_rms_norm(_mk(2, 2 ** 30 + 8), None, _mk(2 ** 30 + 8)), "channels")):
            with pytest.raises(ValueError, match=name):
                call()
    # the library draws the same lines
    for n, code in ((65535, _lib.lib.delta_fwd_launch(_args(_lib.DeltaFwdArgs, 65535), None)),
                    (65536, _lib.lib.delta_fwd_launch(_args(_lib.DeltaFwdArgs, 65536), None))):
        assert code == (1 if n == 65535 else 2)


def _args(cls, n):
    return cls(batch=n, seqlen=1, nheads=1, headdim=64, dstate=64, ngroups=1, nseq=n, dtype=1, scale=1.0)
