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
