"""gated_delta_step writes its cache in place: what autograd is told of it."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("whole", [True, False])
def test_a_step_counts_as_a_write_to_its_states(whole):
    """A gradient that saved the states before the step refuses, as after any write in place, also through a view."""
    from kernels.gated_delta import gated_delta_step
    q, v, g = torch.ones(2, 1, 2, 64, device=DEV), torch.ones(2, 1, 2, 64, device=DEV), -torch.ones(2, 1, 2, device=DEV)
    pool = torch.randn(3, 2, 2, 64, 64, device=DEV)
    cache = torch.randn(2, 2, 64, 64, device=DEV) if whole else pool[1]
    w = torch.ones(1, device=DEV, requires_grad=True)
    y = ((cache if whole else pool) * w).sum()
    before = cache._version
    gated_delta_step(q, q, v, g, g, cache)
    assert cache._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        gated_delta_step(q, q, v, g, g, torch.zeros(2, 2, 64, 64, device=DEV))
