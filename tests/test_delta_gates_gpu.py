"""The delta rule's gates away from the everyday: not a number."""

import pytest
import torch

from oracle import delta_oracle as do_
from test_gated_delta_gpu import DEV

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("at", [0, 70, 139])
def test_nan_gate_is_not_a_reset(at, dt):
    """A gate that is no number leaves none: outputs from its token on, the final state, and its own gradient.  The
    chunks before its own and other heads keep theirs."""
    from kernels.gated_delta import gated_delta_rule
    x = [torch.from_numpy(t)[None].to(DEV) for t in do_.make_delta_inputs(140, 1, 2, 64, 64, 3)]
    q, k, v, do = (x[i].to(dt).requires_grad_() for i in (0, 1, 2, 5))
    beta, g = x[4], x[3].clone()
    clean = gated_delta_rule(q, k, v, g, beta)
    g[0, at, 1] = float("nan")
    g.requires_grad_()
    o, fin = gated_delta_rule(q, k, v, g, beta, return_final_states=True)
    dg, = torch.autograd.grad(o, g, do)
    assert torch.isnan(o[0, at:, 1]).all() and torch.isnan(fin[0, 1]).all() and torch.isnan(dg[0, at, 1])
    assert torch.equal(o[0, :at // 64 * 64, 1], clean[0, :at // 64 * 64, 1]) and torch.equal(o[0, :, 0], clean[0, :, 0])
    assert torch.isfinite(dg[0, :, 0]).all() and torch.isfinite(fin[0, 0]).all()
