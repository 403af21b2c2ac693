"""The delta rule's gates away from the everyday: not a number, many resets in a chunk, steep decays among flat ones.
Tolerances as in test_gated_delta_gpu."""

import numpy as np
import pytest
import torch

from oracle import delta_oracle as do_
from test_gated_delta_gpu import DEV, _case, _hold

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


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gate", [-np.inf, -90.0])
@pytest.mark.parametrize("every", [4, 8, 16])
def test_many_resets_and_steep_decays_in_a_chunk(every, gate, dt):
    """The decays between two steep gates are as good as without them: they are no differences of what the steep ones
    have summed to."""
    def edit(x):
        x[3][every // 2::every] = gate
    _hold(_case([140], 1, 2, 64, 64, dt, seed=17 + every, states=True, g_edit=edit), dt)
