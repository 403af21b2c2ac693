"""How many digits the delta rule keeps on the tensor cores.

A 16-bit result is to carry its own rounding and nothing beside it that shows: against float64 it may be 2 % further
off (2-norm) than the exact result rounded to its type.  (What the arithmetic adds, operand pairs at 2^-16 of a value
and less, is below 1e-4 of that.)"""

import pytest
import torch

from test_gated_delta_gpu import _case, _rel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("G,H,K,V", [(1, 2, 128, 128), (2, 2, 128, 64), (2, 2, 64, 128), (1, 3, 64, 64)])
def test_16_bit_results_are_off_by_their_rounding_alone(G, H, K, V):
    res = _case([200, 200], G, H, K, V, torch.bfloat16, seed=K + V, states=True)
    for m in ("o", "dq", "dk", "dv"):
        got, want = res[m]
        rounded = _rel(torch.from_numpy(want).to(torch.bfloat16), want)
        assert _rel(got, want) <= 1.02 * rounded, m


@pytest.mark.parametrize("beta,gate,dg,dbeta", [(0.98, -1e-3, 1.0e-2, 1.3e-4), (0.9, -1e-2, 1.3e-3, 7.0e-5)])
def test_gate_gradients_where_all_keys_are_alike(beta, gate, dg, dbeta):
    """They are small differences of large terms there: dg is 1 / 1400 of the terms it sums at beta = 0.98.  A float64
    form with nothing but the operands' pairs in it is off by the given shares of dg and dbeta; the kernels may be by
    three times that, a small part of a gradient.  (That a gradient of zero fails is checked, too.)"""
    def edit(x):
        x[1][:] = x[1][:1]
        x[4][:] = beta
        x[3][:] = gate
    res = _case([130], 1, 2, 128, 64, torch.bfloat16, seed=13, states=False, g_edit=edit)
    for m, share in (("dg", dg), ("dbeta", dbeta)):
        got, want = res[m]
        assert 3 * share < 0.1 and _rel(torch.zeros_like(got), want) > 3 * share
        assert _rel(got, want) <= 3 * share, m
    for m in ("dg", "dbeta"):
        exact = _case([130], 1, 2, 128, 64, torch.bfloat16, seed=13, states=False, g_edit=edit, fp32_products=True)[m]
        assert _rel(*exact) < _rel(*res[m])
