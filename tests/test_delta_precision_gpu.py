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
