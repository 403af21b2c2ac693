"""The float64 delta-rule and norm oracles against central differences and against closed forms (CPU)."""

import numpy as np
import pytest

from oracle import delta_oracle as do_

STEP = 1e-5
# central differences in float64: truncation ~ STEP^2 times a third derivative of order 1e3 here, rounding ~ 1e-16 / STEP
# times a loss of order 10: both below 1e-6 of the gradients' norm
DIFF_REL = 1e-6


def _diff(f, x):
    g = np.zeros_like(x)
    for i in np.ndindex(x.shape):
        keep = x[i]
        x[i] = keep + STEP
        up = f()
        x[i] = keep - STEP
        down = f()
        x[i] = keep
        g[i] = (up - down) / (2 * STEP)
    return g


def _rel(a, b):
    return np.linalg.norm(a - b) / max(np.linalg.norm(b), 1e-300)


@pytest.mark.parametrize("G,H", [(1, 1), (1, 2), (2, 4)])
def test_delta_gradients_against_differences(G, H):
    L, K, V, scale = 5, 4, 3, 0.5
    q, k, v, g, beta, do = (x.astype(np.float64) for x in do_.make_delta_inputs(L, G, H, K, V, seed=H))
    r = np.random.default_rng(1)
    s0, d1 = r.standard_normal((H, V, K)), r.standard_normal((H, V, K))

    def loss():
        x = do_.delta_fwd(q, k, v, g, beta, scale, s0)
        return (x["o"] * do).sum() + (x["final"] * d1).sum()

    d = do_.delta_bwd(q, k, v, g, beta, scale, do, s0, d1)
    for name, x in (("dq", q), ("dk", k), ("dv", v), ("dg", g), ("dbeta", beta), ("ds0", s0)):
        assert _rel(d[name], _diff(loss, x)) < DIFF_REL, name


def test_delta_overwrites_what_a_repeated_key_held():
    """beta = 1 without decay: writing a unit key twice leaves the second value alone (the delta rule)."""
    K, V = 4, 3
    k = np.zeros((2, 1, K))
    k[:, 0, 1] = 1.0
    v = np.random.default_rng(0).standard_normal((2, 1, V))
    r = do_.delta_fwd(k, k, v, np.zeros((2, 1)), np.ones((2, 1)), 1.0)
    assert np.allclose(r["final"][0][:, 1], v[1, 0]) and np.allclose(r["o"][1, 0], v[1, 0])


@pytest.mark.parametrize("before", [True, False])
def test_gated_norm_gradients_against_differences(before):
    r = np.random.default_rng(3)
    x, z, dy = (r.standard_normal((2, 6)) for _ in range(3))
    w = r.standard_normal(6)
    d = do_.gated_norm(x, z, w, 1e-5, 3, before, dy)
    f = lambda: (do_.gated_norm(x, z, w, 1e-5, 3, before)["y"] * dy).sum()  # noqa: E731
    for name, t in (("dx", x), ("dz", z), ("dw", w)):
        assert _rel(d[name], _diff(f, t)) < DIFF_REL, name


def test_residual_norm_gradients_against_differences():
    r = np.random.default_rng(4)
    x, res, dy, dh = (r.standard_normal((2, 5)) for _ in range(4))
    w = r.standard_normal(5)
    d = do_.residual_norm(x, res, w, 1e-5, 0.7, dy=dy, dh=dh)

    def f():
        y = do_.residual_norm(x, res, w, 1e-5, 0.7)
        return (y["y"] * dy).sum() + (y["h"] * dh).sum()

    for name, t in (("dx", x), ("dh_total", res), ("dw", w)):
        assert _rel(d[name], _diff(f, t)) < DIFF_REL, name
