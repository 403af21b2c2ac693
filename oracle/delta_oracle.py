"""float64 restatement of the gated delta rule and of the norms around a block (numpy), token by token.

    S_t = a_t S_{t-1} + beta_t (v_t - a_t S_{t-1} k_t) k_t^T,  a_t = exp(g_t),  o_t = scale S_t q_t

Unpinned: the reference has neither operator.  The gradients below are the recurrence's own, walked back
token by token; the tests check them against central differences of the forward.
"""

from __future__ import annotations

import numpy as np


def _expand(x, H):
    return np.repeat(x, H // x.shape[-2], axis=-2)


def delta_fwd(q, k, v, g, beta, scale, s0=None):
    """One sequence: q, k (L, G, K), v (L, H, V), g, beta (L, H), s0 (H, V, K).
    Returns dict(o, final, states (L, H, V, K), faded (L, H, V, K), err (L, H, V))."""
    L, H, V = v.shape
    q, k = _expand(q.astype(np.float64), H), _expand(k.astype(np.float64), H)
    K = k.shape[-1]
    S = np.zeros((H, V, K)) if s0 is None else s0.astype(np.float64)
    o = np.zeros((L, H, V))
    states, faded, err = np.zeros((L, H, V, K)), np.zeros((L, H, V, K)), np.zeros((L, H, V))
    for t in range(L):
        F = np.exp(g[t].astype(np.float64))[:, None, None] * S
        e = v[t] - np.einsum("hvk,hk->hv", F, k[t])
        S = F + (beta[t][:, None] * e)[..., None] * k[t][:, None, :]
        o[t] = scale * np.einsum("hvk,hk->hv", S, q[t])
        states[t], faded[t], err[t] = S, F, e
    return dict(o=o, final=S, states=states, faded=faded, err=err)


def delta_bwd(q, k, v, g, beta, scale, do, s0=None, d_final=None):
    """Gradients of one sequence: dict(dq, dk, dv, dg, dbeta, ds0); dq, dk summed over a group's heads."""
    L, H, V = v.shape
    G, K = q.shape[1], q.shape[2]
    r = delta_fwd(q, k, v, g, beta, scale, s0)
    qe, ke = _expand(q.astype(np.float64), H), _expand(k.astype(np.float64), H)
    dS = np.zeros((H, V, K)) if d_final is None else d_final.astype(np.float64)
    dq, dk, dv = np.zeros((L, H, K)), np.zeros((L, H, K)), np.zeros((L, H, V))
    dg, dbeta = np.zeros((L, H)), np.zeros((L, H))
    for t in reversed(range(L)):
        S, F, e = r["states"][t], r["faded"][t], r["err"][t]
        dS = dS + scale * do[t][..., None] * qe[t][:, None, :]
        dq[t] = scale * np.einsum("hvk,hv->hk", S, do[t])
        du = np.einsum("hvk,hk->hv", dS, ke[t])
        de = beta[t][:, None] * du
        dbeta[t] = (du * e).sum(-1)
        dv[t] = de
        dk[t] = np.einsum("hvk,hv->hk", dS, beta[t][:, None] * e) - np.einsum("hvk,hv->hk", F, de)
        dF = dS - de[..., None] * ke[t][:, None, :]
        dg[t] = (dF * F).sum((-1, -2))
        dS = np.exp(g[t].astype(np.float64))[:, None, None] * dF
    grp = lambda x: x.reshape(L, G, H // G, K).sum(2)  # noqa: E731
    return dict(dq=grp(dq), dk=grp(dk), dv=dv, dg=dg, dbeta=dbeta, ds0=dS)


def make_delta_inputs(L, G, H, K, V, seed):
    """Unit keys with a common part and gates of a trained layer's range, float32 numpy."""
    r = np.random.default_rng(seed)
    unit = lambda x: x / np.linalg.norm(x, axis=-1, keepdims=True)  # noqa: E731
    k = unit(r.standard_normal((L, G, K)) + 0.5 * r.standard_normal((1, G, K)))
    q = unit(r.standard_normal((L, G, K)) + 0.3 * k)
    v = r.standard_normal((L, H, V))
    g = -np.exp(r.uniform(np.log(1e-3), np.log(1.5), (1, H))) * r.uniform(0.2, 2.0, (L, H))
    beta = 1 / (1 + np.exp(-r.standard_normal((L, H))))
    do = r.standard_normal((L, H, V))
    return [x.astype(np.float32) for x in (q, k, v, g, beta, do)]


def _silu(z):
    s = 1 / (1 + np.exp(-z))
    return z * s, s * (1 + z * (1 - s))


def gated_norm(x, z, w, eps, group, before, dy=None):
    """dict(y[, dx, dz, dw]) on (rows, dim) float64."""
    rows, D = x.shape
    gate, dgate = _silu(z)
    t = (x if before else x * gate).reshape(rows, -1, group)
    rstd = ((t ** 2).mean(-1, keepdims=True) + eps) ** -0.5
    th = t * rstd
    hat = th.reshape(rows, D)
    res = dict(y=hat * w * (gate if before else 1.0))
    if dy is not None:
        dn = dy * gate if before else dy
        dh = (dn * w).reshape(t.shape)
        dt = (rstd * (dh - th * (dh * th).mean(-1, keepdims=True))).reshape(rows, D)
        res.update(dx=dt if before else dt * gate, dz=(dy * hat * w if before else dt * x) * dgate,
                   dw=(dn * hat).sum(0))
    return res


def residual_norm(x, r, w, eps, scale, rounded=None, dy=None, dh=None):
    """dict(h, y[, dh_total, dx, dw]); ``rounded``: h as the framework returned it (its norm is y)."""
    h = scale * x + (0.0 if r is None else r)
    n = h if rounded is None else rounded
    rstd = ((n ** 2).mean(-1, keepdims=True) + eps) ** -0.5
    hat = n * rstd
    res = dict(h=h, y=hat * w)
    if dy is not None:
        dn = dy * w
        tot = (0.0 if dh is None else dh) + rstd * (dn - hat * (dn * hat).mean(-1, keepdims=True))
        res.update(dh_total=tot, dx=scale * tot, dw=(dy * hat).sum(0))
    return res
