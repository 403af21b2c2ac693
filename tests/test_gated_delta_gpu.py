"""The gated delta rule on the B200 against the float64 token recurrence, at the sizes, types, masks and
strides where a chunked kernel can go wrong.

Tolerances (relative 2-norm), set from the arithmetic: a 16-bit output carries its own rounding (2^-9 bf16, 2^-12
fp16, about 0.6 of it in the 2-norm) and, from the bf16 tensor-core path, the rounding of a few operands of the
same size: 5e-3 for bf16, 1e-3 for fp16.  fp32 outputs -- states, gate gradients, everything in fp32 -- come from
fp32 sums over at most 64 tokens and 128 channels: 1e-5.  dg_t sums up to 32 x 32 pairs of a chunk, each
of the size scale |do| |v|, which may cancel almost wholly (equal keys with beta near one: what one token writes the
next one erases): it may be off by the unit roundoff of the root of their sum of squares, 2^-24 32 scale |do| |v|,
where that is more than 1e-5 of dg."""

import numpy as np
import pytest
import torch

from oracle import delta_oracle as do_

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOL = {torch.bfloat16: 5e-3, torch.float16: 1e-3, torch.float32: 1e-5}


def _rel(a, b):
    a = a.detach().double().cpu().numpy()
    return np.linalg.norm(a - b) / max(np.linalg.norm(b), 1e-30)


def _round(x, dt):
    return torch.from_numpy(x).to(dt).double().numpy()


def _case(lens, G, H, K, V, dt, seed, states, g_edit=None, packed=False, **kw):
    """Runs forward + backward on the GPU and the oracle sequence by sequence; returns {name: (got, want)}."""
    from kernels.gated_delta import gated_delta_rule
    n, scale = len(lens), K ** -0.5
    per = [do_.make_delta_inputs(L, G, H, K, V, seed + i) for i, L in enumerate(lens)]
    if g_edit is not None:
        for x in per:
            g_edit(x)
    r = np.random.default_rng(seed + 99)
    s0 = r.standard_normal((n, H, V, K)).astype(np.float32) * 0.3 if states else None
    d1 = r.standard_normal((n, H, V, K)).astype(np.float32) * 0.1 if states else None
    join = (lambda xs: np.concatenate(xs)[None]) if packed else np.stack
    t = [torch.from_numpy(join([x[i] for x in per])).to(DEV) for i in range(6)]
    q, k, v, do = (t[i].to(dt) for i in (0, 1, 2, 5))
    g, beta = t[3], t[4]
    leaves = [q, k, v, g, beta] + ([torch.from_numpy(s0).to(DEV)] if states else [])
    for x in leaves:
        x.requires_grad_()
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), device=DEV, dtype=torch.int32) if packed else None
    o, fin = gated_delta_rule(q, k, v, g, beta, scale=scale, initial_states=leaves[5] if states else None,
                              return_final_states=True, cu_seqlens=cu, **kw)
    outs, douts = [o], [do]
    if states:
        outs, douts = [o, fin], [do, torch.from_numpy(d1).to(DEV)]
    grads = torch.autograd.grad(outs, leaves, douts)
    torch.cuda.synchronize()
    # the same forward without a graph takes the buffers of inference
    with torch.no_grad():
        o2, fin2 = gated_delta_rule(q, k, v, g, beta, scale=scale, initial_states=leaves[5] if states else None,
                                    return_final_states=True, cu_seqlens=cu, **kw)
    assert torch.equal(o, o2) and torch.equal(fin, fin2)
    want = {m: [] for m in ("o", "final", "dq", "dk", "dv", "dg", "dbeta", "ds0")}
    for i, x in enumerate(per):
        a = [_round(x[0], dt), _round(x[1], dt), _round(x[2], dt), x[3], x[4]]
        f = do_.delta_fwd(*a, scale, None if s0 is None else s0[i])
        b = do_.delta_bwd(*a, scale, _round(x[5], dt), None if s0 is None else s0[i], None if d1 is None else d1[i])
        for m in want:
            want[m].append(f[m] if m in f else b[m])
    got = dict(o=o, final=fin, dq=grads[0], dk=grads[1], dv=grads[2], dg=grads[3], dbeta=grads[4])
    if states:
        got["ds0"] = grads[5]
    res = {}
    for m, x in got.items():
        res[m] = (x, np.stack(want[m]) if m in ("final", "ds0") else join(want[m]))
    res["size"] = scale * np.linalg.norm((do.detach().double().norm(dim=-1) * v.detach().double().norm(dim=-1)).cpu())
    return res


def _hold(res, dt):
    for m, (got, want) in ((m, x) for m, x in res.items() if m != "size"):
        tol = TOL[got.dtype]
        assert got.shape == want.shape, m
        assert torch.isfinite(got).all(), m
        e = _rel(got, want)
        if m == "dg":
            tol = max(tol, 2.0 ** -24 * 32 * res["size"] / max(np.linalg.norm(want), 1e-30))
        assert e <= tol, f"{m}: relative error {e:.2e} > {tol:.0e}"


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("L", [1, 2, 63, 64, 65, 200])
def test_lengths_and_types(L, dt):
    _hold(_case([L, L], 2, 4, 64, 64, dt, seed=L, states=True), dt)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("G,H,K,V", [(1, 1, 128, 128), (1, 3, 128, 64), (2, 8, 64, 128), (3, 3, 128, 8), (2, 2, 64, 120),
                                     (1, 2, 128, 72)])
def test_head_layouts(G, H, K, V, dt):
    _hold(_case([150], G, H, K, V, dt, seed=H * V, states=False), dt)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_packed_sequences(dt):
    """Lengths zero, one, within a chunk, on its edge and past it; the final state of an empty one is its initial one."""
    _hold(_case([1, 0, 64, 65, 3, 0, 130], 2, 4, 128, 64, dt, seed=5, states=True, packed=True), dt)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_gates_at_their_ends(dt):
    """beta = 0 (nothing written), beta = 1, no decay, and full resets (g = -inf and the lowest fp32) inside a chunk."""
    def edit(x):
        x[4][3:9] = 0.0
        x[4][20] = 1.0
        x[3][30:40] = 0.0
        x[3][50, 0] = -np.inf
        x[3][77] = np.finfo(np.float32).min
    res = _case([140], 1, 2, 64, 64, dt, seed=11, states=True, g_edit=edit)
    _hold(res, dt)
    assert (res["dg"][0][0, 77] == 0).all() and (res["dv"][0][0, 3:9] == 0).all()


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_repeated_keys(dt):
    """All keys alike and beta near one: the chunk's triangular system at its worst."""
    def edit(x):
        x[1][:] = x[1][:1]
        x[4][:] = 0.98
        x[3][:] = -1e-3
    _hold(_case([130], 1, 2, 128, 64, dt, seed=13, states=False, g_edit=edit, fp32_products=True), dt)


def test_repeated_keys_on_operand_pairs():
    """The same on the tensor cores.  Their operand pairs hold 2^-17 of a value on average where fp32 holds 2^-24, so the gate
    gradients, differences of sums of up to 32 x 32 (dg) and 64 (dbeta) products of the size scale |do| |v|, may be off
    by 2^-17 of the root of the sum of squares of those products; everything else holds its tolerance."""
    def edit(x):
        x[1][:] = x[1][:1]
        x[4][:] = 0.98
        x[3][:] = -1e-3
    res = _case([130], 1, 2, 128, 64, torch.bfloat16, seed=13, states=False, g_edit=edit)
    for m, terms in (("dg", 32), ("dbeta", 8)):
        got, want = res.pop(m)
        assert np.linalg.norm(got.double().cpu().numpy() - want) <= 2.0 ** -17 * terms * res["size"], m
    _hold(res, torch.bfloat16)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_strided_and_broadcast_inputs(dt):
    """q, k, v sliced out of one fused projection, a broadcast q, gates in 16 bits and transposed."""
    from kernels.gated_delta import gated_delta_rule
    B, L, G, H, K, V = 2, 90, 2, 4, 64, 64
    gen = torch.Generator(device=DEV).manual_seed(3)
    fused = torch.randn(B, L, 2 * G * K + H * V + 8, device=DEV, generator=gen).to(dt)
    k = torch.nn.functional.normalize(fused[..., G * K:2 * G * K].float().reshape(B, L, G, K), dim=-1).to(dt)
    fused[..., G * K:2 * G * K] = k.reshape(B, L, -1)
    q = fused[..., :G * K].unflatten(-1, (G, K))
    k = fused[..., G * K:2 * G * K].unflatten(-1, (G, K))
    v = fused[..., 2 * G * K:2 * G * K + H * V].unflatten(-1, (H, V))
    g = -torch.rand(B, H, L, device=DEV, generator=gen).transpose(1, 2)
    beta = torch.rand(B, L, H, device=DEV, generator=gen).to(torch.bfloat16)
    a = gated_delta_rule(q, k, v, g, beta)
    b = gated_delta_rule(q.contiguous(), k.contiguous(), v.contiguous(), g.contiguous(), beta.float())
    assert torch.equal(a, b)
    qb = q[:, :1].expand(B, L, G, K)
    assert torch.equal(gated_delta_rule(qb, k, v, g, beta), gated_delta_rule(qb.contiguous(), k, v, g, beta))
    # a base that is not 16-byte aligned
    off = torch.empty(B * L * H * V + 1, device=DEV, dtype=dt)[1:].view(B, L, H, V).copy_(v)
    assert torch.equal(gated_delta_rule(q, k, off, g, beta), a)


def test_runs_are_equal_bit_by_bit_and_follow_the_stream():
    from kernels.gated_delta import gated_delta_rule
    x = [torch.from_numpy(t)[None].to(DEV) for t in do_.make_delta_inputs(300, 2, 4, 128, 128, 3)]
    q, k, v, do = (x[i].bfloat16().requires_grad_() for i in (0, 1, 2, 5))
    g, beta = x[3].requires_grad_(), x[4].requires_grad_()

    def run():
        o = gated_delta_rule(q, k, v, g, beta)
        return [o, *torch.autograd.grad(o, [q, k, v, g, beta], do)]

    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_empty_calls():
    from kernels.gated_delta import gated_delta_rule
    mk = lambda *s: torch.empty(*s, device=DEV)  # noqa: E731
    s0 = torch.randn(2, 4, 64, 64, device=DEV)
    o, fin = gated_delta_rule(mk(2, 0, 2, 64), mk(2, 0, 2, 64), mk(2, 0, 4, 64), mk(2, 0, 4), mk(2, 0, 4),
                              initial_states=s0, return_final_states=True)
    assert o.shape == (2, 0, 4, 64) and torch.equal(fin, s0)
    assert gated_delta_rule(mk(0, 5, 2, 64), mk(0, 5, 2, 64), mk(0, 5, 4, 64), mk(0, 5, 4), mk(0, 5, 4)).numel() == 0


# ---- the recurrent step ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,G,H,K,V", [(1, 2, 4, 128, 128), (3, 1, 2, 64, 72), (5, 3, 3, 128, 8), (2, 1, 1, 64, 256)])
def test_step_against_the_oracle(T, G, H, K, V, dt):
    from kernels.gated_delta import gated_delta_step
    B, slots, scale = 5, 9, K ** -0.5
    per = [do_.make_delta_inputs(T, G, H, K, V, 10 + i) for i in range(B)]
    states = np.random.default_rng(0).standard_normal((slots, H, V, K)).astype(np.float32)
    at = [7, 0, -1, 3, slots]  # two idle rows
    t = [torch.from_numpy(np.stack([x[i] for x in per])).to(DEV) for i in range(5)]
    cache = torch.from_numpy(states).to(DEV)
    for itype in (torch.int32, torch.int64):
        cache.copy_(torch.from_numpy(states))
        o = gated_delta_step(t[0].to(dt), t[1].to(dt), t[2].to(dt), t[3], t[4], cache, scale=scale,
                             state_indices=torch.tensor(at, device=DEV, dtype=itype))
        want = states.astype(np.float64).copy()
        for b, x in enumerate(per):
            if not 0 <= at[b] < slots:
                assert (o[b] == 0).all()
                continue
            r = do_.delta_fwd(_round(x[0], dt), _round(x[1], dt), _round(x[2], dt), x[3], x[4], scale, states[at[b]])
            want[at[b]] = r["final"]
            assert _rel(o[b], r["o"]) <= TOL[dt]
        assert _rel(cache, want) <= TOL[torch.float32]
        untouched = [i for i in range(slots) if i not in at]
        assert torch.equal(cache[untouched].cpu(), torch.from_numpy(states[untouched]))


def test_steps_continue_a_prefill():
    """Prefill + steps = one longer prefill, without the token axis and with the cache in order."""
    from kernels.gated_delta import gated_delta_rule, gated_delta_step
    B, L, n, G, H, K, V = 2, 70, 4, 2, 4, 128, 64
    x = [do_.make_delta_inputs(L + n, G, H, K, V, 40 + i) for i in range(B)]
    q, k, v, g, beta = (torch.from_numpy(np.stack([y[i] for y in x])).to(DEV) for i in range(5))
    whole, fin = gated_delta_rule(q, k, v, g, beta, return_final_states=True)
    _, st = gated_delta_rule(q[:, :L], k[:, :L], v[:, :L], g[:, :L], beta[:, :L], return_final_states=True)
    for t in range(L, L + n):
        o = gated_delta_step(q[:, t], k[:, t], v[:, t], g[:, t], beta[:, t], st)
        assert o.shape == (B, H, V)
        assert _rel(o, whole[:, t].double().cpu().numpy()) <= TOL[torch.float32]
    assert _rel(st, fin.double().cpu().numpy()) <= TOL[torch.float32]


def test_step_on_strided_cache_and_graph():
    from kernels.gated_delta import gated_delta_step
    B, H, K, V = 3, 2, 64, 64
    x = [do_.make_delta_inputs(1, H, H, K, V, i) for i in range(B)]
    q, k, v, g, beta = (torch.from_numpy(np.stack([y[i] for y in x])).to(DEV) for i in range(5))
    pool = torch.randn(B, 2, H, V, K, device=DEV)  # two layers' caches in one allocation
    keep = pool.clone()
    ref = pool[:, 1].clone()
    want = gated_delta_step(q, k, v, g, beta, ref)
    got = gated_delta_step(q, k, v, g, beta, pool[:, 1])
    assert torch.equal(got, want) and torch.equal(pool[:, 1], ref) and torch.equal(pool[:, 0], keep[:, 0])
    pool.copy_(keep)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = gated_delta_step(q, k, v, g, beta, pool[:, 1])
    torch.cuda.synchronize()
    pool.copy_(keep)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(pool[:, 1], ref)


# ---- refusals -------------------------------------------------------------------------------------------------


def test_refusals():
    from kernels.gated_delta import gated_delta_rule, gated_delta_step

    def args(B=1, L=4, G=2, H=4, K=64, V=64, dt=torch.bfloat16):
        mk = lambda *s: torch.zeros(*s, device=DEV, dtype=dt)  # noqa: E731
        f = lambda *s: torch.zeros(*s, device=DEV)  # noqa: E731
        return [mk(B, L, G, K), mk(B, L, G, K), mk(B, L, H, V), f(B, L, H), f(B, L, H)]

    for kw in (dict(G=3), dict(K=96), dict(V=12), dict(V=136), dict(dt=torch.float64)):
        with pytest.raises(ValueError):
            gated_delta_rule(*args(**kw))
    a = args()
    with pytest.raises(ValueError):
        gated_delta_rule(a[0], a[1].float(), *a[2:])
    with pytest.raises(ValueError):
        gated_delta_rule(*a[:3], a[3][:, :2], a[4])
    with pytest.raises(ValueError):
        gated_delta_rule(*[x.cpu() for x in a])
    with pytest.raises(ValueError):
        gated_delta_rule(*a, initial_states=torch.zeros(2, 4, 64, 64, device=DEV))
    with pytest.raises(ValueError):
        gated_delta_rule(*args(B=2), cu_seqlens=torch.tensor([0, 4], device=DEV))
    with pytest.raises(ValueError):
        gated_delta_rule(*a, cu_seqlens=torch.tensor([0.0, 4.0], device=DEV))
    st = torch.zeros(3, 4, 64, 64, device=DEV)
    with pytest.raises(ValueError):
        gated_delta_step(*a, st.to(torch.bfloat16))
    with pytest.raises(ValueError):
        gated_delta_step(*a, st.transpose(2, 3))
    with pytest.raises(ValueError):
        gated_delta_step(*args(B=4), st)
    with pytest.raises(ValueError):
        gated_delta_step(*a, st, state_indices=torch.zeros(2, device=DEV, dtype=torch.int32))
    a[2].requires_grad_()
    with pytest.raises(ValueError):
        gated_delta_step(*a, st)


def test_device_status_is_clear():
    """No bounded wait of the tensor-core kernels ran out in any of the calls above."""
    import ctypes

    from kernels import _lib
    word = ctypes.c_uint32(0)
    _lib.check(_lib.lib.delta_device_status(ctypes.byref(word), 1, _lib.stream_ptr(torch.device(DEV))), "status")
    assert word.value == 0
