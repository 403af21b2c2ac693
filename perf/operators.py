"""The delta-rule and block-norm operators as measured cases: inputs, plain forms, exact forms and least work.

Operators: the gated delta rule over whole sequences (forward, and forward + backward), its recurrent step on a
state cache, the gated RMS norm behind a block and the residual RMS norm before the next one.  ``own`` chooses
between the plain form (elementary torch operations in 32 bits) and the framework's calls.
"""

import math
import os
import random
import sys

import torch

own = False

CHUNK = 64  # tokens per chunk of the plain delta-rule form
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
DEV = "cuda"


def _framework():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ema-kernels_b200")
    for p in (pkg, os.path.join(os.getcwd(), "ema-kernels_b200")):
        if os.path.isdir(p) and p not in sys.path:
            sys.path.insert(0, p)
    from kernels import block_norm, gated_delta

    return gated_delta, block_norm


# ---- the cases ------------------------------------------------------------------------------------------------


def listed():
    delta = {"op": "delta", "G": 16, "H": 32, "K": 128, "V": 128, "dtype": "bf16", "nseq": 0, "states": False}
    step = {"op": "step", "T": 1, "G": 16, "H": 32, "K": 128, "V": 128, "dtype": "bf16"}
    return [
        # a training step's layer: four full sequences, value heads in pairs on shared query / key heads
        {**delta, "name": "delta_train", "train": True, "B": 4, "L": 4096},
        # fine-tuning on packed documents of uneven lengths, carried states on both ends
        {**delta, "name": "delta_train_packed", "train": True, "B": 1, "L": 6001, "nseq": 9, "G": 8, "H": 8, "V": 64,
         "states": True},
        # a small full-precision run, the sequence no multiple of anything
        {**delta, "name": "delta_train_f32", "train": True, "B": 2, "L": 333, "G": 2, "H": 4, "K": 64, "V": 64,
         "dtype": "f32", "states": True},
        # prefill of one long prompt, continued from a state and into one
        {**delta, "name": "delta_prefill_long", "train": False, "B": 1, "L": 16384, "states": True},
        # a server's prefill batch: many short prompts packed end to end, some of one token
        {**delta, "name": "delta_prefill_packed", "train": False, "B": 1, "L": 8111, "nseq": 40, "G": 4, "H": 16,
         "states": True},
        # one user's decoding: latency
        {**step, "name": "step_one", "B": 1, "slots": 4},
        # a full decoding batch on a larger state cache
        {**step, "name": "step_batch", "B": 256, "slots": 320},
        # a few drafted tokens per row, small value heads
        {**step, "name": "step_draft", "B": 24, "T": 5, "G": 16, "H": 16, "V": 64, "slots": 24, "dtype": "f16"},
        # the norm of every head's output with its gate, training
        {"name": "gated_norm_train", "op": "gated_norm", "train": True, "rows": 8 * 4096 * 32, "D": 128, "group": 128,
         "before": True, "dtype": "bf16"},
        # the gate before a norm over all channels, a decoding batch
        {"name": "gated_norm_decode", "op": "gated_norm", "train": False, "rows": 17, "D": 4096, "group": 4096,
         "before": False, "dtype": "bf16"},
        # residual add and norm before the next block, training, residual stream in 32 bits
        {"name": "residual_norm_train", "op": "residual_norm", "train": True, "rows": 8 * 4096, "D": 2048,
         "dtype": "bf16", "residual": "f32", "scale": 0.7},
        # the same for a decoding batch of an odd width
        {"name": "residual_norm_decode", "op": "residual_norm", "train": False, "rows": 5, "D": 1000, "dtype": "f16",
         "residual": "f16", "scale": 1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["delta_train", "delta_forward", "step", "gated_norm", "residual_norm"])
    if op.startswith("delta"):
        train = op == "delta_train"
        G = rng.choice([1, 2, 3, 4, 8, 16])
        H = G * rng.choice([1, 1, 2, 4])
        H = H if H <= 32 else G
        full = rng.random() < 0.15  # full precision: small runs
        L = _log(rng, 1, 700 if full else 8192 if train else 16384)
        most = max(1, (8 * 700 if full else 4 * 4096 * 32 // 2) // (L * H))
        packed = L > 16 and rng.random() < 0.35
        return {"op": "delta", "train": train, "B": 1 if packed else _log(rng, 1, min(most, 16)), "L": L,
                "nseq": _log(rng, 2, min(48, L // 4)) if packed else 0, "G": G, "H": H, "K": rng.choice([64, 128]),
                "V": rng.choice([64, 128]), "dtype": "f32" if full else "bf16", "states": rng.random() < 0.5}
    if op == "step":
        H = rng.choice([1, 2, 4, 8, 16, 32])
        B = _log(rng, 1, 256)
        return {"op": "step", "B": B, "T": rng.choice([1, 1, 1, 2, 3, 4, 8]), "G": max(1, H // rng.choice([1, 2, 4])),
                "H": H, "K": rng.choice([64, 128]), "V": rng.choice([64, 128]), "slots": B + _log(rng, 1, 64),
                "dtype": rng.choice(["bf16", "f16", "f32"])}
    train = rng.random() < 0.5
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "gated_norm":
        group = rng.choice([64, 96, 128, 256, 1000, 1024, 2048, 4096])
        D = group * rng.choice([1, 1, 2, 8] if group <= 512 else [1])
        rows = _log(rng, 1, 64 * 1024 * 1024 // D)
        return {"op": "gated_norm", "train": train, "rows": rows, "D": D, "group": group,
                "before": rng.random() < 0.5, "dtype": dtype}
    D = rng.choice([64, 777, 1000, 1024, 2048, 2560, 4096, 5120, 8192])
    rows = _log(rng, 1, 64 * 1024 * 1024 // D)
    return {"op": "residual_norm", "train": train, "rows": rows, "D": D, "dtype": dtype,
            "residual": rng.choice(["f32", dtype]), "scale": rng.choice([1.0, 0.7, 0.25])}


def _lengths(case):
    """The packed sequences' lengths: uneven, one of a single token, one empty where there are over eight."""
    n, total = case["nseq"], case["L"]
    r = random.Random(1000 * n + total)
    w = [math.exp(r.gauss(0.0, 1.0)) for _ in range(n)]
    if n > 8:
        w[n // 2] = 0.0
    cut = [0]
    for i in range(n):
        cut.append(min(total, round(total * sum(w[: i + 1]) / sum(w))))
    cut[-1] = total
    got = [b - a for a, b in zip(cut, cut[1:])]
    if n > 8 and got[0] > 1:  # one token alone
        got[1] += got[0] - 1
        got[0] = 1
    return got


# ---- inputs ------------------------------------------------------------------------------------------------------


def _unit(x):
    return x / x.square().sum(-1, keepdim=True).sqrt()


def _delta_inputs(case, seed):
    """Unit keys with a common part, unit queries, and gates as a layer's decay and write-strength maps give them."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 7919 + 17)
    dt = DTYPES[case["dtype"]]
    B, L = case["B"], case.get("L", case.get("T"))
    G, H, K, V = (case[n] for n in "GHKV")

    def rn(*s):
        return torch.randn(*s, device=DEV, generator=g)

    def ru(*s):
        return torch.rand(*s, device=DEV, generator=g)

    common = rn(1, 1, G, K)
    k = _unit(rn(B, L, G, K) + 0.5 * common)
    q = _unit(rn(B, L, G, K) + 0.3 * k)
    v = rn(B, L, H, V)
    rate = torch.exp(ru(H) * math.log(16.0))
    step = torch.exp(math.log(1e-3) + ru(H) * math.log(100.0))
    bias = step + torch.log(-torch.expm1(-step))
    raw = 0.5 * rn(B, L, H) + bias
    decay = -rate * torch.where(raw > 20, raw, torch.log1p(torch.exp(raw)))
    beta = 1 / (1 + torch.exp(-rn(B, L, H)))
    s = {"q": q.to(dt), "k": k.to(dt), "v": v.to(dt), "g": decay, "beta": beta, "scale": K ** -0.5}
    return s, rn


def prepare(case, seed):
    op = case["op"]
    if op == "delta":
        s, rn = _delta_inputs(case, seed)
        dt = DTYPES[case["dtype"]]
        n = case["nseq"] or case["B"]
        H, K, V = case["H"], case["K"], case["V"]
        s.update(op=op, train=case["train"], s0=None, ds1=None, cu=None, longest=case["L"])
        if case["nseq"]:
            lens = _lengths(case)
            s["longest"] = max(lens)
            s["cu"] = torch.tensor([0] + lens, device=DEV, dtype=torch.int64).cumsum(0).to(torch.int32)
        if case["states"]:
            s["s0"] = 0.3 * rn(n, H, V, K)
        if case["train"]:
            s["do"] = rn(case["B"], case["L"], H, V).to(dt)
            if case["states"]:
                s["ds1"] = 0.1 * rn(n, H, V, K)
            for name in ("q", "k", "v", "g", "beta", "s0"):
                if s[name] is not None:
                    s[name].requires_grad_()
        return s
    if op == "step":
        s, rn = _delta_inputs(case, seed)
        s.update(op=op, states=0.3 * rn(case["slots"], case["H"], case["V"], case["K"]))
        at = list(range(case["slots"]))
        random.Random(seed).shuffle(at)
        s["index"] = torch.tensor(at[: case["B"]], device=DEV, dtype=torch.int32)
        return s
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 7919 + 29)
    dt = DTYPES[case["dtype"]]
    rows, D = case["rows"], case["D"]

    def rn(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    s = {"op": op, "train": case["train"], "x": rn(rows, D).to(dt), "weight": 1 + 0.2 * rn(D), "eps": 1e-5}
    if op == "gated_norm":
        s.update(z=rn(rows, D).to(dt), group=case["group"], before=case["before"])
        leaves = ("x", "z", "weight")
    else:
        s.update(residual=(2 * rn(rows, D)).to(DTYPES[case["residual"]]), scale=case["scale"])
        leaves = ("x", "residual", "weight")
        if case["train"]:
            s["dh"] = rn(rows, D).to(DTYPES[case["residual"]])
    if case["train"]:
        s["dy"] = rn(rows, D).to(dt)
        for name in leaves:
            s[name].requires_grad_()
    return s


# ---- plain forms --------------------------------------------------------------------------------------------------


def _unit_lower_inverse(A):
    """(I + A)^-1 of strictly lower triangular A: diagonal blocks joined pairwise, sizes 1, 2, 4, ..."""
    C = A.shape[-1]
    T = torch.ones(*A.shape[:-2], C, 1, 1, device=A.device, dtype=A.dtype)
    s = 1
    while s < C:
        n = C // (2 * s)
        blocks = A.reshape(*A.shape[:-2], n, 2 * s, n, 2 * s).diagonal(dim1=-4, dim2=-2).movedim(-1, -3)
        upper, lower = T[..., 0::2, :, :], T[..., 1::2, :, :]
        joint = -(lower @ (blocks[..., s:, :s] @ upper))
        T = torch.cat([torch.cat([upper, torch.zeros_like(upper)], -1), torch.cat([joint, lower], -1)], -2)
        s *= 2
    return T[..., 0, :, :]


def _plain_delta(q, k, v, g, beta, s0, scale):
    """32-bit chunked form on (n, l, heads, ...) tensors: o and the final state."""
    n, L, H, V = v.shape
    q, k = (t.repeat_interleave(H // t.shape[2], 2) for t in (q, k))
    K = k.shape[-1]
    nc = -(-L // CHUNK)

    def chunks(t):
        t = torch.cat([t, t.new_zeros(n, nc * CHUNK - L, *t.shape[2:])], 1)
        return t.reshape(n, nc, CHUNK, *t.shape[2:]).transpose(2, 3)  # (n, nc, H, C, ...)

    q, k, v, g, beta = (chunks(t) for t in (q, k, v, g, beta))
    b = g.cumsum(-1)
    at = torch.arange(CHUNK, device=v.device)
    low = at[:, None] >= at[None, :]
    gamma = torch.exp(torch.where(low, b[..., :, None] - b[..., None, :], -math.inf))
    kk = (k @ k.transpose(-1, -2)) * gamma
    T = _unit_lower_inverse(torch.where(at[:, None] > at[None, :], kk * beta[..., None, :], 0.0))
    P = scale * (q @ k.transpose(-1, -2)) * gamma
    grow = torch.exp(b)[..., None]
    qs, ks = q * (scale * grow), k * grow
    kend = k * torch.exp(b[..., -1:] - b)[..., None]
    end = torch.exp(b[..., -1])[..., None, None]
    S = s0 if s0 is not None else v.new_zeros(n, H, V, K)
    out = []
    for c in range(nc):
        U = (T[:, c] @ (v[:, c] - ks[:, c] @ S.transpose(-1, -2))) * beta[:, c, :, :, None]
        out.append(qs[:, c] @ S.transpose(-1, -2) + P[:, c] @ U)
        S = end[:, c] * S + U.transpose(-1, -2) @ kend[:, c]
    o = torch.stack(out, 1).transpose(2, 3).reshape(n, nc * CHUNK, H, V)[:, :L]
    return o, S


def _rows_of(cu, longest):
    """Each sequence's rows of the packed tensor, padded to the longest, and which of them are its own."""
    at = cu[:-1, None].long() + torch.arange(longest, device=cu.device)[None, :]
    return at.clamp(max=int(2 ** 31 - 1)), at < cu[1:, None]


def _run_plain_delta(s):
    names = [n for n in ("q", "k", "v", "g", "beta", "s0") if s[n] is not None]
    with torch.set_grad_enabled(s["train"]):
        f = {n: s[n].detach().float().requires_grad_(s["train"]) for n in names}
        args = [f[n] for n in ("q", "k", "v", "g", "beta")]
        if s["cu"] is not None:
            at, mine = _rows_of(s["cu"], s["longest"])
            at = torch.where(mine, at, 0)
            args = [torch.where(mine.reshape(*mine.shape, *[1] * (t.dim() - 2)), t[0][at], 0.0) for t in args]
        o, S = _plain_delta(*args, f.get("s0"), s["scale"])
        if s["cu"] is not None:
            total = s["q"].shape[1]
            seq = torch.searchsorted(s["cu"][1:].long(), torch.arange(total, device=o.device), right=True)
            o = o[seq, torch.arange(total, device=o.device) - s["cu"].long()[seq]][None]
        res = {"o": o.detach().to(s["v"].dtype)}
        if s["s0"] is not None:
            res["final"] = S.detach()
        if s["train"]:
            outs, douts = ([o, S], [s["do"].float(), s["ds1"]]) if s["ds1"] is not None else ([o], [s["do"].float()])
            grads = torch.autograd.grad(outs, [f[n] for n in names], douts)
            res.update({"d" + n: d.to(s[n].dtype) for n, d in zip(names, grads)})
    return res


def _run_plain_step(s):
    dt = s["v"].dtype
    q, k, v, g, beta = (s[n].float() for n in ("q", "k", "v", "g", "beta"))
    H = v.shape[2]
    q, k = (t.repeat_interleave(H // t.shape[2], 2) for t in (q, k))
    at = s["index"].long()
    S = s["states"][at]
    out = []
    for t in range(v.shape[1]):
        S = S * torch.exp(g[:, t])[..., None, None]
        u = beta[:, t, :, None] * (v[:, t] - (S @ k[:, t, :, :, None])[..., 0])
        S = S + u[..., :, None] * k[:, t, :, None, :]
        out.append(s["scale"] * (S @ q[:, t, :, :, None])[..., 0])
    s["states"][at] = S
    return {"o": torch.stack(out, 1).to(dt), "states": s["states"]}


def _run_plain_gated_norm(s):
    with torch.set_grad_enabled(s["train"]):
        f = [s[n].detach().float().requires_grad_(s["train"]) for n in ("x", "z", "weight")]
        x, z, w = f
        gate = z / (1 + torch.exp(-z))
        t = x if s["before"] else x * gate
        t = t.reshape(x.shape[0], -1, s["group"])
        y = (t * torch.rsqrt(t.square().mean(-1, keepdim=True) + s["eps"])).reshape(x.shape) * w
        y = y * gate if s["before"] else y
        res = {"y": y.detach().to(s["x"].dtype)}
        if s["train"]:
            grads = torch.autograd.grad(y, f, s["dy"].float())
            res.update({"d" + n: d.to(s[n].dtype) for n, d in zip(("x", "z", "weight"), grads)})
    return res


def _run_plain_residual_norm(s):
    with torch.set_grad_enabled(s["train"]):
        f = [s[n].detach().float().requires_grad_(s["train"]) for n in ("x", "residual", "weight")]
        x, r, w = f
        h = r + s["scale"] * x
        h = h + (h.detach().to(s["residual"].dtype).float() - h.detach())  # the norm is of h as it is returned
        y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + s["eps"]) * w
        res = {"y": y.detach().to(s["x"].dtype), "h": h.detach().to(s["residual"].dtype)}
        if s["train"]:
            grads = torch.autograd.grad([y, h], f, [s["dy"].float(), s["dh"].float()])
            res.update({"d" + n: d.to(s[n].dtype) for n, d in zip(("x", "residual", "weight"), grads)})
    return res


# ---- the framework's calls --------------------------------------------------------------------------------------


def _run_own(s):
    gated_delta, block_norm = _framework()
    op = s["op"]
    if op == "delta":
        names = [n for n in ("q", "k", "v", "g", "beta", "s0") if s[n] is not None]
        out = gated_delta.gated_delta_rule(s["q"], s["k"], s["v"], s["g"], s["beta"], scale=s["scale"],
                                           initial_states=s["s0"], return_final_states=s["s0"] is not None,
                                           cu_seqlens=s["cu"])
        o, S = out if s["s0"] is not None else (out, None)
        res = {"o": o.detach()}
        if S is not None:
            res["final"] = S.detach()
        if s["train"]:
            outs, douts = ([o, S], [s["do"], s["ds1"]]) if s["ds1"] is not None else ([o], [s["do"]])
            grads = torch.autograd.grad(outs, [s[n] for n in names], douts)
            res.update({"d" + n: d for n, d in zip(names, grads)})
        return res
    if op == "step":
        o = gated_delta.gated_delta_step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["states"], scale=s["scale"],
                                         state_indices=s["index"])
        return {"o": o, "states": s["states"]}
    if op == "gated_norm":
        y = block_norm.rms_norm_gated(s["x"], s["z"], s["weight"], eps=s["eps"], group_size=s["group"],
                                      norm_before_gate=s["before"])
        outs, douts, names = [y], ["dy"], ("x", "z", "weight")
        res = {"y": y.detach()}
    else:
        y, h = block_norm.residual_rms_norm(s["x"], s["residual"], s["weight"], eps=s["eps"], scale=s["scale"])
        outs, douts, names = [y, h], ["dy", "dh"], ("x", "residual", "weight")
        res = {"y": y.detach(), "h": h.detach()}
    if s["train"]:
        grads = torch.autograd.grad(outs, [s[n] for n in names], [s[n] for n in douts])
        res.update({"d" + n: d for n, d in zip(names, grads)})
    return res


def run(state):
    if own:
        return _run_own(state)
    return {"delta": _run_plain_delta, "step": _run_plain_step, "gated_norm": _run_plain_gated_norm,
            "residual_norm": _run_plain_residual_norm}[state["op"]](state)


# ---- least work --------------------------------------------------------------------------------------------------


def work(case):
    es = BYTES[case["dtype"]]
    if case["op"] in ("delta", "step"):
        G, H, K, V = (case[n] for n in "GHKV")
        tokens = case["B"] * case.get("L", case.get("T"))
        qk, vo, gates, state = tokens * G * K * es, tokens * H * V * es, tokens * H * 4, H * V * K * 4
        if case["op"] == "step":
            return {"bytes": 2 * qk + 2 * vo + 2 * gates + 2 * case["B"] * state, "flops": 6 * tokens * H * K * V}
        n = (case["nseq"] or case["B"]) if case["states"] else 0
        w = {"bytes": 2 * qk + 2 * vo + 2 * gates + 2 * n * state, "flops": 6 * tokens * H * K * V}
        if case["train"]:
            w = {"bytes": w["bytes"] + 4 * qk + 3 * vo + 4 * gates + 3 * n * state,
                 "flops": w["flops"] + 16 * tokens * H * K * V}
        return w
    n = case["rows"] * case["D"]
    if case["op"] == "gated_norm":  # x z -> y; and x z dy -> dx dz
        return {"bytes": n * es * (8 if case["train"] else 3) + 4 * case["D"], "flops": n * (30 if case["train"] else 10)}
    rs = BYTES[case["residual"]]  # x r -> y h; and h dy dh -> dx dr
    return {"bytes": n * (2 * es + 2 * rs) + (n * (2 * es + 3 * rs) if case["train"] else 0) + 4 * case["D"],
            "flops": n * (20 if case["train"] else 8)}


# ---- 64 bits -----------------------------------------------------------------------------------------------------


def _exact_delta(q, k, v, g, beta, s0, do, ds1, scale):
    """Token by token in 64 bits, on (n, heads, l, ...); with `do` also the gradients, walking back through the
    tokens with the states recomputed from one kept per 64 tokens."""
    n, H, L, V = v.shape
    K = k.shape[-1]
    a = g.exp()
    S = s0.clone() if s0 is not None else v.new_zeros(n, H, V, K)

    def read(S, r):
        return torch.matmul(S, r.unsqueeze(-1)).squeeze(-1)

    def token(S, t):
        S = S * a[:, :, t, None, None]
        e = v[:, :, t] - read(S, k[:, :, t])
        return S + (beta[:, :, t, None] * e).unsqueeze(-1) * k[:, :, t].unsqueeze(-2), S, e

    o = torch.empty_like(v)
    kept = []
    for t in range(L):
        if do is not None and t % 64 == 0:
            kept.append(S)
        S = token(S, t)[0]
        o[:, :, t] = scale * read(S, q[:, :, t])
    if do is None:
        return o, S, None
    dS = ds1.clone() if ds1 is not None else torch.zeros_like(S)
    dq, dk, dv, dg, db = (torch.zeros_like(t) for t in (q, k, v, g, beta))
    for c in reversed(range(len(kept))):
        after, faded, err, R = [], [], [], kept[c]
        for t in range(64 * c, min(L, 64 * c + 64)):
            R, F, e = token(R, t)
            after.append(R)
            faded.append(F)
            err.append(e)
        for t in reversed(range(64 * c, min(L, 64 * c + 64))):
            St, F, e = after.pop(), faded.pop(), err.pop()
            kt, dot = k[:, :, t], do[:, :, t]
            dq[:, :, t] = scale * read(St.transpose(-1, -2), dot)
            dS = dS + (scale * dot).unsqueeze(-1) * q[:, :, t].unsqueeze(-2)
            du = read(dS, kt)
            de = beta[:, :, t, None] * du
            db[:, :, t] = (du * e).sum(-1)
            dv[:, :, t] = de
            dk[:, :, t] = read(dS.transpose(-1, -2), beta[:, :, t, None] * e) - read(F.transpose(-1, -2), de)
            dF = dS - de.unsqueeze(-1) * kt.unsqueeze(-2)
            dg[:, :, t] = (dF * F).sum((-1, -2))
            dS = a[:, :, t, None, None] * dF
    return o, S, {"q": dq, "k": dk, "v": dv, "g": dg, "beta": db, "s0": dS}


def _exact_run_delta(case, s):
    H, G = case["H"], case["G"]

    def wide(t):
        return t.detach().double()

    names = ("q", "k", "v", "g", "beta")
    full = {n: wide(s[n]) for n in names}
    do = wide(s["do"]) if case["train"] else None
    lens = _lengths(case) if case["nseq"] else [case["L"]] * case["B"]
    n, longest = len(lens), max(lens)

    def rows(t):  # (n, heads, longest, ...): each sequence from its own start, zeros behind it
        t = t.reshape(-1, *t.shape[2:])
        got, at = t.new_zeros(n, longest, *t.shape[1:]), 0
        for i, m in enumerate(lens):
            got[i, :m] = t[at: at + m]
            at += m
        return got.transpose(1, 2)

    def back(t, like):
        t = t.transpose(1, 2)
        return torch.cat([t[i, :m] for i, m in enumerate(lens)]).reshape(like.shape)

    own_head = torch.arange(H, device=DEV) // (H // G)
    args = {m: rows(full[m]) for m in names}
    args["q"], args["k"] = args["q"][:, own_head], args["k"][:, own_head]
    s0 = wide(s["s0"]) if s["s0"] is not None else None
    ds1 = wide(s["ds1"]) if s["ds1"] is not None else None
    o, S, d = _exact_delta(*(args[m] for m in names), s0, rows(do) if do is not None else None, ds1, s["scale"])
    res = {"o": back(o, s["v"])}
    if s0 is not None:
        res["final"] = S
    if d is not None:
        for m in ("q", "k"):
            d[m] = d[m].reshape(n, G, H // G, longest, -1).sum(2)
        res.update({"d" + m: back(d[m], s[m]) for m in names})
        if s0 is not None:
            res["ds0"] = d["s0"]
    return res


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op == "delta":
            return _exact_run_delta(case, s)
        if op == "step":
            q, k, v, g, beta = (s[n].double().transpose(1, 2) for n in ("q", "k", "v", "g", "beta"))
            own_head = torch.arange(case["H"], device=DEV) // (case["H"] // case["G"])
            at = s["index"].long()
            states = s["states"].double()
            o, S, _ = _exact_delta(q[:, own_head], k[:, own_head], v, g, beta, states[at], None, None, s["scale"])
            states[at] = S
            return {"o": o.transpose(1, 2), "states": states}
        x, w = s["x"].double(), s["weight"].double()
        rows, D = x.shape
        if op == "gated_norm":
            z = s["z"].double()
            sig = torch.sigmoid(z)
            gate, dgate = z * sig, sig * (1 + z * (1 - sig))
            m = case["group"]
            t = (x if s["before"] else x * gate).reshape(rows, D // m, m)
            rstd = (t.pow(2).sum(-1, keepdim=True) / m + s["eps"]).pow(-0.5)
            hat = (t * rstd).reshape(rows, D)
            res = {"y": hat * w * gate if s["before"] else hat * w}
            if case["train"]:
                dy = s["dy"].double()
                dn = dy * gate if s["before"] else dy
                dhat = (dn * w).reshape(rows, D // m, m)
                ht = hat.reshape(rows, D // m, m)
                dt = (rstd * (dhat - ht * (dhat * ht).sum(-1, keepdim=True) / m)).reshape(rows, D)
                if s["before"]:
                    res.update(dx=dt, dz=dy * hat * w * dgate)
                else:
                    res.update(dx=dt * gate, dz=dt * x * dgate)
                res["dweight"] = (dn * hat).sum(0)
            return res
        h = (s["residual"].double() + s["scale"] * x).to(s["residual"].dtype).double()
        rstd = (h.pow(2).sum(-1, keepdim=True) / D + s["eps"]).pow(-0.5)
        hat = h * rstd
        res = {"y": hat * w, "h": s["residual"].double() + s["scale"] * x}
        if case["train"]:
            dy = s["dy"].double()
            dhat = dy * w
            dh = s["dh"].double() + rstd * (dhat - hat * (dhat * hat).sum(-1, keepdim=True) / D)
            res.update(dx=s["scale"] * dh, dresidual=dh, dweight=(dy * hat).sum(0))
        return res
