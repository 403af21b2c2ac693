"""The delta-rule operators as a model uses them: train on packed sequences, prefill a batch of prompts, decode.

A stack of blocks, each

    y, h = residual_rms_norm(x, h)                         the residual stream h stays fp32
    q, k, v, z, gates = W_in y                             q and k of a group are shared by its heads; k, q normalised
    o = gated_delta_rule(q, k, v, g, beta)                 decoding: gated_delta_step on the block's cache of states
    x = W_out rms_norm_gated(o, z)                         a norm for each head, then the gate silu(z)

is trained to recall: a sequence lists pairs (key, value), then asks for some of the keys again, and only the
answers count.  Then the prompts (of unequal lengths, packed end to end) are prefilled in one call that leaves
each one's states in a cache slot, and the answers are decoded token by token, all rows in one step.

    python ema-kernels_b200/examples/delta_block.py [--steps 400] [--layers 2]
"""

from __future__ import annotations

import argparse
import os
import sys

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from kernels.block_norm import residual_rms_norm, rms_norm_gated  # noqa: E402
from kernels.gated_delta import gated_delta_rule, gated_delta_step  # noqa: E402


class DeltaBlock(nn.Module):
    """norm -> projections -> gated delta rule -> gated norm -> projection, on a bf16 branch and an fp32 stream."""

    def __init__(self, width, nheads, headdim, ngroups, dstate):
        super().__init__()
        self.nheads, self.headdim, self.ngroups, self.dstate = nheads, headdim, ngroups, dstate
        self.sizes = [ngroups * dstate, ngroups * dstate, nheads * headdim, nheads * headdim, 2 * nheads]
        bf = dict(bias=False, dtype=torch.bfloat16)
        self.norm_in = nn.Parameter(torch.ones(width))
        self.norm_out = nn.Parameter(torch.ones(headdim))
        self.w_in = nn.Linear(width, sum(self.sizes), **bf)
        self.w_out = nn.Linear(nheads * headdim, width, **bf)
        # slow decays to begin with, so that a pair is still there when its key is asked for
        self.decay = nn.Parameter(torch.linspace(-6.0, -3.0, nheads))

    def _inputs(self, y):
        """q, k, v, z in the layouts of the rule, the log decay g <= 0 and the write strength beta in (0, 1)."""
        q, k, v, z, gates = self.w_in(y).split(self.sizes, dim=-1)
        lead = y.shape[:-1]
        q, k = (F.normalize(t.view(*lead, self.ngroups, self.dstate), dim=-1).to(torch.bfloat16) for t in (q, k))
        v, z = (t.view(*lead, self.nheads, self.headdim) for t in (v, z))
        a, b = gates.float().view(*lead, 2, self.nheads).unbind(-2)
        return q, k, v, z, -F.softplus(a + self.decay), torch.sigmoid(b)

    def _out(self, o, z):
        weight = self.norm_out.repeat(self.nheads)
        o = rms_norm_gated(o.flatten(-2), z.flatten(-2), weight, group_size=self.headdim)
        return self.w_out(o)

    def forward(self, x, h, cu_seqlens=None, want_states=False):
        y, h = residual_rms_norm(x, h, self.norm_in)
        q, k, v, z, g, beta = self._inputs(y)
        o = gated_delta_rule(q, k, v, g, beta, return_final_states=want_states, cu_seqlens=cu_seqlens)
        o, states = o if want_states else (o, None)
        return self._out(o, z), h, states

    def step(self, x, h, states, slots):
        """One token for each row; states (slots, nheads, headdim, dstate) change in place."""
        y, h = residual_rms_norm(x, h, self.norm_in)
        q, k, v, z, g, beta = self._inputs(y)
        return self._out(gated_delta_step(q, k, v, g, beta, states, state_indices=slots), z), h


class DeltaLM(nn.Module):
    def __init__(self, vocab, width=256, layers=2, nheads=4, headdim=64, ngroups=2, dstate=64):
        super().__init__()
        self.embed = nn.Embedding(vocab, width)
        self.blocks = nn.ModuleList(DeltaBlock(width, nheads, headdim, ngroups, dstate) for _ in range(layers))
        self.norm = nn.Parameter(torch.ones(width))
        self.head = nn.Linear(width, vocab, bias=False, dtype=torch.bfloat16)

    def _embed(self, tokens, before):
        """Each token's embedding plus, turned by one channel, the one before it: a value sees its key."""
        e = self.embed(tokens)
        return e + torch.roll(self.embed(before), 1, dims=-1)

    def _logits(self, x, h):
        y, _ = residual_rms_norm(x, h, self.norm)
        return self.head(y).float()

    def forward(self, tokens, before, cu_seqlens=None, want_states=False):
        h = self._embed(tokens, before)
        x, states = torch.zeros_like(h, dtype=torch.bfloat16), []
        for block in self.blocks:
            x, h, s = block(x, h, cu_seqlens, want_states)
            states.append(s)
        return self._logits(x, h), states

    def step(self, tokens, before, caches, slots):
        h = self._embed(tokens, before)
        x = torch.zeros_like(h, dtype=torch.bfloat16)
        for block, cache in zip(self.blocks, caches):
            x, h = block.step(x, h, cache, slots)
        return self._logits(x, h)


def recall_batch(pairs, asks, vocab, gen):
    """One sequence a count in ``pairs``: k1 v1 ... kn vn, then ``asks`` known keys each followed by its value,
    packed end to end.  Returns tokens, each one's predecessor, cu_seqlens, and the positions of the asked keys."""
    half, seqs, at, cu = vocab // 2, [], [], [0]
    for n in pairs:
        keys = torch.randperm(half - 1, generator=gen)[:n] + 1
        values = torch.randint(half, vocab, (n,), generator=gen)
        pick = torch.randperm(n, generator=gen)[:asks]
        order = torch.cat([torch.arange(n), pick])
        seqs.append(torch.stack([keys[order], values[order]], 1).flatten())
        at.append(cu[-1] + 2 * n + 2 * torch.arange(asks))
        cu.append(cu[-1] + len(seqs[-1]))
    tokens, cu = torch.cat(seqs), torch.tensor(cu)
    before = torch.roll(tokens, 1)
    before[cu[:-1]] = 0
    return tokens, before, cu, torch.stack(at)


def train(model, steps, vocab, gen, device, batch=16, asks=4, most=24, report=None):
    opt = torch.optim.AdamW(model.parameters(), lr=3e-3, weight_decay=0.0)
    losses = []
    for i in range(steps):
        pairs = torch.randint(asks, most + 1, (batch,), generator=gen).tolist()
        tokens, before, cu, at = recall_batch(pairs, asks, vocab, gen)
        tokens, before, at = tokens.to(device), before.to(device), at.to(device).flatten()
        logits, _ = model(tokens[None], before[None], cu.to(device, torch.int32))
        loss = F.cross_entropy(logits[0, at], tokens[at + 1])
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        losses.append(loss.detach())
        if report and (i % 50 == 0 or i + 1 == steps):
            report(f"step {i:4d}  loss {loss.item():.3f}")
    return torch.stack(losses).tolist()


@torch.no_grad()
def recall(model, vocab, gen, device, rows=8, asks=4, most=24):
    """Prefill the lists, decode the questions.  Returns (share answered right, the decoded steps' logits and those
    of one whole call over the same tokens, as (rows, 2 asks, vocab))."""
    pairs = torch.randint(asks, most + 1, (rows,), generator=gen).tolist()
    tokens, before, cu, at = recall_batch(pairs, asks, vocab, gen)
    whole, _ = model(tokens[None].to(device), before[None].to(device), cu.to(device, torch.int32))
    ask = torch.cat([at[:, :1] + j for j in range(2 * asks)], 1)  # every position behind the lists
    listed = torch.ones(len(tokens), dtype=torch.bool)
    listed[ask.flatten()] = False
    cu_list = torch.tensor([0] + pairs).mul(2).cumsum(0).to(device, torch.int32)
    _, states = model(tokens[listed][None].to(device), before[listed][None].to(device), cu_list, want_states=True)
    slots = torch.randperm(rows + 3, generator=gen)[:rows].to(device, torch.int32)
    caches = [s.new_zeros(rows + 3, *s.shape[1:]).index_copy_(0, slots.long(), s) for s in states]
    got = [model.step(tokens[ask[:, j:j + 1]].to(device), before[ask[:, j:j + 1]].to(device), caches, slots)
           for j in range(2 * asks)]
    got, whole = torch.cat(got, 1), whole[0, ask.to(device)]
    right = (got[:, ::2].argmax(-1).cpu() == tokens[ask[:, 1::2]]).float().mean().item()
    return right, got, whole


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=400)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--vocab", type=int, default=128)
    ap.add_argument("--seed", type=int, default=0)
    args = ap.parse_args()
    if not torch.cuda.is_available():
        raise SystemExit("delta_block: needs a CUDA device (B200)")
    torch.manual_seed(args.seed)
    device, gen = torch.device("cuda"), torch.Generator().manual_seed(args.seed)
    model = DeltaLM(args.vocab, layers=args.layers).to(device)
    train(model, args.steps, args.vocab, gen, device, report=print)
    right, got, whole = recall(model, args.vocab, gen, device)
    print(f"decoded answers right: {100 * right:.0f} %   decoding against one whole call: "
          f"{(got - whole).abs().max().item():.3f} of logits up to {whole.abs().max().item():.1f}")


if __name__ == "__main__":
    main()
