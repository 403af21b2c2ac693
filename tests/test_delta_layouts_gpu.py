"""The delta rule on layouts and calls beside the plain ones: views with heads before tokens, packed calls whose
sequences leave tokens out, more chunks than blocks, indices of 64 bits."""

import numpy as np
import pytest
import torch

from oracle import delta_oracle as do_
from test_gated_delta_gpu import DEV, _case, _hold

pytestmark = pytest.mark.gpu


def _inputs(L, G, H, K, V, dt, B=1, seed=0):
    per = [do_.make_delta_inputs(L, G, H, K, V, seed + i) for i in range(B)]
    t = [torch.from_numpy(np.stack([x[i] for x in per])).to(DEV) for i in range(6)]
    return [t[0].to(dt), t[1].to(dt), t[2].to(dt), t[3], t[4]], t[5].to(dt)


def _run(args, do, **kw):
    from kernels.gated_delta import gated_delta_rule
    args = [t.detach().requires_grad_() for t in args]
    o = gated_delta_rule(*args, **kw)
    return [o, *torch.autograd.grad(o, args, do)]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [64, 72, 128])
def test_heads_before_tokens(V, dt):
    """q, k, v, do (batch, heads, tokens, channels) turned into place, and tokens before the batch."""
    args, do = _inputs(130, 2, 4, 64, V, dt, B=2, seed=1)
    want = _run(args, do)
    for a, b in ((1, 2), (0, 1)):
        turned = [t.transpose(a, b).contiguous().transpose(a, b) for t in (*args, do)]
        assert not turned[2].is_contiguous()
        for got, ref in zip(_run(turned[:5], turned[5]), want):
            assert torch.equal(got, ref)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
def test_tokens_outside_every_sequence(itype, dt):
    """Zeros in o and every gradient, whatever stands there; the sequences' own results do not see it."""
    args, do = _inputs(150, 2, 4, 128, 64, dt, seed=2)
    cu = torch.tensor([5, 70, 70, 131], device=DEV, dtype=itype)
    want = _run(args, do, cu_seqlens=cu)
    out = torch.ones(150, dtype=torch.bool, device=DEV)
    out[5:131] = False
    spoilt = [t.clone() for t in (*args, do)]
    for t in spoilt:
        t[:, out] = float("nan")
    for got, ref in zip(_run(spoilt[:5], spoilt[5], cu_seqlens=cu), want):
        assert torch.equal(got, ref) and (got[:, out] == 0).all()
    alone = _run([t[:, 5:70] for t in args], do[:, 5:70])
    for got, ref in zip(want, alone):
        assert torch.equal(got[:, 5:70], ref)


def test_offsets_of_64_bits_are_clamped_not_cut():
    """Past 32 bits an offset means the call's end, as it does below them."""
    args, do = _inputs(100, 1, 2, 64, 64, torch.bfloat16, seed=3)
    a = _run(args, do, cu_seqlens=torch.tensor([-2 ** 40, 30, 2 ** 32], device=DEV))
    b = _run(args, do, cu_seqlens=torch.tensor([0, 30, 100], device=DEV))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("G,H,K,V", [(16, 16, 128, 128), (16, 48, 64, 64)])
def test_more_chunks_than_blocks(G, H, K, V):
    """Several (chunk, group) tasks for each block of the persistent gradient kernel."""
    _hold(_case([190] * 9, G, H, K, V, torch.bfloat16, seed=4, states=True), torch.bfloat16)


def test_more_chunks_than_blocks_packed():
    """The same with empty chunk slots between them."""
    lens = [0, 130, 1, 0, 0, 64, 190, 65, 0, 7, 128, 3, 190, 0, 170]
    _hold(_case(lens, 32, 32, 64, 64, torch.bfloat16, seed=5, states=True, packed=True), torch.bfloat16)
