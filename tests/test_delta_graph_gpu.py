"""The delta rule and the block norms captured in a CUDA graph: replays on other inputs give what eager calls give."""

import numpy as np
import pytest
import torch

from oracle import delta_oracle as do_

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _inputs(L, dt, seed):
    per = do_.make_delta_inputs(L, 2, 4, 64, 64, seed)
    return [torch.from_numpy(np.ascontiguousarray(a)[None]).to(DEV, dt if i in (0, 1, 2, 5) else torch.float32)
            for i, a in enumerate(per)]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("train", [False, True])
def test_block_replays(train, dt):
    from kernels.block_norm import residual_rms_norm, rms_norm_gated
    from kernels.gated_delta import gated_delta_rule
    first, second = _inputs(150, dt, 1), _inputs(150, dt, 2)
    cu = torch.tensor([0, 20, 20, 150], device=DEV, dtype=torch.int32)
    w = torch.ones(256, device=DEV)

    def run(q, k, v, g, beta, do):
        leaves = [t.requires_grad_() for t in (q, k, v, g, beta)] if train else [q, k, v, g, beta]
        o, fin = gated_delta_rule(*leaves, return_final_states=True, cu_seqlens=cu)
        y = rms_norm_gated(o.flatten(-2), leaves[2].flatten(-2), w, group_size=64)
        y, h = residual_rms_norm(y, None, w)
        grads = torch.autograd.grad([y, h], leaves, [do.flatten(-2)] * 2) if train else []
        return [y.detach(), h.detach(), fin.detach(), *grads]

    want = [run(*[t.clone() for t in x]) for x in (first, second)]
    static = [t.clone() for t in first]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(*static)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = run(*static)
    torch.cuda.synchronize()
    for x, ref in zip((second, first), reversed(want)):
        with torch.no_grad():
            for a, b in zip(static, x):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, ref))
