"""The example model: the two norms, the rule on packed sequences (forward, backward) and the step, together."""

import importlib.util
import os

import pytest
import torch

_PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ema-kernels_b200", "examples",
                     "delta_block.py")
_spec = importlib.util.spec_from_file_location("delta_block", _PATH)
ex = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(ex)


def test_recall_batch_asks_for_listed_pairs():
    tokens, before, cu, at = ex.recall_batch([4, 9, 7], 4, 64, torch.Generator().manual_seed(1))
    assert cu.tolist() == [0, 16, 42, 64] and len(tokens) == 64 and at.shape == (3, 4)
    for i, n in enumerate([4, 9, 7]):
        s = tokens[cu[i]:cu[i + 1]]
        listed = dict(zip(s[:2 * n:2].tolist(), s[1:2 * n:2].tolist()))
        assert before[cu[i]] == 0 and torch.equal(before[cu[i] + 1:cu[i + 1]], s[:-1])
        for j in at[i].tolist():
            assert listed[tokens[j].item()] == tokens[j + 1].item()


@pytest.mark.gpu
def test_trains_and_decodes_as_it_prefills():
    torch.manual_seed(0)
    dev, gen, vocab = torch.device("cuda"), torch.Generator().manual_seed(0), 32
    model = ex.DeltaLM(vocab, width=128, layers=2).to(dev)
    losses = ex.train(model, 30, vocab, gen, dev, batch=8, most=8)
    assert all(x == x for x in losses)
    assert sum(losses[-5:]) < sum(losses[:5])
    for p in model.parameters():
        assert p.grad is None or torch.isfinite(p.grad).all()
    _, got, whole = ex.recall(model, vocab, gen, dev, rows=5, most=8)
    # the same roundings to bf16 (2^-9 each at most, some eight a layer in sequence, two layers and the head) fall
    # differently in calls of other shapes: 2 * 8 * 2^-8 = 2^-4 of the largest logit
    assert (got - whole).abs().max() <= 2.0 ** -4 * whole.abs().max()
