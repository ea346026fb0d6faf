"""The recurrent draft model's operators together, as examples/recurrent_draft.py
uses them: distillation lowers the loss, a step continues the scan, and the
teacher keeps more of a trained model's drafts."""

import os
import sys

import pytest

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def test_distil_draft_verify():
    import recurrent_draft as E
    losses, before, after, texts = E.main(steps=300)
    # a KL divergence of a table that the model can hold: a quarter of where it
    # began is far from converged and far from chance
    assert losses[-1] < 0.25 * losses[0]
    assert after > 0.3 and after > 3 * before
    assert all(0 <= t < E.VOCAB for text in texts for t in text)
    assert all(len(t) > 16 for t in texts)  # a round adds a token at least


def test_steps_continue_what_the_scan_computes():
    """Token by token, with the 8-bit norm, the logits are the sequence's within the
    8-bit rounding: 2^-4 of an element at most, averaged over 128 of them."""
    import torch
    import recurrent_draft as E
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    model = E.DraftModel(g)
    tokens = torch.randint(E.VOCAB, (3, 20), device="cuda", generator=g)
    with torch.no_grad():
        want = model.logits(tokens)
        states = [torch.zeros(3, E.DIM, device="cuda") for _ in range(E.LAYERS)]
        for t in range(20):
            got = model.step(tokens[:, t], states, states)
            off = (got - want[:, t]).norm() / want[:, t].norm()
            assert off < 2.0 ** -4
