"""examples/selective_policy.py: it runs, its steps continue what the sequence gives, and
its gradients are those of differences."""

import os
import sys

import pytest

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def test_a_few_steps_run():
    import torch
    import selective_policy as E
    model, history = E.main(steps=3)
    assert len(history) == 3 and all(0.0 <= r <= 1.0 for r in history)
    assert all(torch.isfinite(p).all() for p in model.parameters())


def test_sampling_draws_with_the_log_probabilities_of_the_sequence():
    """Token by token and over the whole sequence: the same model.  Each of the two layers
    and the head adds up to 128 products a number, in another order: 8 * 128 roundings of
    numbers of the size of the logits, about 10, at most."""
    import torch
    import selective_policy as E
    from oxitorch_b200 import functional as F
    generator = torch.Generator(device="cuda").manual_seed(3)
    model = E.Model(generator)
    tokens, logp = E.sample(model, 5, 20, generator)
    with torch.no_grad():
        want = F.token_logprobs(model.logits(tokens[:, :-1]), tokens[:, 1:])
    assert (logp - want).abs().max() <= 8 * 128 * 2.0 ** -24 * 10


def test_gradients_are_those_of_differences():
    """The loss along a random direction of every parameter: (f(p + h d) - f(p - h d)) / 2h.
    f32's rounding of a loss of about 1 leaves 2^-24 * 2 / 2h = 6e-6 at h = 1e-2 times the
    sums' tens of roundings, the third derivative h^2 / 6 times its size: 2e-2 of the
    direction's length covers both."""
    import torch
    import selective_policy as E
    from oxitorch_b200 import functional as F
    generator = torch.Generator(device="cuda").manual_seed(4)
    model = E.Model(generator)
    tokens, old = E.sample(model, 8, 24, generator)
    starts = torch.rand(8, 24, device="cuda", generator=generator) < 0.1
    advantages = torch.ones(8, 24, device="cuda")

    with torch.no_grad():
        now = F.token_logprobs(model.logits(tokens[:, :-1], starts), tokens[:, 1:])

    def loss():  # with ratios of about 0.9, which are not clipped
        return F.policy_loss(model.logits(tokens[:, :-1], starts), tokens[:, 1:], now + 0.1, advantages,
                             ref_logp=old - 0.2, clip=(0.99, 1e6), kl_coef=0.1)[0]
    grads = torch.autograd.grad(loss(), model.parameters())
    for p, g in zip(model.parameters(), grads):
        d = torch.randn(p.shape, device="cuda", generator=generator)
        d /= d.norm()
        h = 1e-2
        with torch.no_grad():
            keep = p.clone()
            p += h * d
            up = loss().item()
            p.copy_(keep - h * d)
            down = loss().item()
            p.copy_(keep)
        want, got = (up - down) / (2 * h), (g * d).sum().item()
        assert abs(got - want) <= 2e-2 * max(g.norm().item(), 1e-2)
