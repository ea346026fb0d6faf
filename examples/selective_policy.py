"""A selective state space model that samples sequences by itself and is trained on
the rewarded ones.

    python examples/selective_policy.py [--steps 150]

A layer is

    u, z = x W_in                     two projections in one product
    u = causal_conv(u)                the last four tokens, then SiLU
    dt, B, C = u W_bc                 what makes the scan selective
    x = x + selective_scan(u, dt W_dt, A, B, C, D, z) W_out

Sequences are sampled a token at a time (causal_conv_step, selective_step, from the
states that they keep); a token is rewarded if it follows from the one two places
before it by a fixed rule, which the model has to find out.  Training takes several
clipped policy steps on each batch of samples, with a KL term towards the model as it
was in the beginning, and clips the gradients by their norm.  Matrix products are
torch's.
"""

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from oxitorch_b200 import functional as F  # noqa: E402
from oxitorch_b200.optim import AdamW  # noqa: E402
from oxitorch_b200.tensor_ops import clip_global_norm_  # noqa: E402

VOCAB, DIM, INNER, STATE, RANK, WIDTH, LAYERS = 64, 64, 128, 16, 4, 4, 2


class Model:
    def __init__(self, generator):
        def matrix(rows, cols, scale=1.0):
            w = torch.randn(rows, cols, device="cuda", generator=generator) * (scale / rows ** 0.5)
            return w.requires_grad_()

        def constant(*shape, value=0.0):
            return torch.full(shape, value, device="cuda").requires_grad_()
        self.embedding, self.head = matrix(VOCAB, DIM, scale=VOCAB ** 0.5), matrix(DIM, VOCAB)
        decays = torch.log(torch.arange(1.0, STATE + 1, device="cuda")).expand(INNER, STATE)
        self.layers = [{"in": matrix(DIM, 2 * INNER), "conv": matrix(INNER, WIDTH, scale=INNER ** 0.5 / 2),
                        "conv_bias": constant(INNER), "bc": matrix(INNER, RANK + 2 * STATE),
                        "dt": matrix(RANK, INNER), "dt_bias": constant(INNER, value=-2.0),
                        "log_A": decays.clone().requires_grad_(), "D": constant(INNER, value=1.0),
                        "out": matrix(INNER, DIM)} for _ in range(LAYERS)]

    def parameters(self):
        return [self.embedding, self.head, *(p for layer in self.layers for p in layer.values())]

    @staticmethod
    def _selected(p, u):
        dbc = u @ p["bc"]
        return dbc[..., :RANK] @ p["dt"], dbc[..., RANK:RANK + STATE], dbc[..., RANK + STATE:]

    def logits(self, tokens, starts=None):
        """[batch, length, vocab] for packed sequences; starts marks their first tokens."""
        x = F.embedding(tokens.reshape(-1), self.embedding).view(*tokens.shape, DIM)
        for p in self.layers:
            u, z = (x @ p["in"]).split(INNER, -1)
            u, _ = F.causal_conv(u, p["conv"], p["conv_bias"], starts=starts)
            delta, B, C = self._selected(p, u)
            y, _ = F.selective_scan(u, delta, -torch.exp(p["log_A"]), B, C, p["D"], z, p["dt_bias"], starts=starts)
            x = x + y @ p["out"]
        return x @ self.head

    def states(self, batch):
        return [(torch.zeros(batch, WIDTH - 1, INNER, device="cuda"), torch.zeros(batch, INNER, STATE, device="cuda"))
                for _ in range(LAYERS)]

    @torch.no_grad()
    def step(self, tokens, states):
        """One token [batch]; moves the states on and returns the logits [batch, vocab]."""
        x = F.embedding(tokens, self.embedding)
        for p, (inputs, state) in zip(self.layers, states):
            u, z = (x @ p["in"]).split(INNER, -1)
            u = F.causal_conv_step(u, p["conv"], p["conv_bias"], inputs)
            delta, B, C = self._selected(p, u)
            y = F.selective_step(u, delta, -torch.exp(p["log_A"]), B, C, state, p["D"], z, p["dt_bias"])
            x = x + y @ p["out"]
        return x @ self.head


def sample(model, batch, length, generator):
    """Tokens [batch, length + 1] from the model, the first at random, and the
    log-probabilities [batch, length] that those after it were drawn with."""
    tokens = torch.randint(VOCAB, (batch,), device="cuda", generator=generator)
    states, out, logps = model.states(batch), [tokens], []
    for _ in range(length):
        logits = model.step(tokens, states)
        race = torch.empty_like(logits).exponential_(generator=generator)
        tokens = (F.softmax_fwd(logits) / race).argmax(-1)
        logps.append(F.token_logprobs(logits, tokens))
        out.append(tokens)
    return torch.stack(out, 1), torch.stack(logps, 1)


def rewards(tokens, rule):
    """1 for each token after the second that the rule gives for the one two before it."""
    right = torch.zeros(tokens.shape[0], tokens.shape[1] - 1, device=tokens.device)
    right[:, 1:] = (tokens[:, 2:] == rule[tokens[:, :-2]]).float()
    return right


def train_step(model, reference, optimizer, rule, generator, batch=64, length=32, passes=2):
    """Samples, then takes a few policy steps on them; returns the mean reward, the losses
    and the gradients' norms before clipping."""
    tokens, old = sample(model, batch, length, generator)
    reward = rewards(tokens, rule)
    advantages = reward - reward.mean()
    with torch.no_grad():
        ref = F.token_logprobs(reference.logits(tokens[:, :-1]), tokens[:, 1:])
    losses, norms = [], []
    for _ in range(passes):
        loss, _ = F.policy_loss(model.logits(tokens[:, :-1]), tokens[:, 1:], old, advantages, ref_logp=ref,
                                clip=(0.2, 0.28), kl_coef=0.001)
        for p in model.parameters():
            p.grad = None
        loss.backward()
        norms.append(clip_global_norm_([p.grad for p in model.parameters()], 1.0))
        optimizer.step()
        losses.append(loss.detach())
    return reward.mean(), losses, norms


def main(steps=150):
    generator = torch.Generator(device="cuda")
    generator.manual_seed(0)
    model, rule = Model(generator), torch.randperm(VOCAB, device="cuda", generator=generator)
    generator.manual_seed(0)
    reference = Model(generator)
    optimizer = AdamW(model.parameters(), lr=2e-3, weight_decay=0.0)
    history = [train_step(model, reference, optimizer, rule, generator)[0] for _ in range(steps)]
    history = torch.stack(history).tolist()
    print(f"mean reward {history[0]:.3f} -> {history[-1]:.3f} in {steps} steps")
    return model, history


if __name__ == "__main__":
    parser = argparse.ArgumentParser()
    parser.add_argument("--steps", type=int, default=150)
    main(parser.parse_args().steps)
