"""A recurrent draft model, distilled from a teacher's top logits and then used to
draft tokens that the teacher verifies.

    python examples/recurrent_draft.py [--steps 300]

The "teacher" is a fixed random bigram table: the distribution of the next token
given the last one.  Training sees only its 16 best logits per position, as a
stored distillation set would hold them.  A layer is

    y, r = add_rms_norm(x, r)     the residual's addition and the norm
    x = gated_scan(y W) V         the recurrence mixes the sequence
    y, r = add_rms_norm(x, r)
    x = swiglu(y G, y U) D        the MLP

and drafting runs the same layers a token at a time: gated_step, and the norm
before the MLP with its output in 8 bits, as an 8-bit matrix product would take
it.  Matrix products are torch's.
"""

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from oxitorch_b200 import functional as F  # noqa: E402
from oxitorch_b200.optim import AdamW  # noqa: E402

VOCAB, DIM, HIDDEN, LAYERS, TOP = 512, 128, 256, 2, 16


class DraftModel:
    def __init__(self, generator):
        def matrix(rows, cols):
            return (torch.randn(rows, cols, device="cuda", generator=generator) / rows ** 0.5).requires_grad_()

        def ones(n):
            return torch.ones(n, device="cuda", requires_grad=True)
        self.embedding = matrix(VOCAB, DIM)
        self.layers = [{"norm1": ones(DIM), "mix": matrix(DIM, 2 * DIM), "out": matrix(DIM, DIM),
                        "norm2": ones(DIM), "up": matrix(DIM, 2 * HIDDEN), "down": matrix(HIDDEN, DIM)}
                       for _ in range(LAYERS)]
        self.norm, self.head = ones(DIM), matrix(DIM, VOCAB)

    def parameters(self):
        return [self.embedding, self.norm, self.head, *(p for layer in self.layers for p in layer.values())]

    def logits(self, tokens, starts=None):
        """[batch, length, vocab] for packed sequences; starts marks their first tokens."""
        batch, length = tokens.shape
        r = F.embedding(tokens.reshape(-1), self.embedding).view(batch, length, DIM)
        x = torch.zeros_like(r)
        for p in self.layers:
            y, r = F.add_rms_norm(x, r, p["norm1"], grad_mode="exact")
            mixed = y @ p["mix"]
            h, _ = F.gated_scan(mixed[..., :DIM], mixed[..., DIM:], starts=starts)
            y, r = F.add_rms_norm(h @ p["out"], r, p["norm2"], grad_mode="exact")
            gate, up = (y @ p["up"]).split(HIDDEN, -1)
            x = F.swiglu(gate.contiguous(), up.contiguous()) @ p["down"]
        y, _ = F.add_rms_norm(x, r, self.norm, grad_mode="exact")
        return y @ self.head

    @torch.no_grad()
    def step(self, tokens, states, out):
        """One token [batch] from the layers' states to `out`; returns [batch, vocab]."""
        r = F.embedding(tokens, self.embedding)
        x = torch.zeros_like(r)
        for p, state, after in zip(self.layers, states, out):
            y, r, _ = F.add_rms_norm_fwd(x, r, p["norm1"])
            mixed = y @ p["mix"]
            h = F.gated_step(mixed[:, :DIM], mixed[:, DIM:], state, out=after)
            q, scale, r = F.add_rms_norm_quant(h @ p["out"], r, p["norm2"], block=None)
            gate, up = (q.float() * scale @ p["up"]).split(HIDDEN, -1)
            x = F.swiglu_fwd(gate.contiguous(), up.contiguous()) @ p["down"]
        y, _, _ = F.add_rms_norm_fwd(x, r, self.norm)
        return y @ self.head


def train(model, teacher, steps, generator, batch=16, length=128, lr=3e-3):
    """Distils the teacher's top logits; returns the losses."""
    best = teacher.topk(TOP, -1)
    optimizer = AdamW(model.parameters(), lr=lr, weight_decay=0.0)
    losses = []
    for _ in range(steps):
        tokens = torch.randint(VOCAB, (batch, length), device="cuda", generator=generator)
        starts = torch.rand(batch, length, device="cuda", generator=generator) < 2 / length
        loss = F.distill_loss(model.logits(tokens, starts), best.values[tokens], best.indices[tokens])
        for p in model.parameters():
            p.grad = None
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return torch.stack(losses).tolist()


@torch.no_grad()
def draft_and_verify(model, teacher, prompt, rounds, generator, drafted=4):
    """Continues prompt [batch] for some rounds; returns the tokens of each batch row
    and the share of drafted tokens that the teacher kept."""
    batch = prompt.shape[0]

    def exponential(*shape):
        return torch.empty(*shape, device="cuda").exponential_(generator=generator)
    # the state before the last token of each row, and room for one after each draft
    states = [torch.zeros(drafted + 2, batch, DIM, device="cuda") for _ in range(LAYERS)]
    last, kept, texts = prompt, 0, [[int(t)] for t in prompt]
    each = torch.arange(batch, device="cuda")
    for _ in range(rounds):
        tokens, probs, current = [], [], last
        for k in range(drafted + 1):
            logits = model.step(current, [s[k] for s in states], [s[k + 1] for s in states])
            if k == drafted:  # only its state is wanted, in case all are kept
                break
            probs.append(F.softmax_fwd(logits))
            current = (probs[-1] / exponential(batch, VOCAB)).argmax(-1)
            tokens.append(current)
        tokens = torch.stack(tokens, 1)
        target = F.softmax_fwd(teacher[torch.cat([last[:, None], tokens], 1)])
        out, accepted = F.verify_draft(target, torch.stack(probs, 1), tokens,
                                       torch.rand(batch, drafted, device="cuda", generator=generator),
                                       exponential(batch, VOCAB))
        # back to the state before the new last token: what was drafted beyond the
        # kept tokens is forgotten
        for s in states:
            s[0] = s[accepted + 1, each]
        last = out[each, accepted]
        kept += int(accepted.sum())
        for row, text in zip(out.tolist(), texts):
            text += [t for t in row if t >= 0]
    return texts, kept / (rounds * batch * drafted)


def main(steps=300):
    generator = torch.Generator(device="cuda")
    generator.manual_seed(0)
    teacher = 3.0 * torch.randn(VOCAB, VOCAB, device="cuda", generator=generator)
    model = DraftModel(generator)
    prompt = torch.randint(VOCAB, (8,), device="cuda", generator=generator)
    _, before = draft_and_verify(model, teacher, prompt, 16, generator)
    losses = train(model, teacher, steps, generator)
    texts, after = draft_and_verify(model, teacher, prompt, 16, generator)
    print(f"distillation loss {losses[0]:.3f} -> {losses[-1]:.3f} in {steps} steps")
    print(f"drafted tokens kept by the teacher: {before:.0%} untrained, {after:.0%} trained")
    print(f"{sum(len(t) - 1 for t in texts)} tokens in {16 * len(texts)} verifications")
    return losses, before, after, texts


if __name__ == "__main__":
    parser = argparse.ArgumentParser()
    parser.add_argument("--steps", type=int, default=300)
    main(parser.parse_args().steps)
