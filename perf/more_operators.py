"""Workloads of a selective state space model's training step and of its serving, for measuring them.

What such a model needs beside the layers of the recurrent draft model when it
is trained further on rewarded samples, from the first layer to the optimizer:

  conv    causal_conv (a short depthwise convolution over the sequence, then
          SiLU), forward and VJP, and causal_conv_step (one token from the
          inputs kept of the last ones);
  scan    selective_scan (h_t = exp(dt_t A) h_{t-1} + dt_t B_t x_t, y_t = C_t h_t
          + D x_t, gated by silu(z); dt = softplus(delta + delta_bias)), forward
          and VJP, and selective_step (one token from a state to the next);
  policy  policy_loss (the clipped policy loss of sampled tokens with a KL term
          towards a reference), the loss, the tokens' log-probabilities and the
          gradient of the logits;
  clip    clip_global_norm_ (the norm over all gradients of a model, and the
          gradients scaled where it is too large).

``run`` computes them in elementary torch operations, or with ``own`` set by
the calls of ``oxitorch_b200.functional`` and ``oxitorch_b200.tensor_ops``.
``exact`` computes them in 64 bits from their definitions.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}
CLIP = (0.2, 0.28)  # how far below and above 1 the ratio of the policies counts


# ---- the cases ---------------------------------------------------------------------

def listed():
    return [
        # one decoded token of 8 sequences at the width of the framework's own layer workloads (4096)
        {"name": "conv step, 8 tokens", "op": "conv", "what": "step", "batch": 8, "length": 1, "dim": 4096, "width": 4, "dtype": "f32", "packed": False},
        # a training step on 8192 tokens in 16 bits
        {"name": "conv train, bf16", "op": "conv", "what": "train", "batch": 4, "length": 2048, "dim": 4096, "width": 4, "dtype": "bf16", "packed": False},
        # several documents packed into rows of odd length, odd width, forward only
        {"name": "conv forward, packed", "op": "conv", "what": "forward", "batch": 3, "length": 4097, "dim": 1001, "width": 3, "dtype": "f32", "packed": True},
        # one decoded token of a server's 64 sequences
        {"name": "scan step, 64 tokens", "op": "scan", "what": "step", "batch": 64, "length": 1, "dim": 4096, "state": 16, "dtype": "bf16", "packed": False, "gated": True},
        # a training step on 8192 tokens, in f32 like the framework's own layers
        {"name": "scan train, f32", "op": "scan", "what": "train", "batch": 4, "length": 2048, "dim": 4096, "state": 16, "dtype": "f32", "packed": False, "gated": True},
        # packed prompts of odd length and width, forward only
        {"name": "scan prompt, packed", "op": "scan", "what": "forward", "batch": 3, "length": 4097, "dim": 1001, "state": 24, "dtype": "bf16", "packed": True, "gated": True},
        # one long sequence in 16 bits: few channels, so the time axis has to be split
        {"name": "scan train, long", "op": "scan", "what": "train", "batch": 1, "length": 32769, "dim": 1024, "state": 16, "dtype": "bf16", "packed": False, "gated": False},
        # a small batch of sampled tokens at the framework's vocabulary of 32000
        {"name": "policy, small batch", "op": "policy", "what": "train", "rows": 48, "vocab": 32000, "dtype": "f32", "kl": 0.0, "temperature": 1.0},
        # a training step at that vocabulary, with the KL term
        {"name": "policy, f32", "op": "policy", "what": "train", "rows": 8192, "vocab": 32000, "dtype": "f32", "kl": 0.05, "temperature": 1.0},
        # a large vocabulary in 16 bits, samples drawn at another temperature
        {"name": "policy, large vocabulary", "op": "policy", "what": "train", "rows": 8192, "vocab": 131072, "dtype": "bf16", "kl": 0.05, "temperature": 0.8},
        # the gradients of a small draft model: many short tensors
        {"name": "clip, small model", "op": "clip", "what": "train", "layers": 8, "dim": 256, "state": 16, "vocab": 1000, "dtype": "f32", "clipped": True},
        # those of one as wide as the framework's own layer workloads: 1.5 GB
        {"name": "clip, large model", "op": "clip", "what": "train", "layers": 2, "dim": 4096, "state": 16, "vocab": 32000, "dtype": "f32", "clipped": True},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["conv", "scan", "policy", "clip"])
    dtype = rng.choice(["f32", "bf16"])
    if op in ("conv", "scan"):
        what = rng.choice(["train", "train", "forward", "step"])
        dim = _spread(rng, 64, 8192)
        state = rng.choice([4, 10, 16, 16, 24, 32, 64, 128]) if op == "scan" else 4
        most = 2**29 // (16 if op == "conv" else state)
        batch = _spread(rng, 1, 256 if what == "step" else 16)
        length = 1 if what == "step" else _spread(rng, 1, max(1, min(65537, most // (dim * batch))))
        case = {"op": op, "what": what, "batch": batch, "length": length, "dim": dim, "dtype": dtype,
                "packed": what != "step" and rng.random() < 0.5}
        if op == "conv":
            return case | {"width": rng.choice([2, 3, 4, 4, 5, 8])}
        return case | {"state": state, "gated": rng.random() < 0.5}
    if op == "policy":
        vocab = _spread(rng, 1000, 262144)
        return {"op": op, "what": "train", "rows": _spread(rng, 1, min(16384, 2**28 // vocab)), "vocab": vocab,
                "dtype": dtype, "kl": rng.choice([0.0, 0.05, 0.2]), "temperature": rng.choice([1.0, 0.8, 1.5])}
    dim = _spread(rng, 32, 4096)
    layers = _spread(rng, 1, max(1, min(64, 2**28 // (6 * dim * dim + 2000))))
    vocab = _spread(rng, 1000, max(1000, min(131072, 2**26 // dim)))
    return {"op": op, "what": "train", "layers": layers, "dim": dim, "state": 16, "vocab": vocab, "dtype": dtype,
            "clipped": rng.random() < 0.8}


def _gradients(case):
    """The shapes of a model's parameters: an embedding, layers of twice its width inside, a norm and a head."""
    d, n = case["dim"], case["state"]
    rank = -(-d // 16)
    layer = [(d,), (4 * d, d), (2 * d, 4), (2 * d,), (rank + 2 * n, 2 * d), (2 * d, rank), (2 * d,), (2 * d, n), (2 * d,), (d, 2 * d)]
    return [(case["vocab"], d)] + layer * case["layers"] + [(d,), (case["vocab"], d)]


# ---- their inputs --------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, device="cuda", generator=g) * scale

    def uniform(*shape):
        return torch.rand(*shape, device="cuda", generator=g)

    s = dict(case)
    if case["op"] in ("conv", "scan"):
        t, shape = DTYPES[case["dtype"]], (case["batch"], case["length"], case["dim"])
        batch, _, dim = shape
        token = shape[:1] + shape[2:] if case["what"] == "step" else shape
        s["x"] = normal(*token).to(t)
        s["starts"] = uniform(*shape[:2]) < 0.002 if case["packed"] else None
        leaves = ["x"]
        if case["op"] == "conv":
            width = case["width"]
            s["weight"], s["bias"] = normal(dim, width, scale=width**-0.5), normal(dim, scale=0.1)
            s["x0"] = normal(batch, width - 1, dim).to(t)
            leaves += ["weight", "bias", "x0"]
            s["after"] = torch.empty_like(s["x0"])
            like = s["x0"]
        else:
            n = case["state"]
            s["delta"] = normal(*token, scale=0.5).to(t)
            # steps from a thousandth to a tenth, decays from 1 to the number of states: what the layer starts from
            step = torch.exp(uniform(dim) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
            s["delta_bias"] = step + torch.log(-torch.expm1(-step))
            s["A"] = -(torch.arange(1, n + 1, device="cuda") * torch.exp(normal(dim, n, scale=0.1)))
            s["B"], s["C"] = normal(*token[:-1], n).to(t), normal(*token[:-1], n).to(t)
            s["D"] = 1.0 + normal(dim, scale=0.1)
            s["z"] = normal(*token).to(t) if case["gated"] else None
            s["h0"] = normal(batch, dim, n, scale=0.1)
            leaves += ["delta", "A", "B", "C", "D", "delta_bias", "h0"] + (["z"] if case["gated"] else [])
            s["after"] = torch.empty_like(s["h0"])
            like = s["h0"]
        if case["what"] == "train":
            s["dy"], s["dlast"] = normal(*shape).to(t), normal(*like.shape).to(like.dtype)
            s["leaves"] = leaves
            for k in leaves:
                s[k].requires_grad_()
    elif case["op"] == "policy":
        rows, vocab, tau = case["rows"], case["vocab"], case["temperature"]
        logits = torch.randn(rows, vocab, device="cuda", generator=g, dtype=DTYPES[case["dtype"]]) * 2
        tokens = torch.randint(vocab, (rows, 1), device="cuda", generator=g)
        # sampled tokens are likely ones
        logits.scatter_(1, tokens, (normal(rows, 1) * 3 + 10).to(logits.dtype))
        z = logits.float() / tau
        now = (z.gather(1, tokens) - torch.logsumexp(z, 1, keepdim=True)).squeeze(1)
        del z
        s["old_logp"] = now + normal(rows, scale=0.2)  # the policy that sampled them, some steps ago
        s["ref_logp"] = now + normal(rows, scale=0.3) if case["kl"] else None
        s["advantages"] = 0.5 + normal(rows)  # rewarded samples, mostly
        # one token in sixteen is padding
        s["tokens"] = torch.where(uniform(rows) < 1 / 16, -1, tokens.squeeze(1))
        s["logits"] = logits.requires_grad_()
    else:
        shapes, t = _gradients(case), DTYPES[case["dtype"]]
        total = sum(math.prod(v) for v in shapes)
        scale = (10.0 if case["clipped"] else 0.1) / total**0.5
        s["grads"] = [normal(*v, scale=scale).to(t) for v in shapes]
        # the clipped ones go into one bucket, in order
        s["bucket"] = torch.empty(total, device="cuda", dtype=t)
        s["out"] = [v.view(w) for v, w in zip(s["bucket"].split([math.prod(v) for v in shapes]), shapes)]
        s["max_norm"] = 1.0
    return s


# ---- one pass ------------------------------------------------------------------------

def run(s):
    key = s["op"] + " " + s["what"]
    if own:
        return _OWN[key](s)
    with torch.no_grad():
        return _PLAIN[key](s)


def _own_train(s, y, last):
    grads = torch.autograd.grad((y, last), [s[k] for k in s["leaves"]], (s["dy"], s["dlast"]))
    return {"y": y, "last": last} | {"d" + k: v for k, v in zip(s["leaves"], grads)}


def _own_conv_train(s):
    from oxitorch_b200 import functional as F
    return _own_train(s, *F.causal_conv(s["x"], s["weight"], s["bias"], s["x0"], s["starts"], activation="silu"))


def _own_conv_forward(s):
    from oxitorch_b200 import functional as F
    y, last = F.causal_conv(s["x"], s["weight"], s["bias"], s["x0"], s["starts"], activation="silu")
    return {"y": y, "last": last}


def _own_conv_step(s):
    from oxitorch_b200 import functional as F
    y = F.causal_conv_step(s["x"], s["weight"], s["bias"], s["x0"], out=s["after"], activation="silu")
    return {"y": y, "last": s["after"]}


def _own_scan(s):
    from oxitorch_b200 import functional as F
    return F.selective_scan(s["x"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"],
                            delta_bias=s["delta_bias"], h0=s["h0"], starts=s["starts"])


def _own_scan_train(s):
    return _own_train(s, *_own_scan(s))


def _own_scan_forward(s):
    y, last = _own_scan(s)
    return {"y": y, "last": last}


def _own_scan_step(s):
    from oxitorch_b200 import functional as F
    y = F.selective_step(s["x"], s["delta"], s["A"], s["B"], s["C"], s["h0"], D=s["D"], z=s["z"],
                         delta_bias=s["delta_bias"], out=s["after"])  # kept apart: a rejected draft goes back to h0
    return {"y": y, "last": s["after"]}


def _own_policy(s):
    from oxitorch_b200 import functional as F
    loss, logp = F.policy_loss(s["logits"], s["tokens"], s["old_logp"], s["advantages"], ref_logp=s["ref_logp"],
                               clip=CLIP, kl_coef=s["kl"], temperature=s["temperature"])
    (grad,) = torch.autograd.grad(loss, (s["logits"],))
    return {"loss": loss, "logp": logp, "dlogits": grad}


def _own_clip(s):
    from oxitorch_b200 import tensor_ops as T
    norm = T.clip_global_norm_(s["grads"], s["max_norm"], out=s["out"])
    return {"norm": norm, "clipped": s["bucket"]}


def _plain_taps(s):
    """[x0, x] in 32 bits, and for each tap back in time which tokens it reaches within their sequence (None: all)."""
    x = s["x"].float()
    wide = torch.cat([s["x0"].float(), x], 1)
    if s["starts"] is None:
        return wide, [None] * s["width"]
    sequence = torch.nn.functional.pad(s["starts"].long().cumsum(1), (s["width"] - 1, 0))
    length = x.shape[1]
    return wide, [(sequence[:, -length:] == sequence[:, s["width"] - 1 - k:][:, :length]).unsqueeze(-1) for k in range(s["width"])]


def _plain_conv(s):
    wide, reach = _plain_taps(s)
    length, width = s["x"].shape[1], s["width"]
    taps = [wide[:, width - 1 - k:][:, :length] for k in range(width)]
    taps = [v if r is None else torch.where(r, v, 0.0) for v, r in zip(taps, reach)]
    u = s["bias"].expand_as(s["x"]).clone()
    for k, v in enumerate(taps):
        u += s["weight"][:, width - 1 - k] * v
    last = wide[:, length:]
    if s["starts"] is not None:  # what belongs to the row's last sequence
        sequence = torch.nn.functional.pad(s["starts"].long().cumsum(1), (width - 1, 0))
        last = torch.where((sequence[:, length:] == sequence[:, -1:]).unsqueeze(-1), last, 0.0)
    return taps, reach, u, last


def _plain_conv_forward(s):
    _, _, u, last = _plain_conv(s)
    t = s["x"].dtype
    return {"y": (u * torch.sigmoid(u)).to(t), "last": last.to(t)}


def _plain_conv_train(s):
    taps, reach, u, last = _plain_conv(s)
    t, width, length = s["x"].dtype, s["width"], s["x"].shape[1]
    sig = torch.sigmoid(u)
    du = s["dy"].float() * (sig + u * sig * (1 - sig))
    dwide = torch.zeros(u.shape[0], length + width - 1, u.shape[2], device=u.device)
    dweight = torch.empty_like(s["weight"])
    for k in range(width):
        d = du if reach[k] is None else torch.where(reach[k], du, 0.0)
        dwide[:, width - 1 - k:][:, :length] += s["weight"][:, width - 1 - k] * d
        dweight[:, width - 1 - k] = (du * taps[k]).sum((0, 1))
    dlast = s["dlast"].float()
    if s["starts"] is not None:
        sequence = torch.nn.functional.pad(s["starts"].long().cumsum(1), (width - 1, 0))
        dlast = torch.where((sequence[:, length:] == sequence[:, -1:]).unsqueeze(-1), dlast, 0.0)
    dwide[:, length:] += dlast
    return {"y": (u * sig).to(t), "last": last.to(t), "dx": dwide[:, width - 1:].to(t), "dweight": dweight,
            "dbias": du.sum((0, 1)), "dx0": dwide[:, :width - 1].to(t)}


def _plain_conv_step(s):
    wide = torch.cat([s["x0"].float(), s["x"].float().unsqueeze(1)], 1)
    u = (wide * s["weight"].t()).sum(1) + s["bias"]
    return {"y": (u * torch.sigmoid(u)).to(s["x"].dtype), "last": wide[:, 1:].to(s["x"].dtype)}


def _doubling(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1 from zero: each round doubles the span a place has seen."""
    n = 1
    while n < a.shape[1]:
        b = torch.cat([b[:, :n], torch.addcmul(b[:, n:], a[:, n:], b[:, :-n])], 1)
        a = torch.cat([a[:, :n], a[:, n:] * a[:, :-n]], 1)
        n *= 2
    return b


def _softplus(v):
    return v.clamp(min=0) + torch.log1p(torch.exp(-v.abs()))


def _plain_scan(s):
    """Steps, decays [batch, length, dim, state] (zero where a sequence starts) and states."""
    x = s["x"].float()
    raw = s["delta"].float() + s["delta_bias"]
    dt = _softplus(raw)
    a = torch.exp(dt.unsqueeze(-1) * s["A"])
    if s["starts"] is not None:
        a[s["starts"]] = 0.0
    v = (dt * x).unsqueeze(-1) * s["B"].float().unsqueeze(2)
    v[:, 0] += a[:, 0] * s["h0"]
    return x, raw, dt, a, _doubling(a, v)


def _plain_scan_out(s, x, h):
    y = (h * s["C"].float().unsqueeze(-2)).sum(-1) + s["D"] * x
    if s["z"] is None:
        return y, y
    z = s["z"].float()
    return y, y * z * torch.sigmoid(z)


def _plain_scan_forward(s):
    x, _, _, _, h = _plain_scan(s)
    return {"y": _plain_scan_out(s, x, h)[1].to(s["x"].dtype), "last": h[:, -1].clone()}


def _plain_scan_train(s):
    t = s["x"].dtype
    x, raw, dt, a, h = _plain_scan(s)
    inner, y = _plain_scan_out(s, x, h)
    got = {"y": y.to(t), "last": h[:, -1].clone()}
    dy = s["dy"].float()
    if s["z"] is not None:
        z = s["z"].float()
        sig = torch.sigmoid(z)
        got["dz"] = (dy * inner * (sig + z * sig * (1 - sig))).to(t)
        dy = dy * z * sig
    del inner, y
    got["dD"] = (dy * x).sum((0, 1))
    got["dC"] = (h * dy.unsqueeze(-1)).sum(2).to(t)
    lam = dy.unsqueeze(-1) * s["C"].float().unsqueeze(2)
    lam[:, -1] += s["dlast"]
    later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    lam = _doubling(later.flip(1), lam.flip(1)).flip(1)
    del later
    got["dh0"] = lam[:, 0] * a[:, 0]
    got["dB"] = (lam * (dt * x).unsqueeze(-1)).sum(2).to(t)
    through = (lam * s["B"].float().unsqueeze(2)).sum(-1)  # the gradient of dt x
    got["dx"] = (through * dt + s["D"] * dy).to(t)
    lam *= a
    lam *= torch.cat([s["h0"].unsqueeze(1), h[:, :-1]], 1)  # the gradient of dt A
    del h, a
    ddt = through * x + (lam * s["A"]).sum(-1)
    got["dA"] = (lam * dt.unsqueeze(-1)).sum((0, 1))
    ddelta = ddt * torch.sigmoid(raw)
    got["ddelta"], got["ddelta_bias"] = ddelta.to(t), ddelta.sum((0, 1))
    return got


def _plain_scan_step(s):
    x = s["x"].float()
    dt = _softplus(s["delta"].float() + s["delta_bias"])
    h = torch.exp(dt.unsqueeze(-1) * s["A"]) * s["h0"] + (dt * x).unsqueeze(-1) * s["B"].float().unsqueeze(1)
    return {"y": _plain_scan_out(s, x, h)[1].to(s["x"].dtype), "last": h}


def _plain_policy(s):
    logits, tokens, tau = s["logits"], s["tokens"], s["temperature"]
    rows = logits.shape[0]
    best = logits.amax(-1, keepdim=True)
    e = ((logits.float() - best.float()) / tau).exp()
    total = e.sum(-1, keepdim=True)
    there = tokens >= 0
    at = tokens.clamp(min=0).unsqueeze(-1)
    # a few numbers a row in 64 bits: the ratio may lie next to where it is clipped
    logp = (logits.gather(1, at).double() - best.double()) / tau - total.double().log()
    logp = torch.where(there, logp.squeeze(-1), 0.0)
    ratio = torch.exp(logp - s["old_logp"])
    free = ratio * s["advantages"]
    held = ratio.clamp(1 - CLIP[0], 1 + CLIP[1]) * s["advantages"]
    each = -torch.minimum(free, held)
    by = torch.where(free <= held, -free, 0.0)  # the loss's derivative by logp
    if s["ref_logp"] is not None:
        gap = s["ref_logp"] - logp
        each = each + s["kl"] * (torch.exp(gap) - gap - 1)
        by = by + s["kl"] * (1 - torch.exp(gap))
    loss = torch.where(there, each, 0.0).sum() / rows
    by = (torch.where(there, by, 0.0).unsqueeze(-1) / (rows * tau)).float()
    grad = e / total * -by
    grad.scatter_add_(1, at, by)
    return {"loss": loss.float(), "logp": logp.float(), "dlogits": grad.to(logits.dtype)}


def _plain_clip(s):
    squares = [g.float().square().sum(dtype=torch.float64) for g in s["grads"]]
    norm = torch.stack(squares).sum().sqrt()
    scale = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    flat = [(g.float() * scale).to(g.dtype).reshape(-1) for g in s["grads"]]
    return {"norm": norm.float(), "clipped": torch.cat(flat)}


_OWN = {"conv train": _own_conv_train, "conv forward": _own_conv_forward, "conv step": _own_conv_step,
        "scan train": _own_scan_train, "scan forward": _own_scan_forward, "scan step": _own_scan_step,
        "policy train": _own_policy, "clip train": _own_clip}
_PLAIN = {"conv train": _plain_conv_train, "conv forward": _plain_conv_forward, "conv step": _plain_conv_step,
          "scan train": _plain_scan_train, "scan forward": _plain_scan_forward, "scan step": _plain_scan_step,
          "policy train": _plain_policy, "clip train": _plain_clip}


# ---- what a pass cannot do without -----------------------------------------------------

def work(case):
    """Each pass reads its inputs once and writes its outputs once; an operation for every add, product and exponential."""
    op, what = case["op"], case["what"]
    if op in ("conv", "scan"):
        n, w = case["batch"] * case["length"] * case["dim"], SIZE[case["dtype"]]
        marks = case["batch"] * case["length"] if case["packed"] else 0
        both = 2 if what == "train" else 1  # forward, and the VJP on the same inputs
        if op == "conv":
            k = case["width"]
            ends = 2 * case["batch"] * (k - 1) * case["dim"] * w
            small = 4 * case["dim"] * (k + 1) * both
            # x -> y; x, dy -> dx
            moved = (5 if what == "train" else 2) * n * w
            return {"bytes": moved + both * (ends + marks) + small, "flops": (2 * k + 4) * n + (both - 1) * (6 * k + 10) * n}
        k, z = case["state"], 1 if case["gated"] else 0
        ends = 8 * case["batch"] * case["dim"] * k
        small = 4 * case["dim"] * (k + 2) * both
        rows = 2 * case["batch"] * case["length"] * k * w
        # x, delta, z -> y; x, delta, z, dy -> dx, ddelta, dz
        moved = (3 + z + (5 + 2 * z if what == "train" else 0)) * n * w
        flops = (7 * k + 10) * n + (both - 1) * (20 * k + 25) * n
        return {"bytes": moved + both * (ends + marks) + small + (3 if what == "train" else 1) * rows, "flops": flops}
    if op == "policy":  # logits -> dlogits, the loss
        n = case["rows"] * case["vocab"]
        return {"bytes": 2 * n * SIZE[case["dtype"]] + 28 * case["rows"], "flops": 5 * n}
    n = sum(math.prod(v) for v in _gradients(case))  # gradients -> clipped ones
    return {"bytes": 2 * n * SIZE[case["dtype"]], "flops": 3 * n}


# ---- in 64 bits ------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "policy":
        return _exact_policy(s)
    with torch.no_grad():
        if case["op"] == "conv":
            return _exact_conv(s)
        if case["op"] == "scan":
            return _exact_scan(s)
        return _exact_clip(s)


def _exact_conv(s):
    width, step = s["width"], s["what"] == "step"
    x = s["x"].unsqueeze(1) if step else s["x"]
    batch, length, dim = x.shape
    wide = torch.cat([s["x0"], x], 1).double()
    place = torch.arange(width - 1, width - 1 + length, device=x.device).expand(batch, length)
    first = torch.zeros_like(place)  # the first place of [x0, x] that belongs to a token's sequence
    if s["starts"] is not None:
        first = torch.where(s["starts"], place, 0).cummax(1).values
    each = torch.arange(batch, device=x.device).unsqueeze(1)
    u = s["bias"].double() + torch.zeros(batch, length, dim, device=x.device, dtype=torch.float64)
    mine = []
    for k in range(width):  # weight[:, k] meets the input width - 1 - k tokens before
        at = place - (width - 1 - k)
        ok = (at >= first).unsqueeze(-1)
        mine.append((at, ok))
        u += s["weight"][:, k].double() * wide[each, at] * ok
    y = u / (1 + torch.exp(-u))
    kept = (torch.arange(length, length + width - 1, device=x.device) >= first[:, -1:]).unsqueeze(-1)
    last = wide[:, length:] * kept
    if s["what"] != "train":
        return {"y": y.squeeze(1) if step else y, "last": last}
    sig = 1 / (1 + torch.exp(-u))
    du = s["dy"].double() * sig * (1 + u * (1 - sig))
    dwide = torch.zeros_like(wide)
    dwide[:, length:] += s["dlast"].double() * kept
    dweight = torch.zeros_like(s["weight"], dtype=torch.float64)
    for k, (at, ok) in enumerate(mine):
        d = du * ok
        dweight[:, k] = torch.einsum("btd,btd->d", d, wide[each, at])
        dwide[:, k:k + length] += d * s["weight"][:, k].double()
    return {"y": y, "last": last, "dx": dwide[:, width - 1:], "dweight": dweight,
            "dbias": torch.einsum("btd->d", du), "dx0": dwide[:, :width - 1]}


def _exact_scan(s):
    step = s["what"] == "step"
    x, delta, B, C = (v.double().unsqueeze(1) if step else v.double() for v in (s["x"], s["delta"], s["B"], s["C"]))
    z = None if s["z"] is None else s["z"].double().unsqueeze(1) if step else s["z"].double()
    A, D = s["A"].double(), s["D"].double()
    length = x.shape[1]
    raw = delta + s["delta_bias"].double()
    dt = torch.logaddexp(raw, torch.zeros_like(raw))
    a = torch.exp(torch.einsum("btd,dn->btdn", dt, A))
    if s["starts"] is not None:
        a.masked_fill_(s["starts"][:, :, None, None], 0.0)
    h = torch.einsum("btd,btn->btdn", dt * x, B)
    before = s["h0"].double()
    for t in range(length):
        before = h[:, t].addcmul_(a[:, t], before)
    inner = torch.einsum("btdn,btn->btd", h, C) + D * x
    y = inner if z is None else inner * z / (1 + torch.exp(-z))
    last = h[:, -1].clone()
    if s["what"] != "train":
        return {"y": y.squeeze(1) if step else y, "last": last}
    got = {"y": y, "last": last}
    dy = s["dy"].double()
    if z is not None:
        sig = 1 / (1 + torch.exp(-z))
        got["dz"] = dy * inner * sig * (1 + z * (1 - sig))
        dy = dy * z * sig
    got["dD"], got["dC"] = torch.einsum("btd,btd->d", dy, x), torch.einsum("btdn,btd->btn", h, dy)
    lam = torch.einsum("btd,btn->btdn", dy, C)
    lam[:, -1] += s["dlast"].double()
    for t in range(length - 2, -1, -1):
        lam[:, t].addcmul_(a[:, t + 1], lam[:, t + 1])
    got["dB"] = torch.einsum("btdn,btd->btn", lam, dt * x)
    through = torch.einsum("btdn,btn->btd", lam, B)
    got["dx"] = through * dt + D * dy
    lam.mul_(a)
    del a
    got["dh0"] = lam[:, 0].clone()
    lam[:, 0] *= s["h0"].double()
    lam[:, 1:] *= h[:, :-1]
    del h
    ddelta = (torch.einsum("btdn,dn->btd", lam, A) + through * x) / (1 + torch.exp(-raw))
    got["dA"] = torch.einsum("btdn,btd->dn", lam, dt)
    got["ddelta"], got["ddelta_bias"] = ddelta, torch.einsum("btd->d", ddelta)
    return got


def _exact_policy(s):
    logits = s["logits"].detach().double().requires_grad_()
    there = s["tokens"] >= 0
    logp = torch.log_softmax(logits / s["temperature"], 1)
    logp = logp[torch.arange(len(there), device=logits.device), s["tokens"].clamp(min=0)]
    ratio = torch.exp(logp - s["old_logp"].double())
    adv = s["advantages"].double()
    each = -torch.where(adv >= 0, ratio.clamp(max=1 + CLIP[1]), ratio.clamp(min=1 - CLIP[0])) * adv
    if s["ref_logp"] is not None:
        each = each + s["kl"] * (torch.expm1(s["ref_logp"].double() - logp) - (s["ref_logp"].double() - logp))
    loss = (each * there).sum() / len(there)
    (grad,) = torch.autograd.grad(loss, logits)
    return {"loss": loss.detach(), "logp": (logp * there).detach(), "dlogits": grad}


def _exact_clip(s):
    norm = torch.sqrt(sum(torch.dot(g.reshape(-1).double(), g.reshape(-1).double()) for g in s["grads"]))
    flat = torch.cat([g.reshape(-1) for g in s["grads"]]).double()
    factor = s["max_norm"] / (norm + 1e-6)
    return {"norm": norm, "clipped": flat * factor if factor < 1 else flat}
