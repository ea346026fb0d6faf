"""Workloads of the recurrent draft model's operators, for measuring them.

Four operators that a small recurrent language model needs when it is distilled
from a larger one and then drafts tokens for it:

  norm     add_rms_norm (the residual's addition, then RMSNorm), forward and
           VJP, and add_rms_norm_quant (the same norm written in 8 bits, with
           a scale for each block of 128 columns);
  scan     gated_scan (h_t = a_t h_{t-1} + (1 - a_t) x_t with a = sigmoid of
           the gate), forward and VJP over a whole sequence, and gated_step
           (one token from a state to the next);
  distill  distill_loss (cross-entropy against a teacher's top logits minus
           the teacher's entropy), the loss and the student's gradient;
  verify   verify_draft (which drafted tokens the target keeps, and the token
           that follows them), from given random numbers.

``run`` computes them in elementary torch operations, or with ``own`` set by
the calls of ``oxitorch_b200.functional``.  ``exact`` computes them in 64 bits
from their definitions.
"""

import math

import torch

own = False

EPS = 1e-6
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}


# ---- the cases ---------------------------------------------------------------------

def listed():
    return [
        # one decoded token of 8 sequences at the width of the framework's own layer workloads (4096)
        {"name": "norm quant, 8 tokens", "op": "norm", "what": "quant", "rows": 8, "cols": 4096, "dtype": "bf16"},
        # a training step at the framework's LayerNorm workload's shape
        {"name": "norm train, f32", "op": "norm", "what": "train", "rows": 16384, "cols": 4096, "dtype": "f32"},
        # a prompt's tokens before a layer in 8 bits; a width whose last block holds 8 columns
        {"name": "norm quant, prompt", "op": "norm", "what": "quant", "rows": 8192, "cols": 5000, "dtype": "bf16"},
        # one decoded token of 8 sequences
        {"name": "scan step, 8 tokens", "op": "scan", "what": "step", "batch": 8, "length": 1, "dim": 4096, "dtype": "f32", "packed": False},
        # a training step on 8192 tokens, in f32 like the framework's own layers
        {"name": "scan train, f32", "op": "scan", "what": "train", "batch": 4, "length": 2048, "dim": 4096, "dtype": "f32", "packed": False},
        # several documents packed into rows of odd length, odd width, forward only
        {"name": "scan forward, packed", "op": "scan", "what": "forward", "batch": 3, "length": 4097, "dim": 1001, "dtype": "f32", "packed": True},
        # one long sequence in 16 bits: few channels, so the time axis has to be split
        {"name": "scan train, long", "op": "scan", "what": "train", "batch": 1, "length": 65537, "dim": 1024, "dtype": "bf16", "packed": False},
        # a small batch against a teacher's 16 best logits, at the framework's vocabulary of 32000
        {"name": "distill, small batch", "op": "distill", "what": "train", "rows": 48, "vocab": 32000, "top": 16, "dtype": "f32", "temperature": 2.0},
        # a training step at that vocabulary
        {"name": "distill, f32", "op": "distill", "what": "train", "rows": 8192, "vocab": 32000, "top": 64, "dtype": "f32", "temperature": 1.0},
        # a large vocabulary in 16 bits
        {"name": "distill, large vocabulary", "op": "distill", "what": "train", "rows": 8192, "vocab": 131072, "top": 100, "dtype": "bf16", "temperature": 1.0},
        # one sequence with 4 drafted tokens
        {"name": "verify, 1 sequence", "op": "verify", "what": "serve", "batch": 1, "drafted": 4, "vocab": 32000},
        # a server's batch, a large vocabulary
        {"name": "verify, 64 sequences", "op": "verify", "what": "serve", "batch": 64, "drafted": 7, "vocab": 131072},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["norm", "scan", "distill", "verify"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "norm":
        cols = _spread(rng, 64, 16384)
        rows = _spread(rng, 1, min(32768, 2**26 // cols))
        return {"op": op, "what": rng.choice(["train", "quant"]), "rows": rows, "cols": cols, "dtype": dtype}
    if op == "scan":
        what = rng.choice(["train", "train", "forward", "step"])
        dim = _spread(rng, 64, 8192)
        batch = _spread(rng, 1, 256 if what == "step" else 16)
        length = 1 if what == "step" else _spread(rng, 1, min(65537, 2**25 // (dim * batch)))
        return {"op": op, "what": what, "batch": batch, "length": length, "dim": dim, "dtype": dtype,
                "packed": what != "step" and rng.random() < 0.5}
    if op == "distill":
        vocab = _spread(rng, 1000, 262144)
        return {"op": op, "what": "train", "rows": _spread(rng, 1, min(16384, 2**28 // vocab)), "vocab": vocab,
                "top": _spread(rng, 1, 512), "dtype": dtype, "temperature": rng.choice([1.0, 1.5, 4.0])}
    return {"op": op, "what": "serve", "batch": _spread(rng, 1, 128), "drafted": _spread(rng, 1, 12),
            "vocab": _spread(rng, 1000, 262144)}


# ---- their inputs --------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, device="cuda", generator=g) * scale

    def uniform(*shape):
        return torch.rand(*shape, device="cuda", generator=g)

    s = dict(case)
    if case["op"] == "norm":
        t, shape = DTYPES[case["dtype"]], (case["rows"], case["cols"])
        s["x"] = normal(*shape).to(t)
        s["residual"] = normal(*shape, scale=3.0)  # the residual stream is kept in 32 bits
        s["weight"] = 0.5 + uniform(case["cols"])
        if case["what"] == "train":
            s["dy"], s["dr"] = normal(*shape).to(t), normal(*shape)
            for k in ("x", "residual", "weight"):
                s[k].requires_grad_()
    elif case["op"] == "scan":
        t, shape = DTYPES[case["dtype"]], (case["batch"], case["length"], case["dim"])
        s["x"] = normal(*shape).to(t)
        # gates of a trained layer: from channels that forget in a step to ones that hold for hundreds
        s["gate"] = (normal(*shape) + torch.linspace(-2.0, 6.0, case["dim"], device="cuda")).to(t)
        s["h0"] = normal(case["batch"], case["dim"])
        s["starts"] = uniform(case["batch"], case["length"]) < 0.002 if case["packed"] else None
        if case["what"] == "step":
            s["x"], s["gate"] = s["x"][:, 0].contiguous(), s["gate"][:, 0].contiguous()
            s["state"] = torch.empty_like(s["h0"])
        if case["what"] == "train":
            s["dh"], s["dlast"] = normal(*shape).to(t), normal(case["batch"], case["dim"])
            for k in ("x", "gate", "h0"):
                s[k].requires_grad_()
    elif case["op"] == "distill":
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        t = DTYPES[case["dtype"]]
        logits = torch.randn(rows, vocab, device="cuda", generator=g, dtype=t) * 2
        # the teacher's best tokens: distinct, spread over the vocabulary, likely for the student too
        first = torch.randint(vocab, (rows, 1), device="cuda", generator=g)
        ids = (first + torch.arange(top, device="cuda") * (vocab // top)) % vocab
        value = (10.0 - 0.1 * torch.arange(top, device="cuda") + normal(rows, top)).sort(-1, descending=True).values
        logits.scatter_(1, ids, (value + normal(rows, top)).to(t))
        # some rows hold fewer than `top`, and one in sixteen (padding tokens) none
        kept = torch.randint(1, 2 * top, (rows, 1), device="cuda", generator=g)
        kept = torch.where(uniform(rows, 1) < 1 / 16, 0, kept)
        s["teacher_ids"] = torch.where(torch.arange(top, device="cuda") < kept, ids, -1)
        s["teacher_logits"] = value
        s["logits"] = logits.requires_grad_()
    else:
        batch, drafted, vocab = case["batch"], case["drafted"], case["vocab"]
        logits = normal(batch, drafted + 1, vocab, scale=3.0)
        s["target"] = torch.softmax(logits, -1)
        s["draft"] = torch.softmax(logits[:, :drafted] + normal(batch, drafted, vocab, scale=0.7), -1)
        race = -torch.log1p(-uniform(batch, drafted, vocab))
        s["tokens"] = (s["draft"] / race).argmax(-1)  # drafted as the draft model would
        s["lengths"] = torch.randint(drafted // 2, drafted + 1, (batch,), device="cuda", generator=g)
        s["uniform"] = uniform(batch, drafted)
        s["race"] = -torch.log1p(-uniform(batch, vocab))
    return s


# ---- one pass ------------------------------------------------------------------------

def run(s):
    key = s["op"] + " " + s["what"]
    if own:
        return _OWN[key](s)
    with torch.no_grad():
        return _PLAIN[key](s)


def _own_norm_train(s):
    from oxitorch_b200 import functional as F
    y, r = F.add_rms_norm(s["x"], s["residual"], s["weight"], EPS, grad_mode="exact")
    dx, dres, dw = torch.autograd.grad((y, r), (s["x"], s["residual"], s["weight"]), (s["dy"], s["dr"]))
    return {"y": y, "r": r, "dx": dx, "dresidual": dres, "dweight": dw}


def _own_norm_quant(s):
    from oxitorch_b200 import functional as F
    q, scale, r = F.add_rms_norm_quant(s["x"], s["residual"], s["weight"], EPS)
    return {"q": q, "scale": scale, "r": r}


def _own_scan_train(s):
    from oxitorch_b200 import functional as F
    h, last = F.gated_scan(s["x"], s["gate"], s["h0"], s["starts"])
    dx, dgate, dh0 = torch.autograd.grad((h, last), (s["x"], s["gate"], s["h0"]), (s["dh"], s["dlast"]))
    return {"h": h, "last": last, "dx": dx, "dgate": dgate, "dh0": dh0}


def _own_scan_forward(s):
    from oxitorch_b200 import functional as F
    h, last = F.gated_scan(s["x"], s["gate"], s["h0"], s["starts"])
    return {"h": h, "last": last}


def _own_scan_step(s):
    from oxitorch_b200 import functional as F
    h = F.gated_step(s["x"], s["gate"], s["h0"], out=s["state"])  # kept apart: a rejected draft goes back to h0
    return {"h": h, "state": s["state"]}


def _own_distill(s):
    from oxitorch_b200 import functional as F
    loss = F.distill_loss(s["logits"], s["teacher_logits"], s["teacher_ids"], s["temperature"])
    (grad,) = torch.autograd.grad(loss, (s["logits"],))
    return {"loss": loss, "dlogits": grad}


def _own_verify(s):
    from oxitorch_b200 import functional as F
    tokens, accepted = F.verify_draft(s["target"], s["draft"], s["tokens"], s["uniform"], s["race"], s["lengths"])
    return {"tokens": tokens, "accepted": accepted}


def _plain_norm(s):
    r = s["x"].float() + s["residual"]
    rstd = torch.rsqrt((r * r).mean(-1, keepdim=True) + EPS)
    return r, rstd, r * rstd * s["weight"]


def _plain_norm_train(s):
    r, rstd, y = _plain_norm(s)
    t, dy = s["x"].dtype, s["dy"].float()
    xhat = r * rstd
    g = dy * s["weight"]
    d = s["dr"] + rstd * (g - xhat * (g * xhat).mean(-1, keepdim=True))
    return {"y": y.to(t), "r": r, "dx": d.to(t), "dresidual": d, "dweight": (dy * xhat).sum(0)}


def _plain_norm_quant(s):
    r, _, y = _plain_norm(s)
    rows, cols = y.shape
    blocks = -(-cols // 128)
    padded = torch.zeros(rows, blocks * 128, device=y.device)
    padded[:, :cols] = y
    padded = padded.view(rows, blocks, 128)
    scale = (padded.abs().amax(-1) / 448.0).clamp(min=2.0**-126)
    q = (padded / scale.unsqueeze(-1)).view(rows, -1)[:, :cols].to(torch.float8_e4m3fn)
    return {"q": q, "scale": scale, "r": r}


def _doubling(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1 from zero: each round doubles the span a place has seen."""
    n = 1
    while n < a.shape[1]:
        b = torch.cat([b[:, :n], b[:, n:] + a[:, n:] * b[:, :-n]], 1)
        a = torch.cat([a[:, :n], a[:, n:] * a[:, :-n]], 1)
        n *= 2
    return b


def _plain_scan(s):
    x, gate = s["x"].float(), s["gate"].float()
    a, b = torch.sigmoid(gate), torch.sigmoid(-gate)
    keep = a if s["starts"] is None else torch.where(s["starts"].unsqueeze(-1), 0.0, a)
    v = b * x
    v[:, 0] += keep[:, 0] * s["h0"]
    return x, a, b, keep, _doubling(keep, v)


def _plain_scan_forward(s):
    h = _plain_scan(s)[-1]
    return {"h": h.to(s["x"].dtype), "last": h[:, -1].clone()}


def _plain_scan_train(s):
    t = s["x"].dtype
    x, a, b, keep, h = _plain_scan(s)
    dh = s["dh"].to(torch.float32, copy=True)
    dh[:, -1] += s["dlast"]
    later = torch.cat([keep[:, 1:], torch.zeros_like(keep[:, :1])], 1)
    lam = _doubling(later.flip(1), dh.flip(1)).flip(1)
    prev = torch.cat([s["h0"].unsqueeze(1), h[:, :-1]], 1)
    if s["starts"] is not None:
        prev = torch.where(s["starts"].unsqueeze(-1), 0.0, prev)
    return {"h": h.to(t), "last": h[:, -1].clone(), "dx": (lam * b).to(t),
            "dgate": (lam * (prev - x) * a * b).to(t), "dh0": lam[:, 0] * keep[:, 0]}


def _plain_scan_step(s):
    x, gate = s["x"].float(), s["gate"].float()
    state = torch.sigmoid(gate) * s["h0"] + torch.sigmoid(-gate) * x
    return {"h": state.to(s["x"].dtype), "state": state}


def _plain_distill(s):
    logits, ids, tau = s["logits"], s["teacher_ids"], s["temperature"]
    rows = logits.shape[0]
    z = logits.float() / tau
    z = z - z.amax(-1, keepdim=True)
    e = z.exp()
    total = e.sum(-1, keepdim=True)
    there = ids >= 0
    at = ids.clamp(min=0)
    tz = torch.where(there, s["teacher_logits"].float() / tau, -torch.inf)
    best = tz.amax(-1, keepdim=True)
    tz = tz - torch.where(best == -torch.inf, 0.0, best)
    te = tz.exp()
    tsum = te.sum(-1, keepdim=True)
    some = tsum > 0
    p = torch.where(some, te / tsum, 0.0)
    gap = (tz - tsum.log()) - (z.gather(1, at) - total.log())
    loss = torch.where(p > 0, p * gap, 0.0).sum() * (tau * tau / rows)
    grad = torch.where(some, e / total, 0.0)
    grad.scatter_add_(1, at, -p)
    return {"loss": loss, "dlogits": (grad * (tau / rows)).to(logits.dtype)}


def _plain_verify(s):
    target, draft, tokens, lengths = s["target"], s["draft"], s["tokens"], s["lengths"]
    batch, drafted, vocab = draft.shape
    place = torch.arange(drafted, device=tokens.device)
    p = target[:, :drafted].gather(2, tokens.unsqueeze(-1)).squeeze(-1)
    q = draft.gather(2, tokens.unsqueeze(-1)).squeeze(-1)
    fine = (s["uniform"] * q < p) & (place < lengths.unsqueeze(-1))
    accepted = fine.long().cumprod(-1).sum(-1)
    each = torch.arange(batch, device=tokens.device)
    p = target[each, accepted]
    q = torch.where((accepted < lengths).unsqueeze(-1), draft[each, accepted.clamp(max=drafted - 1)], 0.0)
    left = (p - q).clamp(min=0)
    left = torch.where(left.amax(-1, keepdim=True) > 0, left, p)
    following = (left / s["race"]).argmax(-1)
    wide = torch.arange(drafted + 1, device=tokens.device)
    padded = torch.cat([tokens, tokens[:, :1]], 1)
    at = accepted.unsqueeze(-1)
    return {"tokens": torch.where(wide < at, padded, torch.where(wide == at, following.unsqueeze(-1), -1)),
            "accepted": accepted}


_OWN = {"norm train": _own_norm_train, "norm quant": _own_norm_quant, "scan train": _own_scan_train,
        "scan forward": _own_scan_forward, "scan step": _own_scan_step, "distill train": _own_distill,
        "verify serve": _own_verify}
_PLAIN = {"norm train": _plain_norm_train, "norm quant": _plain_norm_quant, "scan train": _plain_scan_train,
          "scan forward": _plain_scan_forward, "scan step": _plain_scan_step, "distill train": _plain_distill,
          "verify serve": _plain_verify}


# ---- what a pass cannot do without -----------------------------------------------------

def work(case):
    """Each input read once, each output written once; an operation for every add, product and exponential."""
    op, what = case["op"], case["what"]
    if op == "norm":
        n, w = case["rows"] * case["cols"], SIZE[case["dtype"]]
        if what == "quant":  # x, residual -> r, q, scales
            return {"bytes": n * (w + 4 + 4 + 1) + n // 32 + 4 * case["cols"], "flops": 8 * n}
        # forward x, residual -> r, y; VJP r, dy, dr -> dresidual and, in 16 bits, dx of its own
        return {"bytes": n * (w + 4 + 4 + w) + n * (4 + w + 4 + 4 + (w if w == 2 else 0)) + 8 * case["cols"],
                "flops": 18 * n}
    if op == "scan":
        n, w = case["batch"] * case["length"] * case["dim"], SIZE[case["dtype"]]
        ends = 4 * case["batch"] * case["dim"]
        marks = case["batch"] * case["length"] if case["packed"] else 0
        if what == "train":  # x, gate -> h; x, gate, dh -> dx, dgate
            return {"bytes": 8 * n * w + 4 * ends + 2 * marks, "flops": 24 * n}
        return {"bytes": 3 * n * w + 2 * ends + marks, "flops": 8 * n}
    if op == "distill":  # logits -> dlogits, the loss
        n, k = case["rows"] * case["vocab"], case["rows"] * case["top"]
        return {"bytes": 2 * n * SIZE[case["dtype"]] + 12 * k, "flops": 5 * n}
    # a row of the target's, one of the draft's and one of the race for each sequence
    return {"bytes": 12 * case["batch"] * case["vocab"], "flops": 3 * case["batch"] * case["vocab"]}


# ---- in 64 bits ------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "norm":
            return _exact_norm(s)
        if case["op"] == "scan":
            return _exact_scan(s)
        if case["op"] == "distill":
            return _exact_distill(s)
    return None  # whole numbers only


def _exact_norm(s):
    r = s["x"].double() + s["residual"].double()
    cols = r.shape[1]
    size = (r.square().sum(1, keepdim=True) / cols + EPS).sqrt()
    unit = r / size
    y = unit * s["weight"].double()
    if s["what"] == "train":
        dy, dr = s["dy"].double(), s["dr"].double()
        # y_c = w_c r_c / size, d size / d r_j = r_j / (cols size)
        along = (dy * y).sum(1, keepdim=True) / (cols * size)
        d = dr + dy * s["weight"].double() / size - along * unit
        return {"y": y, "r": r, "dx": d, "dresidual": d, "dweight": (dy * unit).sum(0)}
    parts = y.split(128, 1)
    scale = torch.stack([v.abs().amax(1) for v in parts], 1) / 448
    q = torch.cat([_e4m3(v / scale[:, i:i + 1]) for i, v in enumerate(parts)], 1)
    return {"q": q, "scale": scale, "r": r}


def _e4m3(v):
    """The nearest value with 4 bits of mantissa and an exponent of at least -6, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0**-6))) - 3)
    return torch.round(v / step) * step


def _exact_scan(s):
    x, gate = s["x"].double(), s["gate"].double()
    h = s["h0"].double()
    if s["what"] == "step":
        h = (h + torch.exp(-gate) * x) / (1 + torch.exp(-gate))
        return {"h": h, "state": h}
    batch, length, dim = x.shape
    a = 1 / (1 + torch.exp(-gate))
    b = 1 / (1 + torch.exp(gate))
    keep = a.clone()
    if s["starts"] is not None:
        keep[s["starts"]] = 0.0
    v = b * x
    before, out = torch.empty_like(x), torch.empty_like(x)
    for t in range(length):
        before[:, t] = h
        h = torch.addcmul(v[:, t], keep[:, t], h)
        out[:, t] = h
    if s["what"] == "forward":
        return {"h": out, "last": h}
    lam, carry = s["dh"].double(), s["dlast"].double()
    for t in range(length - 1, -1, -1):
        lam[:, t] += carry
        carry = keep[:, t] * lam[:, t]
    if s["starts"] is not None:
        before[s["starts"]] = 0.0
    return {"h": out, "last": h, "dx": lam * b, "dgate": lam * (before - x) * a * b, "dh0": carry}


def _exact_distill(s):
    tau, ids = s["temperature"], s["teacher_ids"]
    logits = s["logits"].detach().double() / tau
    rows = logits.shape[0]
    log_q = logits - torch.logsumexp(logits, 1, keepdim=True)
    del logits
    there = ids >= 0
    some = there.any(1, keepdim=True)
    teacher = s["teacher_logits"].double() / tau
    teacher = teacher.masked_fill(~there, -torch.inf)
    log_p = teacher - torch.logsumexp(teacher.masked_fill(~some, 0.0), 1, keepdim=True)
    log_p = log_p.masked_fill(~there, -torch.inf)
    p = log_p.exp()
    gap = (log_p - log_q.gather(1, ids.clamp(min=0))).masked_fill(~there, 0.0)
    loss = (p * gap).sum() * tau**2 / rows
    grad = log_q.exp_().mul_(some)
    grad.scatter_add_(1, ids.clamp(min=0), -p)
    return {"loss": loss, "dlogits": grad.mul_(tau / rows)}
