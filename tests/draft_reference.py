"""The recurrent draft model's operators in 64 bits, from their definitions, and
bounds for what f32 arithmetic may be off by.

Inputs are numpy arrays of any float type; everything is computed in float64.
The ``*_bound`` functions give, per output, the largest error that f32
arithmetic with EPS = 2^-24 relative per operation can leave, by carrying each
operation's error along with its magnitude; constants are counts of roundings.
"""

import numpy as np

EPS = 2.0 ** -24
E4M3_MAX = 448.0


def f64(a):
    return None if a is None else np.asarray(a, dtype=np.float64)


# ---- add_rms_norm ----------------------------------------------------------------

def add_rms_norm(x, residual, w, eps):
    """(y, r, inv) over the last axis."""
    r = f64(x) + f64(residual)
    inv = 1.0 / np.sqrt((r * r).mean(-1, keepdims=True) + eps)
    return r * inv * f64(w), r, inv


def add_rms_norm_grad(x, residual, w, eps, dy, dr, exact=True):
    """(dresidual, dw) and their error bounds; dx is dresidual."""
    _, r, inv = add_rms_norm(x, residual, w, eps)
    dy, w = f64(dy), f64(w)
    dr = np.zeros_like(r) if dr is None else f64(dr)
    u, g = r * inv, dy * w
    mean = (g * u).mean(-1, keepdims=True) if exact else 0.0
    mean_abs = np.abs(g * u).mean(-1, keepdims=True) if exact else 0.0
    d = dr + inv * (g - u * mean)
    dw = (dy * u).reshape(-1, r.shape[-1]).sum(0)
    # inv: a sum of cols squares in a tree (at most 32 terms in a row in a
    # thread, then 10 levels), a division, a square root, a reciprocal: 48; the
    # row mean as many again
    bound_d = EPS * (2 * np.abs(dr) + np.abs(inv) * (56 * np.abs(g) + 160 * np.abs(u) * mean_abs))
    rows = dy.size // r.shape[-1]
    # dw: in a row within a CTA (at least 8 rows each, 148 CTAs at least on 148
    # SMs), then the partials
    bound_dw = EPS * (rows / 64 + 128) * np.abs(dy * u).reshape(-1, r.shape[-1]).sum(0)
    return (d, dw), (bound_d, bound_dw)


def e4m3_half_step(v):
    """Half the distance between neighbouring e4m3 values at |v|."""
    return 0.5 * np.exp2(np.floor(np.log2(np.maximum(np.abs(v), 2.0 ** -6))) - 3)


def block_scales(y, block):
    cols = y.shape[-1]
    block = block or cols
    return np.stack([np.maximum(np.abs(y[..., c:c + block]).max(-1) / E4M3_MAX, 2.0 ** -126)
                     for c in range(0, cols, block)], -1)


# ---- gated_scan ------------------------------------------------------------------

def sigmoid_pair(gate):
    g = f64(gate)
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-g)), 1 / (1 + np.exp(g))


def gated_scan(x, gate, h0=None, starts=None):
    """(h, last, h_bound): [batch, length, dim] by the recurrence itself."""
    x = f64(x)
    B, T, D = x.shape
    a, b = sigmoid_pair(gate)
    s = np.zeros((B, D)) if h0 is None else f64(h0).copy()
    m, e = np.abs(s), np.zeros((B, D))
    h, bound = np.empty_like(x), np.empty_like(x)
    for t in range(T):
        if starts is not None:
            new = np.asarray(starts)[:, t].astype(bool)
            s, m, e = (np.where(new[:, None], 0.0, v) for v in (s, m, e))
        # a and b are 4 roundings off, their products and the sum 2 more; the
        # same again for a chunk's product of gates applied to its first state
        e = a[:, t] * e + 12 * EPS * (a[:, t] * m + b[:, t] * np.abs(x[:, t]))
        m = a[:, t] * m + b[:, t] * np.abs(x[:, t])
        s = a[:, t] * s + b[:, t] * x[:, t]
        h[:, t], bound[:, t] = s, e
    return h, s, bound


def gated_scan_grad(x, gate, h0, starts, dh, dlast):
    """(dx, dgate, dh0) and their error bounds."""
    x = f64(x)
    B, T, D = x.shape
    a, b = sigmoid_pair(gate)
    h, _, eh = gated_scan(x, gate, h0, starts)
    mu = np.zeros((B, D)) if dlast is None else f64(dlast).copy()
    m, e = np.abs(mu), np.zeros((B, D))
    dx, dg = np.empty_like(x), np.empty_like(x)
    bx, bg = np.empty_like(x), np.empty_like(x)
    for t in range(T - 1, -1, -1):
        new = None if starts is None else np.asarray(starts)[:, t].astype(bool)[:, None]
        before = (np.zeros((B, D)) if h0 is None else f64(h0)) if t == 0 else h[:, t - 1]
        eb = np.zeros((B, D)) if t == 0 else eh[:, t - 1]
        if new is not None:
            before, eb = np.where(new, 0.0, before), np.where(new, 0.0, eb)
        g = 0.0 if dh is None else f64(dh)[:, t]
        lam, ml = g + mu, np.abs(g) + m
        el = e + EPS * ml
        ab = a[:, t] * b[:, t]
        dx[:, t], dg[:, t] = lam * b[:, t], lam * (before - x[:, t]) * ab
        bx[:, t] = b[:, t] * el + 8 * EPS * b[:, t] * ml
        gap = np.abs(before) + np.abs(x[:, t])
        bg[:, t] = ab * (el * gap + ml * eb + 16 * EPS * ml * gap)
        mu, m = a[:, t] * lam, a[:, t] * ml
        e = a[:, t] * el + 12 * EPS * m
        if new is not None:
            mu, m, e = (np.where(new, 0.0, v) for v in (mu, m, e))
    return (dx, dg, mu), (bx, bg, e)


# ---- distill_loss ----------------------------------------------------------------

def distill(logits, teacher, ids, tau, total_rows=None):
    """(loss, dlogits, loss_bound, dlogits_bound)."""
    s, ids = f64(logits), np.asarray(ids)
    n, vocab = s.shape
    total = total_rows or n
    loss, grad, bound, grad_bound = 0.0, np.zeros_like(s), 0.0, np.zeros_like(s)
    for i in range(n):
        k = (ids[i] >= 0) & (f64(teacher[i]) > -np.inf)
        if not k.any():
            continue
        at, t = ids[i][k], f64(teacher[i])[k] / tau
        tz = t - t.max()
        p = np.exp(tz) / np.exp(tz).sum()
        z = (s[i] - s[i].max()) / tau
        sum_e = np.exp(z).sum()
        q = np.exp(z) / sum_e
        with np.errstate(divide="ignore", invalid="ignore"):
            terms = np.where(p > 0, p * ((tz - np.log(np.exp(tz).sum())) - (z[at] - np.log(sum_e))), 0.0)
        loss += terms.sum()
        grad[i] = q
        np.add.at(grad[i], at, -p)
        # an exponential of z costs 4 + 2 |z| roundings (its argument's included),
        # the sums at most 48, each product and logarithm a few
        fz = np.where(np.isfinite(z), np.abs(z), 0.0)
        cost_p = 64 + 4 * np.abs(np.maximum(tz, -1e3))
        bound += EPS * (p * cost_p * (np.abs(np.maximum(tz, -1e3)) + fz[at] + np.log(sum_e) + 1)).sum()
        grad_bound[i] = EPS * q * (64 + 4 * fz)
        np.add.at(grad_bound[i], at, EPS * p * cost_p)
    c = tau / total
    # values under the smallest normal f32 may be flushed to zero
    return (loss * tau * tau / total, grad * c, bound * tau * tau / total + 2.0 ** -126,
            grad_bound * c + 2.0 ** -120)


# ---- verify_draft -----------------------------------------------------------------

def verify(target, draft, tokens, uniform, race, lengths=None):
    """(out, accepted), each comparison and quotient in f32 as defined."""
    target, race = np.asarray(target, np.float32), np.asarray(race, np.float32)
    B, K = tokens.shape
    out, accepted = np.full((B, K + 1), -1, np.int64), np.zeros(B, np.int64)
    for b in range(B):
        n = K if lengths is None else min(max(int(lengths[b]), 0), K)
        j = 0
        while j < n:
            x = int(tokens[b, j])
            if not 0 <= x < target.shape[2]:
                break
            q = np.float32(1.0) if draft is None else draft[b, j, x]
            if not np.float32(uniform[b, j] * q) < target[b, j, x]:
                break
            out[b, j] = x
            j += 1
        p = target[b, j]
        w = p.copy()
        if j < n:
            if draft is None:
                if 0 <= tokens[b, j] < len(w):
                    w[tokens[b, j]] = 0.0
            else:
                w = p - draft[b, j]
        for weights in (w, p):
            with np.errstate(divide="ignore", invalid="ignore"):
                score = np.where(weights > 0, weights / race[b], -1.0)
            score = np.where(np.isnan(score), -1.0, score)
            if score.max() >= 0:
                out[b, j] = int(score.argmax())
                break
        accepted[b] = j
    return out, accepted
