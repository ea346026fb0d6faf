"""The operators of a selective state space model in 64 bits, from their
definitions, and bounds for what f32 arithmetic may be off by (as in
draft_reference.py: each operation's error is carried along with its magnitude;
constants are counts of roundings of 2^-24).

Inputs are numpy arrays of any float type; everything is computed in float64."""

import numpy as np

EPS = 2.0 ** -24


def f64(a):
    return None if a is None else np.asarray(a, dtype=np.float64)


def sigmoid(v):
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-f64(v)))


def softplus(v):
    return np.logaddexp(f64(v), 0.0)


# ---- causal_conv -----------------------------------------------------------------

def _taps(x, x0, starts, width):
    """taps[k]: the input k tokens before each token, zero before its sequence."""
    x = f64(x)
    B, T, D = x.shape
    before = np.zeros((B, width - 1, D)) if x0 is None else f64(x0)
    wide = np.concatenate([before, x], 1)
    reach = np.ones((width, B, T), bool)
    if starts is not None:
        s = np.asarray(starts).astype(bool)
        for k in range(1, width):  # not over a start at t - k + 1 .. t
            for j in range(min(k, T)):
                reach[k, :, j:] &= ~s[:, :T - j]
    taps = [np.where(reach[k][..., None], wide[:, width - 1 - k:width - 1 - k + T], 0.0) for k in range(width)]
    kept = np.ones((B, width - 1), bool)
    if starts is not None:
        for i in range(width - 1):  # token T - (width - 1) + i
            t = T - (width - 1) + i
            kept[:, i] = ~s[:, max(t + 1, 0):].any(1)
    last = np.where(kept[..., None], wide[:, T:], 0.0)
    return taps, reach, last, kept


def causal_conv(x, w, bias=None, x0=None, starts=None, silu=True):
    """(y, last, y_bound)."""
    w = f64(w)
    width = w.shape[1]
    taps, _, last, _ = _taps(x, x0, starts, width)
    b = 0.0 if bias is None else f64(bias)
    u = b + sum(w[:, width - 1 - k] * v for k, v in enumerate(taps))
    size = np.abs(b) + sum(np.abs(w[:, width - 1 - k] * v) for k, v in enumerate(taps))
    bound = EPS * (width + 2) * size
    if not silu:
        return u, last, bound
    y = u * sigmoid(u)
    # |silu'| < 1.1; the sigmoid's exponential is 8 + 2 |u| roundings off
    return y, last, 1.1 * bound + EPS * np.abs(y) * (16 + 4 * np.abs(u))


def causal_conv_grad(x, w, bias, x0, starts, silu, dy, dlast):
    """(dx, dw, dbias, dx0) and their bounds."""
    w = f64(w)
    D, width = w.shape
    taps, reach, _, kept = _taps(x, x0, starts, width)
    B, T = taps[0].shape[:2]
    b = 0.0 if bias is None else f64(bias)
    u = b + sum(w[:, width - 1 - k] * v for k, v in enumerate(taps))
    bu = EPS * (width + 2) * (np.abs(b) + sum(np.abs(w[:, width - 1 - k] * v) for k, v in enumerate(taps)))
    g = np.zeros((B, T, D)) if dy is None else f64(dy)
    if silu:
        s = sigmoid(u)
        du = g * (s + u * s * (1 - s))
        # |silu''| <= 1/2; both terms of the derivative by themselves
        bdu = np.abs(g) * (0.5 * bu + EPS * (24 + 4 * np.abs(u)) * (s + np.abs(u) * s))
    else:
        du, bdu = g, np.zeros_like(g)
    dwide, bwide = np.zeros((B, T + width - 1, D)), np.zeros((B, T + width - 1, D))
    dw, bw = np.zeros((D, width)), np.zeros((D, width))
    # a run of 64 tokens in a row, the 8 warps of a CTA, then the CTAs' sums
    order = 80 + B * (T // 256 + 1)
    for k in range(width):
        wk, there = w[:, width - 1 - k], reach[k][..., None]
        part = np.where(there, du * wk, 0.0)
        dwide[:, width - 1 - k:width - 1 - k + T] += part
        bwide[:, width - 1 - k:width - 1 - k + T] += np.where(there, np.abs(wk) * bdu, 0.0) + EPS * (width + 2) * np.abs(part)
        dw[:, width - 1 - k] = (du * taps[k]).sum((0, 1))
        bw[:, width - 1 - k] = (bdu * np.abs(taps[k]) + EPS * order * np.abs(du * taps[k])).sum((0, 1))
    if dlast is not None:
        add = np.where(kept[..., None], f64(dlast), 0.0)
        dwide[:, T:] += add
        bwide[:, T:] += 2 * EPS * (np.abs(add) + np.abs(dwide[:, T:]))
    db, bb = du.sum((0, 1)), (bdu + EPS * order * np.abs(du)).sum((0, 1))
    n = width - 1
    return (dwide[:, n:], dw, db, dwide[:, :n]), (bwide[:, n:], bw, bb, bwide[:, :n])


# ---- selective_scan --------------------------------------------------------------

class Scan:
    """The recurrence with its states, their magnitudes (m) and error bounds (e)."""

    def __init__(self, x, delta, A, B, C, D=None, z=None, delta_bias=None, h0=None, starts=None):
        self.x, self.A, self.B, self.C = f64(x), f64(A), f64(B), f64(C)
        b, T, d = self.x.shape
        n = self.A.shape[1]
        self.raw = f64(delta) + (0.0 if delta_bias is None else f64(delta_bias))
        self.dt = softplus(self.raw)
        # relative: the sum raw is |raw| roundings off in the exponential, which with
        # the logarithm after it takes 8 more
        self.edt = EPS * (np.abs(self.raw) + 10)
        self.D = np.zeros(d) if D is None else f64(D)
        self.z = None if z is None else f64(z)
        # decays: 4 roundings of the exponential, and those of dt in its argument; a
        # segment's decay is taken from a sum of up to T steps
        with np.errstate(over="ignore"):
            self.a = np.exp(self.dt[..., None] * self.A)
        self.ea = EPS * 8 + self.dt[..., None] * np.abs(self.A) * (self.edt[..., None] + EPS * (4 + T))
        self.new = np.zeros((b, T), bool) if starts is None else np.asarray(starts).astype(bool)
        self.first = np.zeros((b, d, n)) if h0 is None else f64(h0)
        s, m, e = self.first, np.abs(self.first), np.zeros((b, d, n))
        self.h, self.m, self.e = (np.empty((b, T, d, n)) for _ in range(3))
        self.dtx = self.dt * self.x
        for t in range(T):
            new = self.new[:, t, None, None]
            s, m, e = (np.where(new, 0.0, v) for v in (s, m, e))
            u = self.dtx[:, t, :, None] * self.B[:, t, None, :]
            a, ea = np.where(new, 0.0, self.a[:, t]), self.ea[:, t]
            e = a * e + a * m * ea + 2 * EPS * (a * m + np.abs(u)) + np.abs(u) * (self.edt[:, t, :, None] + 2 * EPS)
            s, m = a * s + u, a * m + np.abs(u)
            self.h[:, t], self.m[:, t], self.e[:, t] = s, m, e
        self.last, self.last_bound = s, e
        c = self.C[:, :, None, :]
        self.inner = (self.h * c).sum(-1) + self.D * self.x
        self.inner_size = (self.m * np.abs(c)).sum(-1) + np.abs(self.D * self.x)
        self.inner_bound = (self.e * np.abs(c)).sum(-1) + EPS * (n + 4) * self.inner_size

    def out(self):
        """(y, y_bound)."""
        if self.z is None:
            return self.inner, self.inner_bound
        g = self.z * sigmoid(self.z)
        return self.inner * g, np.abs(g) * (self.inner_bound + EPS * (18 + 4 * np.abs(self.z)) * self.inner_size)

    def grad(self, dy, dlast):
        """dicts of the gradients and of their bounds, by argument."""
        b, T, d, n = self.h.shape
        got, bound = {}, {}
        g = np.zeros((b, T, d)) if dy is None else f64(dy)
        e, be = g, np.zeros_like(g)
        if self.z is not None:
            s = sigmoid(self.z)
            slope = s + self.z * s * (1 - s)
            got["z"] = g * self.inner * slope
            bound["z"] = np.abs(g) * (np.abs(slope) * self.inner_bound + self.inner_size *
                                      EPS * (28 + 4 * np.abs(self.z)) * (s + np.abs(self.z) * s))
            e = g * self.z * s
            be = EPS * (18 + 4 * np.abs(self.z)) * np.abs(e)
        mu = np.zeros((b, d, n)) if dlast is None else f64(dlast)
        mm, emu = np.abs(mu), np.zeros((b, d, n))
        names = ("x", "delta", "B", "C")
        shapes = ((b, T, d), (b, T, d), (b, T, n), (b, T, n))
        for k, shape in zip(names, shapes):
            got[k], bound[k] = np.empty(shape), np.empty(shape)
        got["A"], bound["A"] = np.zeros((d, n)), np.zeros((d, n))
        sig = sigmoid(self.raw)
        across = 40 + d // 16  # roundings of a sum over channels: lanes, warps, tiles
        for t in range(T - 1, -1, -1):
            new = self.new[:, t, None, None]
            Bt, Ct = self.B[:, t, None, :], self.C[:, t, None, :]
            if t == 0:
                h, mh, eh = self.first, np.abs(self.first), np.zeros((b, d, n))
            else:
                h, mh, eh = self.h[:, t - 1], self.m[:, t - 1], self.e[:, t - 1]
            et, bet = e[:, t, :, None], be[:, t, :, None]
            dt, edt = self.dt[:, t, :, None], self.edt[:, t, :, None]
            dtx = self.dtx[:, t, :, None]
            lam, ml = Ct * et + mu, np.abs(Ct * et) + mm
            el = emu + np.abs(Ct) * bet + 2 * EPS * ml
            mh_t, eh_t = self.m[:, t], self.e[:, t]
            got["C"][:, t] = (self.h[:, t] * et).sum(1)
            bound["C"][:, t] = (eh_t * np.abs(et) + mh_t * (bet + EPS * across * np.abs(et))).sum(1)
            got["B"][:, t] = (lam * dtx).sum(1)
            bound["B"][:, t] = (el * np.abs(dtx) + ml * np.abs(dtx) * (edt + EPS * across)).sum(1)
            through, size = (lam * Bt).sum(-1), (ml * np.abs(Bt)).sum(-1)
            bthrough = (el * np.abs(Bt)).sum(-1) + EPS * (n + 4) * size
            a = np.where(new, 0.0, self.a[:, t])
            mu, mm, emu = a * lam, a * ml, a * el + a * ml * (self.ea[:, t] + 2 * EPS)
            q, mq = mu * h, mm * mh
            bq = emu * mh + mm * eh + 2 * EPS * mq
            rate = (q * self.A).sum(-1)
            brate = (bq * np.abs(self.A)).sum(-1) + EPS * (n + 8) * (mq * np.abs(self.A)).sum(-1)
            xt, dt1, skip = self.x[:, t], self.dt[:, t], self.D
            got["x"][:, t] = dt1 * through + skip * e[:, t]
            bound["x"][:, t] = dt1 * (bthrough + (self.edt[:, t] + 4 * EPS) * size) + np.abs(skip) * (
                be[:, t] + 4 * EPS * np.abs(e[:, t]))
            ddt = xt * through + rate
            ddt_size = np.abs(xt) * size + (mq * np.abs(self.A)).sum(-1)
            bddt = np.abs(xt) * bthrough + brate + 4 * EPS * ddt_size
            got["delta"][:, t] = ddt * sig[:, t]
            bound["delta"][:, t] = sig[:, t] * (bddt + EPS * (16 + 6 * np.abs(self.raw[:, t])) * ddt_size)
            got["A"] += (q * dt).sum(0)
            bound["A"] += (bq * dt + mq * dt * (edt + EPS * (T + b + 40))).sum(0)
        got["h0"], bound["h0"] = mu, emu
        sums = EPS * (T + b + 40)  # tokens in a row within a tile and after it, then the rest
        got["D"] = (e * self.x).sum((0, 1))
        bound["D"] = (np.abs(self.x) * (be + sums * np.abs(e))).sum((0, 1))
        got["delta_bias"] = got["delta"].sum((0, 1))
        bound["delta_bias"] = (bound["delta"] + sums * np.abs(got["delta"])).sum((0, 1))
        return got, bound


# ---- policy_loss -----------------------------------------------------------------

def policy(logits, tokens, old, adv, ref=None, clip=(0.2, 0.2), kl=0.0, tau=1.0, total_rows=None):
    """(loss, logp, dlogits) and their bounds, and how far the ratios are from where
    they are clipped (relative to what f32 may be off there)."""
    s, tokens, old, adv = f64(logits), np.asarray(tokens), f64(old), f64(adv)
    n, vocab = s.shape
    total = total_rows or n
    loss, bloss, margin = 0.0, 0.0, np.inf
    logp, blogp = np.zeros(n), np.zeros(n)
    grad, bgrad = np.zeros_like(s), np.zeros_like(s)
    for i in range(n):
        if tokens[i] < 0:
            continue
        at = tokens[i]
        z = (s[i] - s[i].max()) / tau
        q = np.exp(z)
        sum_e = q.sum()
        q = q / sum_e
        fz = np.where(np.isfinite(z), np.abs(z), 0.0)
        # each exponential 4 + 2 |z| roundings, the sum at most 48
        esum = EPS * ((64 + 4 * fz) * q).sum()
        logp[i] = z[at] - np.log(sum_e)
        blogp[i] = esum + EPS * (4 * fz[at] + 4 * np.log(sum_e) + 2)
        gap = logp[i] - old[i]
        r = np.exp(gap)
        er = blogp[i] + EPS * (np.abs(gap) + 4)
        for edge in (1 - clip[0], 1 + clip[1]):
            margin = min(margin, np.abs(r - edge) / (edge * (er + 4 * EPS)) if edge > 0 else np.inf)
        held = np.clip(r, 1 - clip[0], 1 + clip[1]) * adv[i]
        free = r * adv[i]
        term, by = -min(free, held), 0.0 if free > held else -free
        bterm, bby = (er + 4 * EPS) * np.abs(term), (er + 4 * EPS) * np.abs(by)
        if kl > 0:
            gap = f64(ref)[i] - logp[i]
            e = np.expm1(gap)
            bgap = blogp[i] + EPS * np.abs(gap)
            term += kl * (e - gap)
            bterm += kl * (np.abs(e) * bgap + bgap ** 2 + EPS * 6 * (np.abs(e) + np.abs(gap)))
            by -= kl * e
            bby += kl * ((np.abs(e) + 1) * bgap + EPS * 6 * np.abs(e))
        loss += term / total
        bloss += (bterm + 2 * EPS * np.abs(term)) / total
        c = 1 / (total * tau)
        grad[i] = -by * q * c
        grad[i, at] += by * c
        bgrad[i] = q * c * (bby + np.abs(by) * (EPS * (16 + 4 * fz) + esum))
        bgrad[i, at] += c * (bby + 4 * EPS * np.abs(by))
    # values under the smallest normal f32 may be flushed to zero
    return (loss, logp, grad), (bloss + 2 * EPS * abs(loss) + 2.0 ** -126, blogp + EPS * np.abs(logp), bgrad + 2.0 ** -120), margin


# ---- clip_global_norm_ -----------------------------------------------------------

def clip(tensors, max_norm):
    """(norm, clipped): the factor in 64 bits; f32 rounds it and the product."""
    norm = np.sqrt(sum((f64(t) ** 2).sum() for t in tensors))
    factor = max_norm / (norm + 1e-6)
    return norm, [f64(t) * factor if factor < 1 else f64(t) for t in tensors]
