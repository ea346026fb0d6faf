"""The operators of a selective state space model on the device against their
64-bit references (tests/selective_reference.py).

Tolerances come with the references: per element, the magnitude-weighted count of
f32 roundings; a bfloat16 result may be off by half a unit in its last place (2^-8
of the value) on top."""

import numpy as np
import pytest

import selective_reference as R
from test_gpu_draft import DTYPES, _check, _n, _t

pytestmark = pytest.mark.gpu


# ---- causal_conv --------------------------------------------------------------------

CONV_SHAPES = [(1, 1, 1, 1), (1, 1, 4, 4), (2, 2, 5, 4), (3, 3, 4, 8), (1, 64, 128, 4), (2, 65, 130, 3), (1, 61, 8, 4),
               (2, 600, 36, 4), (1, 517, 7, 2), (3, 70, 256, 5), (2, 129, 12, 6), (1, 130, 64, 7), (2, 1000, 1, 4)]


def _conv_inputs(B, T, D, W, dtype, packed, seed=0):
    g = np.random.default_rng([B, T, D, W, seed])
    n = lambda *s, scale=1.0: scale * g.standard_normal(s)  # noqa: E731
    starts = g.random((B, T)) < 0.2 if packed else None
    return (_t(n(B, T, D), dtype), _t(n(D, W)), _t(n(D)), _t(n(B, W - 1, D), dtype), starts,
            _t(n(B, T, D), dtype), _t(n(B, W - 1, D), dtype))


def _starts(starts):
    import torch
    return None if starts is None else torch.from_numpy(starts).cuda()


def _conv_check(x, w, bias, x0, starts, dy, dlast, activation="silu"):
    import torch
    from oxitorch_b200 import functional as F
    leaves = [t for t in (x, w, bias, x0) if t is not None]
    for t in leaves:
        t.requires_grad_()
    y, last = F.causal_conv(x, w, bias, x0, _starts(starts), activation=activation)
    ref = (_n(x), _n(w), None if bias is None else _n(bias), None if x0 is None else _n(x0), starts)
    want, want_last, bound = R.causal_conv(*ref, silu=activation == "silu")
    _check(y, want, bound, "y")
    np.testing.assert_array_equal(_n(last), want_last)
    outs = [(o, d) for o, d in ((y, dy), (last, dlast)) if d is not None]
    got = torch.autograd.grad([o for o, _ in outs], leaves, [d for _, d in outs])
    want, bounds = R.causal_conv_grad(*ref, activation == "silu", None if dy is None else _n(dy),
                                      None if dlast is None else _n(dlast))
    names = [k for k, t in zip(("dx", "dw", "dbias", "dx0"), (x, w, bias, x0)) if t is not None]
    pick = [i for i, t in enumerate((x, w, bias, x0)) if t is not None]
    for k, i, d in zip(names, pick, got):
        _check(d, want[i], bounds[i], k)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,D,W", CONV_SHAPES)
def test_causal_conv(B, T, D, W, dtype, packed):
    _conv_check(*_conv_inputs(B, T, D, W, dtype, packed))


@pytest.mark.parametrize("dtype", DTYPES)
def test_causal_conv_without_its_options(dtype):
    x, w, bias, x0, starts, dy, dlast = _conv_inputs(2, 70, 20, 4, dtype, True)
    _conv_check(x.clone(), w.clone(), None, None, None, dy, None)
    _conv_check(x.clone(), w.clone(), bias.clone(), None, starts, dy, dlast, activation=None)
    _conv_check(x.clone(), w.clone(), None, x0.clone(), starts, None, dlast)


@pytest.mark.parametrize("D", [3052, 1510])
def test_causal_conv_of_long_runs(D):
    """As many tokens as fill the GPU with long runs a warp, against 64 bits on the device.
    With m = |bias| + sum |w x|: u is off by 5 roundings of m, and SiLU and its derivative,
    whose slopes are below 1.1 and 0.5, by 2^-21 more from ex2 and the reciprocal: 2^-20
    (1 + m) together.  A weight's sum adds up to 256 terms of a run, then 20 partial sums."""
    import torch
    from oxitorch_b200 import functional as F
    T, W = 24000, 4
    g = torch.Generator(device="cuda").manual_seed(D)
    x, dy = (torch.randn(1, T, D, device="cuda", generator=g) for _ in range(2))
    w, bias = torch.randn(D, W, device="cuda", generator=g), torch.randn(D, device="cuda", generator=g)
    y, _ = F.causal_conv_fwd(x, w, bias)
    dx, dw, db, _ = F.causal_conv_bwd(x, w, bias, None, dy)
    pad = torch.nn.functional.pad(x[0].double(), (0, 0, W - 1, 0))
    wd, d = w.double(), dy[0].double()
    u = bias.double() + sum(wd[:, k] * pad[k:k + T] for k in range(W))
    m = bias.double().abs() + sum((wd[:, k] * pad[k:k + T]).abs() for k in range(W))
    s = torch.sigmoid(u)
    assert ((y[0] - u * s).abs() <= 2.0 ** -20 * (1 + m)).all()
    du, mag = d * (s + u * s * (1 - s)), d.abs() * (1 + m)
    later = lambda t: torch.nn.functional.pad(t, (0, 0, 0, W - 1))  # noqa: E731
    dus, mags = later(du), later(mag)
    want = sum(wd[:, W - 1 - k] * dus[k:k + T] for k in range(W))
    size = sum((wd[:, W - 1 - k] * mags[k:k + T]).abs() for k in range(W))
    assert ((dx[0] - want).abs() <= 2.0 ** -19 * size).all()
    for k in range(W):
        tap = pad[k:k + T]
        assert ((dw[:, k] - (du * tap).sum(0)).abs() <= 2.0 ** -15 * (mag * tap.abs()).sum(0)).all()
    assert ((db - du.sum(0)).abs() <= 2.0 ** -15 * mag.sum(0)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [0, 1, 4])
def test_causal_conv_reads_parts_of_a_projection(dtype, offset):
    """x, dy and the weights as views: rows that start anywhere, weights transposed."""
    import torch
    g = np.random.default_rng(offset)
    wide = _t(g.standard_normal((2, 90, 64)), dtype)
    x = wide[..., offset:offset + 24]
    dy = _t(g.standard_normal((90, 2, 40)), dtype).transpose(0, 1)[..., 8:32]
    w = _t(g.standard_normal((4, 24))).t()
    starts = g.random((2, 90)) < 0.1
    _conv_check(x, w, _t(g.standard_normal(48))[::2], _t(g.standard_normal((3, 2, 24)), dtype).transpose(0, 1), starts,
                dy, None)
    assert torch.isfinite(wide).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_causal_conv_starts_stop_nan_and_infinity(dtype, poison):
    """Sequences before and after the poisoned one have the values they have alone."""
    import torch
    from oxitorch_b200 import functional as F
    g = np.random.default_rng(11)
    x, w = _t(g.standard_normal((1, 150, 40)), dtype), _t(g.standard_normal((40, 4)))
    dy = _t(g.standard_normal((1, 150, 40)), dtype)
    starts = torch.zeros(1, 150, dtype=torch.bool, device="cuda")
    starts[0, 60], starts[0, 63] = True, True
    bad = x.clone()
    bad[0, 60:63] = poison
    good, hurt = x.clone().requires_grad_(), bad.requires_grad_()
    y, last = F.causal_conv(good, w, None, None, starts)
    yb, lastb = F.causal_conv(hurt, w, None, None, starts)
    (d,) = torch.autograd.grad(y, good, dy)
    (db,) = torch.autograd.grad(yb, hurt, dy)
    keep = torch.ones(150, dtype=torch.bool, device="cuda")
    keep[60:63] = False
    assert torch.equal(y[:, keep], yb[:, keep]) and torch.equal(d[:, keep], db[:, keep]) and torch.equal(last, lastb)


def test_causal_conv_continues_a_row():
    """Rows cut in pieces of any length, each after the one before it, and token by token."""
    import torch
    from oxitorch_b200 import functional as F
    x, w, bias, x0, _, _, _ = _conv_inputs(2, 200, 24, 4, "bfloat16", False)
    whole, last = F.causal_conv(x, w, bias, x0)
    for cuts in ((0, 1, 2, 5, 70, 200), (0, 64, 65, 200)):
        kept, parts = x0, []
        for lo, hi in zip(cuts, cuts[1:]):
            y, kept = F.causal_conv(x[:, lo:hi], w, bias, kept)
            parts.append(y)
        assert torch.equal(torch.cat(parts, 1), whole) and torch.equal(kept, last)
    state, other = x0.clone(), torch.empty_like(x0)
    for t in range(20):
        if t % 2:
            y = F.causal_conv_step(x[:, t], w, bias, state, out=other)
            state, other = other, state
        else:
            y = F.causal_conv_step(x[:, t], w, bias, state)
        assert torch.equal(y, whole[:, t])
    assert torch.equal(state, x[:, 17:20])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,D,W", [(1, 1, 1), (3, 130, 2), (8, 4096, 4), (300, 33, 8)])
def test_causal_conv_step(B, D, W, dtype):
    from oxitorch_b200 import functional as F
    x, w, bias, x0, _, _, _ = _conv_inputs(B, 1, D, W, dtype, False)
    after = x0.clone()
    y = F.causal_conv_step(x[:, 0], w, None, x0, out=after, activation=None)
    want, last, bound = R.causal_conv(_n(x), _n(w), None, _n(x0), silu=False)
    _check(y, want[:, 0], bound[:, 0], "y")
    np.testing.assert_array_equal(_n(after), last)


def test_causal_conv_empty_and_refusals():
    import torch
    from oxitorch_b200 import functional as F
    x, w, bias, x0, _, dy, dlast = _conv_inputs(2, 0, 6, 4, "float32", False)
    x.requires_grad_()
    x0.requires_grad_()
    y, last = F.causal_conv(x, w, bias, x0)
    assert y.shape == (2, 0, 6) and torch.equal(last, x0)
    dx, dx0 = torch.autograd.grad((y, last), (x, x0), (dy, dlast))
    assert dx.shape == (2, 0, 6) and torch.equal(dx0, dlast)
    y, last = F.causal_conv(torch.empty(0, 3, 6, device="cuda"), w)
    assert y.shape == (0, 3, 6) and last.shape == (0, 3, 6)
    dx, dw, db, _ = F.causal_conv_bwd(torch.empty(0, 3, 6, device="cuda"), w, dy=torch.empty(0, 3, 6, device="cuda"))
    assert not dw.any() and not db.any() and dw.shape == (6, 4)
    x = torch.zeros(2, 5, 6, device="cuda")
    for bad in (dict(x=x[0]), dict(x=x.half()), dict(x=x.cpu()), dict(weight=w[:5]), dict(weight=w.bfloat16()),
                dict(weight=w[:, :0]), dict(bias=bias[:5]), dict(x0=x0[:, :2].detach()), dict(x0=x0.detach().bfloat16()),
                dict(starts=torch.zeros(2, 4, dtype=torch.bool, device="cuda")), dict(activation="relu")):
        with pytest.raises(ValueError):
            F.causal_conv(**{"x": x, "weight": w, "bias": bias, **bad})
    with pytest.raises(NotImplementedError):
        F.causal_conv(x, torch.zeros(6, 9, device="cuda"))
    state = torch.zeros(2, 3, 6, device="cuda")
    flat = torch.zeros(60, device="cuda")
    for bad in (dict(x=x), dict(state=state[:, :2]), dict(state=state.bfloat16()), dict(out=state[:1]),
                dict(state=flat[:36].view(2, 3, 6), out=flat[6:42].view(2, 3, 6)),
                dict(state=state.transpose(0, 1).contiguous().transpose(0, 1)), dict(x=x[:, 0].clone().requires_grad_())):
        with pytest.raises(ValueError):
            F.causal_conv_step(**{"x": x[:, 0], "weight": w, "bias": bias, "state": state, **bad})


# ---- selective_scan -----------------------------------------------------------------

SCAN_SHAPES = [(1, 1, 1, 1), (2, 5, 3, 4), (1, 16, 7, 16), (2, 17, 130, 16), (1, 100, 33, 24), (3, 40, 64, 10),
               (1, 33, 20, 128), (1, 70, 9, 64), (2, 300, 36, 16), (1, 700, 8, 5), (2, 64, 257, 8), (1, 50, 34, 48),
               (1, 47, 12, 96), (1, 160, 132, 31), (4, 15, 512, 2)]


def _scan_inputs(B, T, D, N, dtype, packed, gated=True, seed=0):
    g = np.random.default_rng([B, T, D, N, seed])
    n = lambda *s, scale=1.0: scale * g.standard_normal(s)  # noqa: E731
    step = np.exp(g.uniform(np.log(0.001), np.log(0.3), D))
    args = {"x": _t(n(B, T, D), dtype), "delta": _t(n(B, T, D, scale=0.7), dtype),
            "A": _t(-np.arange(1, N + 1) * np.exp(n(D, N, scale=0.2))), "B": _t(n(B, T, N), dtype),
            "C": _t(n(B, T, N), dtype), "D": _t(n(D)), "z": _t(n(B, T, D), dtype) if gated else None,
            "delta_bias": _t(np.log(np.expm1(step))), "h0": _t(n(B, D, N))}
    starts = g.random((B, T)) < 0.1 if packed else None
    return args, starts, _t(n(B, T, D), dtype), _t(n(B, D, N))


def _scan_check(args, starts, dy, dlast):
    import torch
    from oxitorch_b200 import functional as F
    leaves = {k: t for k, t in args.items() if t is not None}
    for t in leaves.values():
        t.requires_grad_()
    y, last = F.selective_scan(**args, starts=_starts(starts))
    ref = R.Scan(**{k: None if t is None else _n(t) for k, t in args.items()}, starts=starts)
    _check(y, *ref.out(), "y")
    _check(last, ref.last, ref.last_bound, "last")
    outs = [(o, d) for o, d in ((y, dy), (last, dlast)) if d is not None]
    got = torch.autograd.grad([o for o, _ in outs], list(leaves.values()), [d for _, d in outs])
    want, bounds = ref.grad(None if dy is None else _n(dy), None if dlast is None else _n(dlast))
    for k, d in zip(leaves, got):
        _check(d, want[k], bounds[k], "d" + k)
    with torch.no_grad():  # without what the VJP needs: the same bits
        again = F.selective_scan(**args, starts=_starts(starts))
    assert torch.equal(again[0], y) and torch.equal(again[1], last)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,D,N", SCAN_SHAPES)
def test_selective_scan(B, T, D, N, dtype, packed):
    _scan_check(*_scan_inputs(B, T, D, N, dtype, packed, gated=(T + N) % 2 == 0))


@pytest.mark.parametrize("dtype", DTYPES)
def test_selective_scan_without_its_options(dtype):
    args, starts, dy, dlast = _scan_inputs(2, 130, 20, 16, dtype, True)
    plain = {**args, "D": None, "z": None, "delta_bias": None, "h0": None}
    copy = lambda d: {k: None if t is None else t.clone() for k, t in d.items()}  # noqa: E731
    _scan_check(copy(plain), None, dy, None)
    _scan_check(copy(args), starts, None, dlast)
    _scan_check(copy({**args, "D": None}), None, dy, dlast)
    _scan_check(copy({**args, "h0": None, "delta_bias": None}), starts, dy, dlast)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [0, 1, 4])
def test_selective_scan_reads_parts_of_a_projection(dtype, offset):
    g = np.random.default_rng(offset)
    args, starts, _, dlast = _scan_inputs(2, 90, 24, 16, dtype, True)
    wide = _t(g.standard_normal((2, 90, 120)), dtype)
    args["x"], args["z"] = wide[..., offset:offset + 24], wide[..., offset + 24:offset + 48]
    args["B"], args["C"] = wide[..., offset + 60:offset + 76], wide[..., offset + 77:offset + 93]
    args["delta"] = _t(0.7 * g.standard_normal((90, 2, 40)), dtype).transpose(0, 1)[..., 8:32]
    args["A"] = _t(-g.uniform(0.5, 9.0, (16, 24))).t()
    args["h0"] = _t(g.standard_normal((2, 16, 24))).transpose(1, 2)
    dy = _t(g.standard_normal((2, 90, 25)), dtype)[..., :24]
    _scan_check(args, starts, dy, dlast)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [40, 900])
@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_selective_scan_starts_stop_nan_and_infinity(dtype, poison, T):
    """A poisoned sequence between two others, within a segment and over several."""
    import torch
    from oxitorch_b200 import functional as F
    args, _, dy, _ = _scan_inputs(1, T, 20, 16, dtype, False)
    lo, hi = T // 3, 2 * T // 3
    starts = torch.zeros(1, T, dtype=torch.bool, device="cuda")
    starts[0, lo], starts[0, hi] = True, True
    keep = torch.ones(T, dtype=torch.bool, device="cuda")
    keep[lo:hi] = False
    found = []
    for bad in (False, True):
        a = {k: t.clone() for k, t in args.items()}
        if bad:
            a["x"][0, lo + 1], a["B"][0, lo + 2] = poison, poison
        leaves = [a[k].requires_grad_() for k in ("x", "delta", "B", "C", "h0")]
        y, last = F.selective_scan(**a, starts=starts)
        got = torch.autograd.grad((y, last), leaves, (dy, torch.ones_like(last)))
        found.append([y[:, keep], last, *(d[:, keep] for d in got[:4]), got[4]])
    for a, b in zip(*found):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_selective_scan_extremes(dtype):
    """Steps of zero and of dozens, rates of zero, states that never decay and ones
    that do at once, over tiles that are not whole."""
    import torch
    from oxitorch_b200 import functional as F
    args, starts, dy, dlast = _scan_inputs(1, 530, 8, 16, dtype, True)
    args["delta"][0, ::3] = -200.0   # a step of 0
    args["delta"][0, 1::50] = 30.0
    args["A"][:, 0] = 0.0
    args["A"][:, 1] = -1e4
    args["A"][:, 2] = -1e-6
    _scan_check(args, starts, dy, dlast)
    args, _, _, _ = _scan_inputs(1, 21, 8, 16, dtype, False)
    args["A"][:, 3] = -float("inf")  # forgets at once, beside padded tokens too
    y, last = F.selective_scan(**args)
    assert torch.isfinite(y).all() and torch.isfinite(last).all()
    ref = R.Scan(**{k: _n(t) for k, t in args.items() if k != "A"}, A=np.maximum(_n(args["A"]), -1e30))
    np.testing.assert_allclose(_n(last), ref.last, rtol=1e-4, atol=1e-4)


def test_selective_scan_grows_over_segments():
    """With rates above zero the decay of a segment is beyond f32 (exp(128) and exp(89)
    here) where the states are not: zero before the last tokens and behind the first
    ones, or tiny.  A step's factor is off by 2^-24 of an exponent of 3 a few times and by
    ex2's 2^-22, over 64 steps by 2^-14."""
    import torch
    from oxitorch_b200 import functional as F
    args, _, dy, _ = _scan_inputs(1, 4096, 8, 4, "float32", False)
    args = {**args, "h0": None, "z": None, "delta_bias": None}
    args["A"].fill_(2.0)
    args["delta"].fill_(float(np.log(np.expm1(1.0))))  # steps of 1
    args["x"][:, :-20] = 0.0
    dy[:, 20:] = 0.0
    leaves = [args[k].requires_grad_() for k in ("x", "delta", "A", "B", "C")]
    y, last = F.selective_scan(**args)
    got = torch.autograd.grad(y, leaves, dy)
    assert not y[:, :-20].any() and torch.isfinite(y).all()
    ref = R.Scan(**{k: None if t is None else _n(t.detach()) for k, t in args.items()})
    _check(last, ref.last, ref.last_bound, "last")
    back = torch.zeros(8, 4, device="cuda", dtype=torch.float64)  # lam_t for t from 19 to 0
    want = torch.zeros(20, 8, device="cuda", dtype=torch.float64)
    B, C = args["B"].detach()[0].double(), args["C"].detach()[0].double()
    for t in range(19, -1, -1):
        back = back * np.exp(2.0) + C[t] * dy[0, t].double()[:, None]
        want[t] = back @ B[t] + args["D"].double() * dy[0, t].double()
    scale = want.abs().max()
    assert (got[0][0, :20] - want).abs().max() <= 2.0 ** -13 * scale and not got[0][:, 20:].any()
    assert not any(g.any() for g in got[1:])

    args = {k: None if t is None else t.detach()[:, :128].contiguous() if t.dim() == 3 else t.detach()
            for k, t in args.items()}
    args["x"].zero_()
    args["A"].fill_(1.39)
    args["delta"][:, 64:] = -200.0  # steps of 0
    args["h0"] = torch.full((1, 8, 4), 1e-37, device="cuda")
    y, last = F.selective_scan(**args)
    want = float(np.float32(1e-37)) * np.exp(64 * float(np.float32(1.39)))
    np.testing.assert_allclose(_n(last), np.full((1, 8, 4), want), rtol=2.0 ** -13)


def test_selective_scan_nan_reaches_all_that_follows():
    import torch
    from oxitorch_b200 import functional as F
    args, _, _, _ = _scan_inputs(1, 600, 4, 4, "float32", False)
    args["x"][0, 100, 2] = float("nan")
    y, last = F.selective_scan(**args)
    bad = torch.isnan(y[0])
    assert not bad[:100].any() and bad[100:, 2].all() and not bad[:, [0, 1, 3]].any()
    assert torch.isnan(last[0, 2]).all() and torch.isfinite(last[0, [0, 1, 3]]).all()


def test_selective_scan_and_conv_offsets_beyond_32_bits():
    import torch
    from oxitorch_b200 import functional as F
    far = 2 ** 31 + 16
    base = torch.empty(far + 64, dtype=torch.bfloat16, device="cuda")
    view = base.as_strided((2, 3, 8), (far, 8, 1))
    args, _, _, _ = _scan_inputs(2, 3, 8, 16, "bfloat16", False)
    want = F.selective_scan(**args)
    view.copy_(args["x"])
    got = F.selective_scan(**{**args, "x": view})
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    w = torch.randn(8, 4, device="cuda")
    assert torch.equal(F.causal_conv(view, w)[0], F.causal_conv(args["x"], w)[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,D,N", [(1, 1, 1), (3, 130, 16), (8, 512, 16), (70, 33, 10), (2, 20, 128), (5, 9, 7)])
def test_selective_step_continues_a_scan(B, D, N, dtype):
    import torch
    from oxitorch_b200 import functional as F
    T = 3
    args, _, _, _ = _scan_inputs(B, T, D, N, dtype, False, gated=N != 10)
    ref = R.Scan(**{k: None if t is None else _n(t) for k, t in args.items()})
    want, bound = ref.out()
    state, other = args.pop("h0"), torch.full((B, D, N), float("nan"), device="cuda")
    small = {k: args[k] for k in ("A", "D", "delta_bias")}
    for t in range(T):
        at = {k: None if args[k] is None else args[k][:, t] for k in ("x", "delta", "B", "C", "z")}
        if t == 1:
            before = state.clone()
            y = F.selective_step(**at, **small, state=state, out=other)
            assert torch.equal(before, state)
            state = other
        else:
            y = F.selective_step(**at, **small, state=state)
        _check(y, want[:, t], bound[:, t], f"y {t}")
        _check(state, ref.h[:, t], ref.e[:, t], f"state {t}")


def test_selective_scan_empty_and_refusals():
    import torch
    from oxitorch_b200 import functional as F
    args, _, dy, dlast = _scan_inputs(2, 0, 6, 4, "float32", False)
    leaves = [t.requires_grad_() for t in args.values()]
    y, last = F.selective_scan(**args)
    assert y.shape == (2, 0, 6) and torch.equal(last, args["h0"])
    got = dict(zip(args, torch.autograd.grad((y, last), leaves, (dy, dlast))))
    assert torch.equal(got["h0"], dlast) and not got["A"].any() and got["B"].shape == (2, 0, 4)
    args, _, dy, _ = _scan_inputs(2, 5, 6, 4, "float32", False)
    none = {k: t[:0] if k in ("x", "delta", "B", "C", "z", "h0") else t for k, t in args.items()}
    y, last = F.selective_scan(**none)
    assert y.shape == (0, 5, 6) and last.shape == (0, 6, 4)
    for bad in (dict(x=args["x"][0]), dict(x=args["x"].half()), dict(x=args["x"].cpu()), dict(delta=args["delta"][:, :4]),
                dict(delta=args["delta"].bfloat16()), dict(A=args["A"][:5]), dict(A=args["A"].bfloat16()), dict(A=None),
                dict(B=args["B"][..., :3]), dict(C=args["C"][:1]), dict(C=args["C"].bfloat16()), dict(D=args["D"][:5]),
                dict(z=args["z"][..., :5]), dict(delta_bias=args["delta_bias"].bfloat16()), dict(h0=args["h0"][:, :5]),
                dict(starts=torch.zeros(2, 4, dtype=torch.bool, device="cuda"))):
        with pytest.raises(ValueError):
            F.selective_scan(**{**args, **bad})
    big = {k: torch.zeros(*t.shape[:-1], 129, device="cuda") if k in ("A", "B", "C", "h0") else t for k, t in args.items()}
    with pytest.raises(NotImplementedError):
        F.selective_scan(**big)
    with pytest.raises(ValueError):
        F.selective_scan(**{k: t[..., :0] if k in ("A", "B", "C", "h0") else t for k, t in args.items()})
    carry = F.selective_scan_fwd(**args)[2]
    h0 = args.pop("h0")
    for bad in (dict(carry=carry[:-1]), dict(carry=carry.bfloat16()), dict(dy=dy[:1]), dict(dy=dy.bfloat16()),
                dict(dlast=h0[:1])):
        with pytest.raises(ValueError):
            F.selective_scan_bwd(**{**args, "carry": carry, "dy": dy, **bad})
    step = {k: t[:, 0] if k in ("x", "delta", "B", "C", "z") else t for k, t in args.items()}
    flat = torch.zeros(100, device="cuda")
    for bad in (dict(x=args["x"]), dict(state=h0[:1]), dict(state=h0.bfloat16()), dict(B=step["B"][:1]),
                dict(state=flat[:48].view(2, 6, 4), out=flat[4:52].view(2, 6, 4)),
                dict(state=torch.zeros(2, 4, 6, device="cuda").transpose(1, 2)),
                dict(state=h0.clone().requires_grad_()), dict(x=step["x"].clone().requires_grad_())):
        with pytest.raises(ValueError):
            F.selective_step(**{**step, "state": h0, **bad})


# ---- policy_loss --------------------------------------------------------------------

POLICY_SHAPES = [(1, 1), (3, 2), (5, 33), (9, 1000), (4, 4099), (70, 513), (300, 130), (2, 32000), (3, 131073)]


def _policy_inputs(n, vocab, dtype, tau=1.0, seed=0):
    g = np.random.default_rng([n, vocab, seed])
    logits = _t(2 * g.standard_normal((n, vocab)), dtype)
    tokens = g.integers(0, vocab, n)
    s = _n(logits) / tau
    s = s - s.max(1, keepdims=True)
    logp = s[np.arange(n), tokens] - np.log(np.exp(s).sum(1))
    # ratios away from where they are clipped (0.8, 1.28): by more than f32 can be off
    gap = np.log(g.choice([0.5, 0.7, 0.9, 1.0, 1.1, 1.2, 1.4, 1.9], n)) + 0.02 * g.uniform(-1, 1, n)
    old, ref = (logp - gap).astype(np.float32), (logp + 0.4 * g.standard_normal(n)).astype(np.float32)
    if n > 2:
        tokens[g.integers(n)] = -1
    return logits, tokens, old, ref, g.standard_normal(n).astype(np.float32)


def _policy_check(logits, tokens, old, adv, ref=None, clip=(0.2, 0.28), kl=0.0, tau=1.0, total=None):
    import torch
    from oxitorch_b200 import functional as F
    shape = logits.shape[:-1]
    dev = lambda a: None if a is None else torch.from_numpy(np.asarray(a)).cuda().reshape(shape)  # noqa: E731
    (loss, logp, grad), (bl, bp, bg), margin = R.policy(_n(logits).reshape(-1, logits.shape[-1]), tokens, old, adv, ref,
                                                        clip, kl, tau, total)
    assert margin > 1, "an input of the test lies where the ratio is clipped"
    x = logits.detach().requires_grad_()
    got, got_p = F.policy_loss(x, dev(tokens), dev(old), dev(adv), ref_logp=dev(ref), clip=clip, kl_coef=kl, temperature=tau,
                               total_rows=total)
    _check(got.reshape(1), [loss], [bl], "loss")
    _check(got_p.reshape(-1), logp, bp, "logp")
    (d,) = torch.autograd.grad(got, x)
    _check(d.reshape(-1, d.shape[-1]), grad, bg, "dlogits")
    with torch.no_grad():
        again, _ = F.policy_loss(logits, dev(tokens), dev(old), dev(adv), ref_logp=dev(ref), clip=clip, kl_coef=kl,
                                 temperature=tau, total_rows=total)
        assert torch.equal(again, got.detach())
        assert torch.equal(F.token_logprobs(logits, dev(tokens), temperature=tau), got_p)


@pytest.mark.parametrize("kl,tau", [(0.0, 1.0), (0.1, 1.0), (0.05, 0.7)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,vocab", POLICY_SHAPES)
def test_policy_loss(n, vocab, dtype, kl, tau):
    logits, tokens, old, ref, adv = _policy_inputs(n, vocab, dtype, tau)
    _policy_check(logits, tokens, old, adv, ref if kl else None, kl=kl, tau=tau)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,vocab", [(6001, 1003), (1501, 32001), (303, 131073)])
def test_policy_loss_many_rows_to_a_cluster(n, vocab, dtype):
    logits, tokens, old, ref, adv = _policy_inputs(n, vocab, dtype)
    tokens[n // 3:n // 3 + 400] = -1  # clusters that meet only padding for a while
    _policy_check(logits, tokens, old, adv, ref, kl=0.1)


@pytest.mark.parametrize("dtype,vocab", [("float32", 330001), ("bfloat16", 660001)])
def test_policy_loss_rows_wider_than_a_cluster_holds(dtype, vocab):
    logits, tokens, old, ref, adv = _policy_inputs(4, vocab, dtype)
    _policy_check(logits, tokens, old, adv, ref, kl=0.1)


@pytest.mark.parametrize("dtype", DTYPES)
def test_policy_loss_strided_rows_leading_dims_and_total(dtype):
    logits, tokens, old, ref, adv = _policy_inputs(12, 515, dtype)
    wide = _t(np.zeros((12, 600)), dtype)
    for offset in (0, 1, 8):
        view = wide[:, offset:offset + 515]
        view.copy_(logits)
        _policy_check(view, tokens, old, adv, ref, kl=0.1, total=40)
    _policy_check(logits.reshape(3, 4, 515), tokens, old, adv, ref, kl=0.1)


@pytest.mark.parametrize("dtype", DTYPES)
def test_policy_loss_padding_masked_logits_and_bad_values(dtype):
    import torch
    from oxitorch_b200 import _native as N
    from oxitorch_b200 import functional as F
    nan = float("nan")
    logits = torch.randn(6, 700, device="cuda").to(getattr(torch, dtype))
    logits[0] = nan                        # padding: not looked at
    logits[1, 300:] = -float("inf")        # tokens that cannot be sampled
    logits[2, 5] = nan
    logits[3] = -float("inf")
    tokens = torch.tensor([-1, 7, 9, 4, 800, 12], device="cuda")
    zero, one = torch.zeros(6, device="cuda"), torch.ones(6, device="cuda")
    flag = torch.zeros(4, dtype=torch.int32, device="cuda")
    loss, logp, d = F.policy_loss_fwd(logits, tokens, zero, one, zero, kl_coef=0.1, flag=flag)
    assert torch.isnan(loss)
    assert logp[0] == 0 and not d[0].any()
    assert torch.isfinite(logp[[1, 5]]).all() and torch.isnan(logp[[2, 3, 4]]).all()
    assert torch.isfinite(d[[1, 5]]).all() and not d[1, 300:].any() and torch.isnan(d[[2, 3, 4]]).all()
    assert flag.tolist() == [2, 800, 0, 700]
    with pytest.raises(RuntimeError):
        N.check(N.load().oxc_check_error_flag(flag.data_ptr(), 0, -1))
    # a sampled token that has become impossible: ratio 0
    logits = torch.zeros(1, 9, device="cuda")
    logits[0, 3] = -float("inf")
    loss, logp, d = F.policy_loss_fwd(logits, torch.tensor([3], device="cuda"), zero[:1], one[:1])
    assert loss == 0 and logp == -float("inf") and not d.any()
    # a NaN advantage reaches loss and gradient
    loss, _, d = F.policy_loss_fwd(torch.zeros(1, 9, device="cuda"), torch.tensor([3], device="cuda"), zero[:1], one[:1] * nan)
    assert torch.isnan(loss) and torch.isnan(d).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_policy_loss_clipped_rows_have_no_gradient(dtype):
    """Above 1 + above with A > 0, below 1 - below with A < 0; not the other way round."""
    import torch
    from oxitorch_b200 import functional as F
    logits = torch.randn(4, 100, device="cuda").to(getattr(torch, dtype)).requires_grad_()
    tokens = torch.arange(4, device="cuda")
    logp = F.token_logprobs(logits.detach(), tokens)
    old = logp - torch.tensor([0.5, 0.5, -0.5, -0.5], device="cuda")
    adv = torch.tensor([1.0, -1.0, 1.0, -1.0], device="cuda")
    loss, _ = F.policy_loss(logits, tokens, old, adv)
    (d,) = torch.autograd.grad(loss, logits)
    assert [bool(r.any()) for r in d] == [False, True, True, False]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("factor,rows,vocab", [(3.0, 20, 999), (-0.7, 20, 999), (0.3, 151, 32003)])
def test_policy_loss_gradient_is_the_same_whichever_backward_asks(dtype, factor, rows, vocab):
    import torch
    from oxitorch_b200 import functional as F
    logits, tokens, old, ref, adv = _policy_inputs(rows, vocab, dtype)
    dev = lambda a: torch.from_numpy(np.asarray(a)).cuda()  # noqa: E731
    x = logits.requires_grad_()
    loss, logp = F.policy_loss(x, dev(tokens), dev(old), dev(adv), dev(ref), kl_coef=0.1)
    g = torch.tensor(factor, device="cuda")
    a, = torch.autograd.grad(loss, x, g, retain_graph=True)
    b, = torch.autograd.grad(loss, x, g, retain_graph=True)
    one, = torch.autograd.grad(loss, x)
    assert torch.equal(a, b)
    assert torch.equal(a, (one.float() * factor).to(a.dtype))
    assert not logp.requires_grad


def test_policy_loss_no_rows_and_refusals():
    import torch
    from oxitorch_b200 import functional as F
    x = torch.zeros(0, 5, device="cuda", requires_grad=True)
    none = torch.zeros(0, device="cuda")
    loss, logp = F.policy_loss(x, torch.zeros(0, dtype=torch.int64, device="cuda"), none, none, total_rows=4)
    assert loss == 0 and logp.shape == (0,)
    assert torch.autograd.grad(loss, x)[0].shape == (0, 5)
    x, tokens, v = torch.zeros(3, 5, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda"), torch.zeros(3, device="cuda")
    good = dict(logits=x, tokens=tokens, old_logp=v, advantages=v)
    F.policy_loss(**{**good, "tokens": tokens.int()})
    for bad in (dict(logits=x[0]), dict(logits=x.half()), dict(logits=x.cpu()), dict(tokens=tokens.float()),
                dict(tokens=tokens[:2]), dict(old_logp=v[:2]), dict(old_logp=v.double()), dict(advantages=v.bfloat16()),
                dict(ref_logp=v[:2]), dict(kl_coef=0.1), dict(kl_coef=-0.1, ref_logp=v), dict(clip=-0.1), dict(clip=(0.1, -1)),
                dict(temperature=0.0), dict(temperature=float("nan")), dict(total_rows=2), dict(logits=x[:, :0])):
        with pytest.raises(ValueError):
            F.policy_loss(**{**good, **bad})
    with pytest.raises(ValueError):
        F.policy_loss(**{**good, "logits": x.clone().requires_grad_(), "old_logp": v.clone().requires_grad_()})
    with pytest.raises(ValueError):
        F.token_logprobs(x.clone().requires_grad_(), tokens)
    with pytest.raises(ValueError):
        F.token_logprobs(x, tokens[:2])


def test_policy_loss_rows_beyond_32_bits():
    import torch
    from oxitorch_b200 import functional as F
    n, vocab = 2, 50
    far = 2 ** 31 + 8
    base = torch.empty(far + 64, dtype=torch.bfloat16, device="cuda")
    view = base.as_strided((n, vocab), (far, 1))
    # rows 16 bytes aligned in both, so that both are summed in one order
    logits = torch.randn(n, 56, device="cuda").bfloat16()[:, :vocab]
    view.copy_(logits)
    tokens, v = torch.tensor([3, 7], device="cuda"), torch.ones(2, device="cuda")
    for a, b in zip(F.policy_loss_fwd(view, tokens, -v, v), F.policy_loss_fwd(logits, tokens, -v, v)):
        assert torch.equal(a, b)


# ---- global_norm, clip_global_norm_ --------------------------------------------------

def _gradients(sizes, dtypes, scale=1.0, seed=0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(n, device="cuda", generator=g) * scale).to(getattr(torch, dtypes[i % len(dtypes)]))
            for i, n in enumerate(sizes)]


def _clip_check(grads, max_norm, out=None):
    """The norm is off by its rounding to f32 (2^-24) and f64's; a clipped value by the
    factor's rounding and its own."""
    import torch
    from oxitorch_b200 import tensor_ops as T
    norm, want = R.clip([_n(g) for g in grads], max_norm)
    before = [g.clone() for g in grads]
    got = T.global_norm(grads)
    assert got.shape == () and abs(got.item() - norm) <= 2.0 ** -23 * norm
    assert torch.equal(T.clip_global_norm_(grads, max_norm, out=out), got)
    for g, b, w, o in zip(grads, before, want, grads if out is None else out):
        _check(o, w, 2.0 ** -23 * np.abs(w), "clipped")
        if out is not None:
            assert torch.equal(g, b)


@pytest.mark.parametrize("dtypes", [["float32"], ["bfloat16"], ["float32", "bfloat16"]])
@pytest.mark.parametrize("sizes", [[1], [0, 3, 0], [7, 4096, 100003], [5] * 97, [3, 1, 8, 16] * 400,
                                   [8192, 8193, 16384, 16385, 40000], [3000000, 1]])
def test_clip_global_norm(sizes, dtypes):
    import torch
    for max_norm in (1.0, 1e9, 0.0):
        _clip_check(_gradients(sizes, dtypes), max_norm)
        grads = _gradients(sizes, dtypes)
        _clip_check(grads, max_norm, out=[torch.full_like(g, float("nan")) for g in grads])


@pytest.mark.parametrize("dtype", DTYPES)
def test_clip_global_norm_into_a_bucket(dtype):
    """Gradients and outputs that start anywhere within 16 bytes; what lies around them stays."""
    import torch
    from oxitorch_b200 import tensor_ops as T
    sizes = [1, 3, 1000, 8, 5001, 2, 70001]
    grads = _gradients(sizes, [dtype])
    for gap in (0, 1, 3):
        total = sum(sizes) + gap * (len(sizes) + 1)
        bucket, source = (torch.full((total,), 7.0, device="cuda", dtype=grads[0].dtype) for _ in range(2))
        out, views, at = [], [], gap
        for g in grads:
            out.append(bucket[at:at + g.numel()])
            views.append(source[at:at + g.numel()])
            views[-1].copy_(g)
            at += g.numel() + gap
        _clip_check(views, 0.5, out)
        rest = torch.ones(total, dtype=torch.bool, device="cuda")
        at = gap
        for g in grads:
            rest[at:at + g.numel()] = False
            at += g.numel() + gap
        assert (bucket[rest] == 7.0).all()
        _clip_check(grads, 0.5, out)
        T.clip_global_norm_(views, 0.25)
        assert (source[rest] == 7.0).all()


def test_clip_global_norm_ranges_nan_and_infinity():
    import torch
    from oxitorch_b200 import tensor_ops as T
    for scale in (1e-30, 1e25, 1e37):  # whose squares f32 does not hold
        grads = _gradients([1000, 77], ["float32"], scale)
        if scale < 1e37:
            _clip_check(grads, 1e-20 if scale < 1 else 1.0)
        else:
            assert torch.isinf(T.global_norm(grads * 2000)) or torch.isfinite(T.global_norm(grads))
    grads = _gradients([1000, 77], ["float32"])
    grads[1][5] = float("nan")
    keep = [g.clone() for g in grads]
    assert torch.isnan(T.clip_global_norm_(grads, 1.0))
    assert all(torch.equal(a.nan_to_num(9.0), b.nan_to_num(9.0)) for a, b in zip(grads, keep))
    grads[1][5] = float("inf")
    assert torch.isinf(T.clip_global_norm_(grads, 1.0))
    assert not grads[0].any() and torch.isnan(grads[1][5])


def test_clip_global_norm_lists_and_refusals():
    import torch
    from oxitorch_b200 import tensor_ops as T
    a, b = _gradients([12, 20], ["float32"])
    assert T.global_norm([]).item() == 0 and T.clip_global_norm_([None], 1.0).item() == 0
    wide = _gradients([600], ["float32"])[0].view(20, 30)
    _clip_check([wide.t(), a.clone()], 0.5)
    both = [wide.clone().t(), b.clone()]
    assert torch.equal(T.clip_global_norm_([both[0], None, both[1]], 0.5, out=[torch.empty_like(both[0]), None, b.clone()]),
                       T.global_norm(both))
    for grads in ([a, a], [a, a[3:]], [wide, wide.t()], [wide[:, ::2]], [wide[:, :7]], [a.half()], [a.cpu()],
                  [torch.ones(3, 1, device="cuda").expand(3, 4)]):
        with pytest.raises(ValueError):
            T.clip_global_norm_(grads, 1.0)
    with pytest.raises(TypeError):
        T.clip_global_norm_([1.0], 1.0)
    for bad in (dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(out=[b]), dict(out=[a.clone(), b]),
                dict(out=[a.bfloat16()])):
        with pytest.raises(ValueError):
            T.clip_global_norm_(**{"grads": [a], "max_norm": 1.0, **bad})
    with pytest.raises(ValueError):
        T.clip_global_norm_([wide.t()], 1.0, out=[torch.empty(30, 20, device="cuda")])
    with pytest.raises(ValueError):
        T.clip_global_norm_([a.clone().requires_grad_()], 1.0)


# ---- together ------------------------------------------------------------------------

def _model(torch, silu_conv, scan, loss, p, ids, starts, tokens, old, adv, ref):
    x = p["embedding"][ids]
    for q in p["layers"]:
        u, z = (x @ q["in"]).chunk(2, -1)
        u = silu_conv(u, q["conv"], q["conv_bias"], starts)
        dbc = u @ q["bc"]
        rank = q["delta"].shape[0]
        n = q["A"].shape[1]
        delta = dbc[..., :rank] @ q["delta"]
        y = scan(u, delta, -torch.exp(q["A"]), dbc[..., rank:rank + n], dbc[..., rank + n:], q["D"], z, q["bias"], starts)
        x = x + y @ q["out"]
    return loss(x @ p["head"], tokens, old, adv, ref)


def _parameters(torch, g, vocab, dim, inner, n, rank, layers):
    def m(*s, scale=None):
        return torch.randn(*s, generator=g, dtype=torch.float64) * (s[0] ** -0.5 if scale is None else scale)
    return {"embedding": m(vocab, dim, scale=1.0), "head": m(dim, vocab), "layers": [
        {"in": m(dim, 2 * inner), "conv": m(inner, 4, scale=0.5), "conv_bias": m(inner, scale=0.1),
         "bc": m(inner, rank + 2 * n), "delta": m(rank, inner), "A": m(inner, n, scale=0.3), "D": m(inner, scale=1.0),
         "bias": m(inner, scale=0.3) - 3.0, "out": m(inner, dim)} for _ in range(layers)]}


def _leaves(p):
    return [p["embedding"], p["head"], *(t for q in p["layers"] for t in q.values())]


def test_a_training_step_of_them_together():
    """Two layers, packed rows, the policy loss and the clipped gradients, against the
    same model in 64 bits through torch's own autograd.

    About a hundred operators follow each other from a parameter to the loss and back,
    each a few roundings of its result in norm (sums over up to 130 terms: their tree or
    sequence at most 64): 100 * 8 * 2^-24 = 5e-5 of each gradient's norm."""
    import torch
    from oxitorch_b200 import functional as F
    from oxitorch_b200 import tensor_ops as T
    g = torch.Generator().manual_seed(5)
    vocab, dim, inner, n, rank = 60, 16, 40, 16, 3
    wide = _parameters(torch, g, vocab, dim, inner, n, rank, 2)
    ids = torch.randint(vocab, (2, 130), generator=g)
    starts = torch.rand(2, 130, generator=g) < 0.05
    tokens = torch.randint(-1, vocab, (2, 130), generator=g)

    def conv64(u, w, b, starts):
        seq = torch.nn.functional.pad(starts.long().cumsum(1), (3, 0))
        v = torch.nn.functional.pad(u, (0, 0, 3, 0))
        T_ = u.shape[1]
        out = b
        for k in range(4):
            same = (seq[:, k:k + T_] == seq[:, 3:]) & (torch.arange(T_) + k >= 3)
            out = out + w[:, k] * v[:, k:k + T_] * same.unsqueeze(-1)
        return torch.nn.functional.silu(out)

    def scan64(x, delta, A, B, C, D, z, bias, starts):
        dt = torch.nn.functional.softplus(delta + bias)
        h, ys = 0.0, []
        for t in range(x.shape[1]):
            keep = torch.exp(dt[:, t, :, None] * A) * ~starts[:, t, None, None]
            h = keep * h + (dt * x)[:, t, :, None] * B[:, t, None, :]
            ys.append((h * C[:, t, None, :]).sum(-1))
        return (torch.stack(ys, 1) + D * x) * torch.nn.functional.silu(z)

    def loss64(logits, tokens, old, adv, ref):
        logp = torch.log_softmax(logits, -1).gather(-1, tokens.clamp(min=0).unsqueeze(-1)).squeeze(-1)
        r = torch.exp(logp - old)
        each = -torch.minimum(r * adv, r.clamp(0.8, 1.2) * adv) + 0.1 * (torch.exp(ref - logp) - (ref - logp) - 1)
        return (each * (tokens >= 0)).sum() / tokens.numel(), logp.detach()

    zero = torch.zeros(2, 130, dtype=torch.float64)
    with torch.no_grad():
        _, logp = _model(torch, conv64, scan64, loss64, wide, ids, starts, tokens, zero, zero, zero)
    # ratios of about 0.7, 1 and 1.4: none near where they are clipped
    old = logp - torch.log(torch.tensor([0.7, 1.0, 1.4], dtype=torch.float64))[torch.randint(3, (2, 130), generator=g)]
    ref, adv = logp + 0.3 * torch.randn(2, 130, generator=g, dtype=torch.float64), torch.randn(2, 130, generator=g).double()
    narrow = {"embedding": wide["embedding"].float().cuda(), "head": wide["head"].float().cuda(),
              "layers": [{k: t.float().cuda() for k, t in q.items()} for q in wide["layers"]]}
    wide = {"embedding": narrow["embedding"].double().cpu(), "head": narrow["head"].double().cpu(),
            "layers": [{k: t.double().cpu() for k, t in q.items()} for q in narrow["layers"]]}
    for t in _leaves(wide) + _leaves(narrow):
        t.requires_grad_()
    want, _ = _model(torch, conv64, scan64, loss64, wide, ids, starts, tokens, old, adv, ref)
    want_grads = torch.autograd.grad(want, _leaves(wide))

    loss, _ = _model(
        torch, lambda u, w, b, s: F.causal_conv(u, w, b, starts=s)[0],
        lambda x, delta, A, B, C, D, z, bias, s: F.selective_scan(x, delta, A, B, C, D, z, bias, starts=s)[0],
        lambda logits, *a: F.policy_loss(logits, *a, kl_coef=0.1), narrow, ids.cuda(), starts.cuda(), tokens.cuda(),
        old.float().cuda(), adv.float().cuda(), ref.float().cuda())
    grads = list(torch.autograd.grad(loss, _leaves(narrow)))
    assert abs(loss.item() - want.item()) <= 5e-5 * max(1.0, abs(want.item()))
    for a, b in zip(grads, want_grads):
        assert (a.cpu().double() - b).norm() <= 5e-5 * b.norm()
    norm = torch.sqrt(sum((b ** 2).sum() for b in want_grads)).item()
    total = T.clip_global_norm_(grads, 0.5 * norm)
    assert abs(total.item() - norm) <= 5e-5 * norm
    for a, b in zip(grads, want_grads):
        assert (a.cpu().double() - 0.5 * b).norm() <= 1e-4 * 0.5 * b.norm()


def test_decoding_after_a_prompt_gives_the_prompts_outputs():
    """conv and scan over a prompt, then their steps, against the whole sequence."""
    import torch
    from oxitorch_b200 import functional as F
    args, _, _, _ = _scan_inputs(3, 60, 64, 16, "float32", False)
    g = torch.Generator(device="cuda").manual_seed(1)
    w, b = torch.randn(64, 4, device="cuda", generator=g), torch.randn(64, device="cuda", generator=g)
    args.pop("h0")
    x = args.pop("x")
    whole = F.selective_scan(F.causal_conv(x, w, b)[0], **args)[0]
    part = lambda lo, hi: {k: t[:, lo:hi] if k in ("delta", "B", "C", "z") else t for k, t in args.items()}  # noqa: E731
    u, kept = F.causal_conv(x[:, :40], w, b)
    y, state = F.selective_scan(u, **part(0, 40))
    assert torch.equal(y, whole[:, :40])
    for t in range(40, 60):
        at = {k: v[:, 0] if k in ("delta", "B", "C", "z") else v for k, v in part(t, t + 1).items()}
        y = F.selective_step(F.causal_conv_step(x[:, t], w, b, kept), **at, state=state)
        # the two add up a token's states in another order: 16 terms, a few roundings each
        size = (state.abs() * at["C"].abs().unsqueeze(1)).sum(-1) + whole[:, t].abs() + 1
        assert ((y - whole[:, t]).abs() <= 64 * 2.0 ** -24 * size * (1 + at["z"].abs())).all()


def _all_operators(dtype, seed):
    """name -> (inputs, function of them)."""
    import torch
    from oxitorch_b200 import functional as F
    from oxitorch_b200 import tensor_ops as T
    args, starts, dy, dlast = _scan_inputs(2, 300, 36, 16, dtype, True, seed=seed)
    x, w, b, x0, cstarts, cdy, cdlast = _conv_inputs(2, 300, 36, 4, dtype, True, seed=seed)
    logits, tokens, old, ref, adv = _policy_inputs(30, 5001, dtype, seed=seed)
    t = lambda a: torch.from_numpy(np.asarray(a)).cuda()  # noqa: E731
    scan = [*args.values(), _starts(starts), dy, dlast]

    def run_scan(x, delta, A, B, C, D, z, bias, h0, starts, dy, dlast):
        y, last, carry = F.selective_scan_fwd(x, delta, A, B, C, D, z, bias, h0, starts)
        return [y, last, *F.selective_scan_bwd(x, delta, A, B, C, carry, D, z, bias, starts, dy, dlast)]

    def run_conv(x, w, b, x0, starts, dy, dlast):
        return [*F.causal_conv_fwd(x, w, b, x0, starts), *F.causal_conv_bwd(x, w, b, x0, dy, dlast, starts)]

    def run_step(x, delta, A, B, C, D, z, bias, h0, *_):
        out = torch.empty_like(h0)
        return [F.selective_step(x[:, 0], delta[:, 0], A, B[:, 0], C[:, 0], h0, D, z[:, 0], bias, out=out), out]

    def run_clip(*grads):
        out = [torch.empty_like(g) for g in grads]
        return [T.clip_global_norm_(grads, 1.0, out=out), *out]

    def run_conv_step(x, w, b, x0, *_):
        out = torch.empty_like(x0)
        return [F.causal_conv_step(x[:, 0], w, b, x0, out=out), out]
    conv = [x, w, b, x0, _starts(cstarts), cdy, cdlast]
    return {"scan": (scan, run_scan), "conv": (conv, run_conv), "step": (scan, run_step), "conv step": (conv, run_conv_step),
            "policy": ([logits, t(tokens), t(old), t(adv), t(ref)], lambda *a: list(F.policy_loss_fwd(*a, kl_coef=0.1))),
            "clip": ([dy, dlast, x.float(), logits], run_clip)}


@pytest.mark.parametrize("dtype", DTYPES)
def test_selective_ops_captured_in_graphs(dtype):
    """Two graphs that share one pool, replayed in turn on new inputs in the captured
    buffers, give the bits of eager calls."""
    import torch
    buffers, later = _all_operators(dtype, 0), [_all_operators(dtype, s) for s in (1, 2)]
    for name, (inputs, f) in buffers.items():
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            f(*inputs)
        side.synchronize()
        graphs, outs = [], []
        for _ in range(2):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], pool=graphs[0].pool() if len(graphs) > 1 else None):
                outs.append(f(*inputs))
        for new in later:
            fresh = new[name][0]
            for a, b in zip(inputs, fresh):
                a.copy_(b)
            want = [t.clone() for t in f(*fresh)]
            for graph, out in zip(graphs, outs):
                graph.replay()
                torch.cuda.synchronize()
                for i, (a, b) in enumerate(zip(out, want)):
                    assert torch.equal(a, b), f"{name}: output {i}"


@pytest.mark.parametrize("dtype", DTYPES)
def test_selective_ops_on_side_streams_and_repeated(dtype):
    """The same bits at every call, and where two streams run them at once."""
    import torch
    for name, (inputs, f) in _all_operators(dtype, 3).items():
        want = f(*inputs)
        torch.cuda.synchronize()
        streams, found = [torch.cuda.Stream() for _ in range(2)], []
        for _ in range(3):
            for s in streams:
                with torch.cuda.stream(s):
                    found.append(f(*inputs))
        torch.cuda.synchronize()
        for got in found:
            for i, (a, b) in enumerate(zip(got, want)):
                assert torch.equal(a, b), f"{name}: output {i}"


def test_selective_backward_captured_in_a_graph():
    """Forward and backward through autograd in a captured graph; the eager graph of the
    same leaves is gone by then (while it lives, torch's engine waits for its stream)."""
    import torch
    from oxitorch_b200 import functional as F
    args, _, dy, dlast = _scan_inputs(1, 40, 8, 16, "float32", False)
    w = torch.randn(8, 4, device="cuda")
    leaves = [args["x"].requires_grad_(), args["A"].requires_grad_(), w.requires_grad_()]

    def step():
        u, _ = F.causal_conv(args["x"], w)
        y, last = F.selective_scan(u, *[args[k] for k in ("delta", "A", "B", "C", "D", "z", "delta_bias", "h0")])
        return torch.autograd.grad((y, last), leaves, (dy, dlast))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [t.clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_selective_gradients_refuse_to_be_differentiated_again():
    import torch
    from oxitorch_b200 import functional as F
    args, _, dy, _ = _scan_inputs(1, 9, 4, 4, "float32", False)
    x, w = args.pop("x").requires_grad_(), torch.randn(4, 4, device="cuda")
    y, _ = F.selective_scan(x, **args)
    u, _ = F.causal_conv(x, w)
    logits = torch.randn(3, 9, device="cuda", requires_grad=True)
    tokens, v = torch.arange(3, device="cuda"), torch.ones(3, device="cuda")
    loss, _ = F.policy_loss(logits, tokens, -v, v)
    for out, leaf in ((y, x), (u, x), (loss, logits)):
        (d,) = torch.autograd.grad(out.sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(d.sum(), leaf)
    from torch.autograd import forward_ad
    with forward_ad.dual_level(), torch.no_grad():
        dual = forward_ad.make_dual(x.detach(), torch.ones_like(x))
        first = {k: t[:, 0] if k in ("delta", "B", "C", "z") else t for k, t in args.items() if k != "h0"}
        for call in (lambda: F.selective_scan(dual, **args), lambda: F.causal_conv(dual, w),
                     lambda: F.selective_step(dual[:, 0], **first, state=args["h0"]),
                     lambda: F.causal_conv_step(dual[:, 0], w, None, torch.zeros(1, 3, 4, device="cuda")),
                     lambda: F.policy_loss(forward_ad.make_dual(logits.detach(), torch.ones_like(logits)), tokens, -v, v),
                     lambda: F.token_logprobs(forward_ad.make_dual(logits.detach(), torch.ones_like(logits)), tokens)):
            with pytest.raises((NotImplementedError, RuntimeError, ValueError)):
                call()
