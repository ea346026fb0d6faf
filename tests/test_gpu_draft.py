"""The recurrent draft model's operators on the device against their 64-bit
references (tests/draft_reference.py).

Tolerances come with the references: per element, the magnitude-weighted count
of f32 roundings; a bfloat16 result may be off by half a unit in its last place
(2^-8 of the value) on top.  Whole numbers are equal."""

import numpy as np
import pytest

import draft_reference as R

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "bfloat16"]


def _t(a, dtype="float32"):
    import torch
    return torch.from_numpy(np.array(a, np.float32)).cuda().to(getattr(torch, dtype))


def _n(t):
    import torch
    return t.detach().to(torch.float64).cpu().numpy()


def _check(got, want, bound, what):
    """|got - want| <= bound, plus bfloat16's own rounding; NaN and infinity agree."""
    import torch
    g, want = _n(got), np.asarray(want, np.float64)
    bound = np.broadcast_to(np.asarray(bound, np.float64), want.shape)
    assert g.shape == want.shape, f"{what}: {g.shape} vs {want.shape}"
    assert np.array_equal(np.isnan(g), np.isnan(want)), f"{what}: NaN in other places"
    fine = np.isfinite(want)
    assert np.array_equal(g[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), f"{what}: infinities"
    if got.dtype == torch.bfloat16:
        bound = bound + 2.0 ** -8 * (np.abs(want) + bound) + 2.0 ** -133
    off = np.abs(g[fine] - want[fine]) - bound[fine] - 2.0 ** -140
    assert not off.size or off.max() <= 0, f"{what}: {off.max():.3g} beyond its bound"


# ---- add_rms_norm -------------------------------------------------------------------

NORM_SHAPES = [(1, 1), (1, 128), (3, 5), (5, 129), (2, 4096), (37, 1000), (300, 257), (4, 5000), (2, 16384),
               (1, 32768), (1300, 64), (3, 10007)]


def _norm_inputs(rows, cols, dtype, seed=0):
    g = np.random.default_rng(rows * 100003 + cols + seed)
    x, res = g.standard_normal((rows, cols)), 3 * g.standard_normal((rows, cols))
    return _t(x, dtype), _t(res), _t(g.uniform(0.5, 1.5, cols)), _t(g.standard_normal((rows, cols)), dtype), \
        _t(g.standard_normal((rows, cols)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
def test_add_rms_norm_forward(rows, cols, dtype):
    from oxitorch_b200 import functional as F
    x, res, w, _, _ = _norm_inputs(rows, cols, dtype)
    y, r = F.add_rms_norm(x, res, w, 1e-5)
    want_y, _, _ = R.add_rms_norm(_n(x), _n(res), _n(w), 1e-5)
    assert y.dtype == x.dtype
    assert (r == x.float() + res).all()  # one f32 addition
    # 48 roundings in inv, as in the gradient's bound, and two products
    _check(y, want_y, 56 * R.EPS * np.abs(want_y), "y")


@pytest.mark.parametrize("mode", ["ref", "exact"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
def test_add_rms_norm_gradient(rows, cols, dtype, mode):
    import torch
    from oxitorch_b200 import functional as F
    x, res, w, dy, dr = _norm_inputs(rows, cols, dtype)
    for t in (x, res, w):
        t.requires_grad_()
    y, r = F.add_rms_norm(x, res, w, 1e-5, grad_mode=mode)
    dx, dres, dw = torch.autograd.grad((y, r), (x, res, w), (dy, dr))
    (d, want_dw), (bd, bdw) = R.add_rms_norm_grad(_n(x), _n(res), _n(w), 1e-5, _n(dy), _n(dr), mode == "exact")
    assert dx.dtype == x.dtype and dres.dtype == torch.float32
    _check(dres, d, bd, "dresidual")
    _check(dx, d, bd, "dx")
    _check(dw, want_dw, bdw, "dweight")


def test_add_rms_norm_one_output_used():
    import torch
    from oxitorch_b200 import functional as F
    x, res, w, dy, dr = _norm_inputs(7, 96, "bfloat16")
    for t in (x, res, w):
        t.requires_grad_()
    y, r = F.add_rms_norm(x, res, w, 1e-5, grad_mode="exact")
    got = torch.autograd.grad(y, (x, res, w), dy)
    (d, dw), (bd, bdw) = R.add_rms_norm_grad(_n(x), _n(res), _n(w), 1e-5, _n(dy), None)
    for g, want, b in zip(got, (d, d, dw), (bd, bd, bdw)):
        _check(g, want, b, "through y")
    y, r = F.add_rms_norm(x, res, w, 1e-5)
    got = torch.autograd.grad(r, (x, res, w), dr)
    for g, want in zip(got, (_n(dr), _n(dr), np.zeros(96))):
        _check(g, want, 0.0, "through r")


@pytest.mark.parametrize("block", [128, None])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
def test_add_rms_norm_quant(rows, cols, dtype, block):
    import torch
    from oxitorch_b200 import functional as F
    x, res, w, _, _ = _norm_inputs(rows, cols, dtype, seed=1)
    q, scale, r = F.add_rms_norm_quant(x, res, w, 1e-5, block=block)
    y, _, _ = R.add_rms_norm(_n(x), _n(res), _n(w), 1e-5)
    assert q.dtype == torch.float8_e4m3fn and (r == x.float() + res).all()
    want = R.block_scales(y, block)
    _check(scale, want, 60 * R.EPS * want, "scale")
    # q is y / scale rounded to nearest: y / scale is off by the roundings of y,
    # of the scale and of the division, which may also move it past a tie
    z = y / np.repeat(want, block or cols, -1)[:, :cols]
    _check(q.to(torch.float32), z, R.e4m3_half_step(z) * (1 + 2.0 ** -10) + 120 * R.EPS * np.abs(z), "q")


def test_add_rms_norm_quant_extremes():
    import torch
    from oxitorch_b200 import functional as F
    x = torch.zeros(4, 300, device="cuda")
    res = torch.zeros(4, 300, device="cuda")
    res[1, 130] = float("nan")
    res[2, 0] = 1.0  # one column holds all: y = sqrt(cols) there
    res[3] = 1e-30
    w = torch.ones(300, device="cuda")
    q, scale, r = F.add_rms_norm_quant(x, res, w, 1e-6)
    assert (q[0].float() == 0).all() and (scale[0] == 2.0 ** -126).all()
    assert torch.isnan(scale[1]).all() and torch.isnan(q[1].float()).all()  # the row's norm is NaN
    assert q[2, 0].float() == 448 and (q[2, 1:].float() == 0).all()
    assert torch.isfinite(q[3].float()).all() and torch.isfinite(scale[3]).all()
    q, scale, _ = F.add_rms_norm_quant(x, res, torch.full((300,), float("inf"), device="cuda"))
    assert torch.isnan(scale[2]).all()  # the row's zeros times an infinite weight are NaN
    assert torch.isinf(scale[3]).all() and (q[3].view(torch.uint8) & 127 == 127).all()  # inf / inf


@pytest.mark.parametrize("dtype", DTYPES)
def test_add_rms_norm_strided_rows_and_leading_dims(dtype):
    import torch
    from oxitorch_b200 import functional as F
    x, res, w, dy, dr = _norm_inputs(12, 260, dtype)
    wide_x = torch.full((12, 300), 9.0, device="cuda", dtype=x.dtype)
    wide_r = torch.full((12, 301), 9.0, device="cuda")
    wide_x[:, 8:268], wide_r[:, 3:263] = x, res
    want = F.add_rms_norm_fwd(x, res, w)
    got = F.add_rms_norm_fwd(wide_x[:, 8:268], wide_r[:, 3:263], w)
    for a, b, tol in zip(got, want, (2.0 ** -7, 0.0, 1e-6)):  # vector and scalar rows sum in another order
        assert ((a.double() - b.double()).abs() <= tol * b.double().abs()).all()
    cube = F.add_rms_norm_fwd(x.view(3, 4, 260).transpose(0, 1), res.view(3, 4, 260).transpose(0, 1), w)
    assert cube[0].shape == (4, 3, 260) and cube[2].shape == (4, 3)
    assert (cube[1] == want[1].view(3, 4, 260).transpose(0, 1)).all()
    # gradients handed in as expanded views
    xs, rs = x.clone().requires_grad_(), res.clone().requires_grad_()
    y, r = F.add_rms_norm(xs, rs, w, 1e-5, grad_mode="exact")
    (y.float().sum() + r.sum()).backward()
    ones = np.ones((12, 260))
    (d, _), (bd, _) = R.add_rms_norm_grad(_n(x), _n(res), _n(w), 1e-5, ones, ones)
    _check(rs.grad, d, bd, "dresidual of a sum")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(5, 260), (9, 133), (3, 4100), (40, 7)])
def test_add_rms_norm_rows_that_start_anywhere(rows, cols, dtype):
    """Operands whose rows no common alignment fits: views at odd offsets and strides."""
    import torch
    from oxitorch_b200 import functional as F
    x, res, w, dy, dr = _norm_inputs(rows, cols, dtype, seed=3)

    def odd(t, offset, extra):
        wide = torch.full((rows, cols + extra), float("nan"), device="cuda", dtype=t.dtype)
        wide[:, offset:offset + cols] = t
        return wide[:, offset:offset + cols]
    xo, ro, gyo, gro = odd(x, 1, 6), odd(res, 2, 3), odd(dy, 3, 7), odd(dr, 1, 2)
    want_y, want_r, _ = R.add_rms_norm(_n(x), _n(res), _n(w), 1e-5)
    y, r, rstd = F.add_rms_norm_fwd(xo, ro, w, 1e-5)
    _check(y, want_y, 56 * R.EPS * np.abs(want_y), "y")
    assert (r == x.float() + res).all()
    for mode in ("ref", "exact"):
        dx, dres, dw = F.add_rms_norm_bwd(r, w, rstd, gyo, gro, mode)
        (d, want_dw), (bd, bdw) = R.add_rms_norm_grad(_n(x), _n(res), _n(w), 1e-5, _n(dy), _n(dr), mode == "exact")
        _check(dres, d, bd, "dresidual")
        _check(dx, d, bd, "dx")
        _check(dw, want_dw, bdw, "dweight")
    for block in (128, None):
        q, scale, r = F.add_rms_norm_quant(xo, ro, w, 1e-5, block=block)
        want = R.block_scales(want_y, block)
        _check(scale, want, 60 * R.EPS * want, "scale")
        z = want_y / np.repeat(want, block or cols, -1)[:, :cols]
        _check(q.to(torch.float32), z, R.e4m3_half_step(z) * (1 + 2.0 ** -10) + 120 * R.EPS * np.abs(z), "q")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(700, 6), (650, 1001), (600, 1537), (400, 2999), (400, 3000), (300, 3333),
                                       (300, 5001), (200, 5804), (200, 7003), (30, 9000), (30, 10002), (20, 12999),
                                       (9, 16383), (9, 20001)])
def test_add_rms_norm_rows_between_nans(rows, cols, dtype):
    """Rows read by whole vectors that reach into what lies between them: every
    width's own kernel, several rows to a group."""
    import torch
    from oxitorch_b200 import functional as F
    x, res, w, dy, dr = _norm_inputs(rows, cols, dtype, seed=4)

    def apart(t, extra):  # the last row ends with the buffer
        flat = torch.full(((rows - 1) * (cols + extra) + cols,), float("nan"), device="cuda", dtype=t.dtype)
        view = flat.as_strided((rows, cols), (cols + extra, 1))
        view.copy_(t)
        return view
    xa, ra, gya, gra = apart(x, 4), apart(res, 8), apart(dy, 4), apart(dr, 12)
    want_y, _, _ = R.add_rms_norm(_n(x), _n(res), _n(w), 1e-5)
    for dense in (False, True):
        y, r, rstd = F.add_rms_norm_fwd(x if dense else xa, res if dense else ra, w, 1e-5)
        _check(y, want_y, 56 * R.EPS * np.abs(want_y), "y")
        assert (r == x.float() + res).all()
        dx, dres, dw = F.add_rms_norm_bwd(r, w, rstd, dy if dense else gya, dr if dense else gra, "exact")
        (d, want_dw), (bd, bdw) = R.add_rms_norm_grad(_n(x), _n(res), _n(w), 1e-5, _n(dy), _n(dr), True)
        _check(dres, d, bd, "dresidual")
        _check(dx, d, bd, "dx")
        _check(dw, want_dw, bdw, "dweight")
    for block in (128, None):
        q, scale, r = F.add_rms_norm_quant(xa, ra, w, 1e-5, block=block)
        assert (r == x.float() + res).all()
        want = R.block_scales(want_y, block)
        _check(scale, want, 60 * R.EPS * want, "scale")
        z = want_y / np.repeat(want, block or cols, -1)[:, :cols]
        _check(q.to(torch.float32), z, R.e4m3_half_step(z) * (1 + 2.0 ** -10) + 120 * R.EPS * np.abs(z), "q")


def test_add_rms_norm_empty_and_refusals():
    import torch
    from oxitorch_b200 import functional as F
    w = torch.ones(8, device="cuda")
    e = torch.empty(0, 8, device="cuda")
    y, r, rstd = F.add_rms_norm_fwd(e, e, w)
    assert y.shape == (0, 8) and rstd.shape == (0,)
    dx, dres, dw = F.add_rms_norm_bwd(e, w, rstd, e)
    assert (dw == 0).all()
    q, scale, _ = F.add_rms_norm_quant(e, e, w)
    assert q.shape == (0, 8) and scale.shape == (0, 1)
    x = torch.zeros(2, 8, device="cuda")
    for bad in (lambda: F.add_rms_norm(x, x[:1], w), lambda: F.add_rms_norm(x, x.bfloat16(), w),
                lambda: F.add_rms_norm(x.half(), x, w), lambda: F.add_rms_norm(x, x, w[:4]),
                lambda: F.add_rms_norm(x, x.cpu(), w), lambda: F.add_rms_norm_quant(x, x, w, block=64),
                lambda: F.add_rms_norm(x[:, :0], x[:, :0], w[:0])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        z = torch.zeros(1, 32769, device="cuda")
        F.add_rms_norm(z, z, z[0])


# ---- gated_scan -----------------------------------------------------------------------

SCAN_SHAPES = [(1, 1, 1), (2, 1, 130), (1, 2, 64), (3, 63, 33), (2, 64, 128), (2, 65, 256), (1, 127, 100),
               (2, 129, 512), (1, 700, 40), (1, 2049, 260), (5, 300, 1001), (1, 9001, 8), (16, 5001, 64),
               (3, 12900, 130)]


def _scan_inputs(B, T, D, dtype, seed=0, starts=False):
    g = np.random.default_rng(B * 1000003 + T * 1009 + D + seed)
    x, gate = g.standard_normal((B, T, D)), g.standard_normal((B, T, D)) + np.linspace(-2, 6, D)
    dh, h0, dlast = g.standard_normal((B, T, D)), g.standard_normal((B, D)), g.standard_normal((B, D))
    s = None
    if starts:
        import torch
        s = torch.from_numpy(g.random((B, T)) < 0.03).cuda()
    return _t(x, dtype), _t(gate, dtype), _t(h0), _t(dh, dtype), _t(dlast), s


def _scan_check(x, gate, h0, starts, dh, dlast):
    import torch
    from oxitorch_b200 import functional as F
    leaves = [t.detach().requires_grad_() for t in ((x, gate) if h0 is None else (x, gate, h0))]
    h, last = F.gated_scan(*leaves, **({} if h0 is not None else {"h0": None}), starts=starts)
    mask = None if starts is None else starts.cpu().numpy()
    n0 = None if h0 is None else _n(h0)
    want, want_last, bound = R.gated_scan(_n(x), _n(gate), n0, mask)
    assert h.dtype == x.dtype and last.dtype == torch.float32
    _check(h, want, bound, "h")
    _check(last, want_last, bound[:, -1], "last")
    with torch.no_grad():
        again = F.gated_scan(x, gate, h0, starts)
    assert (again[0] == h).all() and (again[1] == last).all()
    outs, seeds = ((h, last), (dh, dlast)) if dlast is not None else ((h,), (dh,))
    if dh is None:
        outs, seeds = (last,), (dlast,)
    got = torch.autograd.grad(outs, leaves, seeds)
    grads, bounds = R.gated_scan_grad(_n(x), _n(gate), n0, mask, None if dh is None else _n(dh),
                                      None if dlast is None else _n(dlast))
    for name, g, wg, b in zip(("dx", "dgate", "dh0"), got, grads, bounds):
        _check(g, wg, b, name)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,D", SCAN_SHAPES)
def test_gated_scan(B, T, D, dtype, packed):
    x, gate, h0, dh, dlast, starts = _scan_inputs(B, T, D, dtype, starts=packed)
    _scan_check(x, gate, h0, starts, dh, dlast)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_scan_without_state_or_with_one_gradient(dtype):
    x, gate, h0, dh, dlast, _ = _scan_inputs(2, 200, 72, dtype)
    _scan_check(x, gate, None, None, dh, None)
    _scan_check(x, gate, None, None, None, dlast)
    _scan_check(x, gate, h0, None, dh, None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [0, 1])
def test_gated_scan_reads_halves_of_a_projection(dtype, offset):
    """x and gate as slices of one tensor, dh batch-first of a time-first one."""
    import torch
    B, T, D = 2, 150, 96
    x, gate, h0, dh, dlast, _ = _scan_inputs(B, T, D, dtype)
    wide = torch.full((B, T, 2 * D + 7), float("nan"), device="cuda", dtype=x.dtype)
    xv, gv = wide[..., offset:offset + D], wide[..., offset + D:offset + 2 * D]
    xv.copy_(x), gv.copy_(gate)
    turned = dh.transpose(0, 1).contiguous().transpose(0, 1)
    assert turned.stride(1) > turned.stride(0)
    _scan_check(xv, gv, h0, None, turned, dlast)
    column = dh[..., :1].expand(B, T, D)  # a last dim that is not dense is copied
    _scan_check(xv, gv, h0, None, column, dlast)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_scan_long_memory_and_extreme_gates(dtype):
    """Gates that hold everything, forget everything, and saturate; a_t = 1 - 6e-8."""
    import torch
    x, gate, h0, dh, dlast, _ = _scan_inputs(1, 1500, 64, dtype)
    gate[:, :, :8] = 16.5
    gate[:, :, 8:16] = -40.0
    gate[:, :, 16:24] = 200.0
    gate[:, :, 24:32] = -200.0
    gate[:, 700, 32:40] = float("inf")
    gate[:, 701, 40:48] = float("-inf")
    _scan_check(x, gate, h0, None, dh, dlast)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_gated_scan_starts_stop_nan_and_infinity(dtype, poison):
    import torch
    from oxitorch_b200 import functional as F
    B, T, D = 1, 400, 130
    x, gate, h0, dh, dlast, _ = _scan_inputs(B, T, D, dtype)
    for new in (64, 130, 399):
        starts = torch.zeros(B, T, dtype=torch.bool, device="cuda")
        starts[:, new] = True
        xp = x.clone()
        xp[:, new - 3] = poison
        h, last = F.gated_scan(xp, gate, h0, starts)
        assert not torch.isfinite(h[:, new - 3:new].float()).any()
        clean, _, bound = R.gated_scan(_n(x)[:, new:], _n(gate)[:, new:])
        _check(h[:, new:], clean, bound, "h after the start")
        # and backwards: gradients after the start do not reach what lies before
        leaves = [t.clone().requires_grad_() for t in (x, gate, h0)]
        bad = dh.clone()
        bad[:, new + 0:] = poison
        h, last = F.gated_scan(*leaves, starts)
        dx, dg, dh0 = torch.autograd.grad(h, leaves, bad)
        (wx, wg, w0), (bx, bg, b0) = R.gated_scan_grad(_n(x)[:, :new], _n(gate)[:, :new], _n(h0), None,
                                                       _n(dh)[:, :new], None)
        _check(dx[:, :new], wx, bx, "dx before the start")
        _check(dg[:, :new], wg, bg, "dgate before the start")
        _check(dh0, w0, b0, "dh0")


def test_gated_scan_nan_reaches_all_that_follows():
    import torch
    from oxitorch_b200 import functional as F
    x, gate, h0, _, _, _ = _scan_inputs(1, 1000, 64, "float32")
    gate[:, 300:] = -60.0  # forgets to nothing within a few tokens, but NaN * 0 is NaN
    x[:, 100, 5] = float("nan")
    h, last = F.gated_scan(x, gate, h0)
    assert torch.isnan(h[0, 100:, 5]).all() and torch.isnan(last[0, 5])
    assert torch.isfinite(h[0, :, :5]).all() and torch.isfinite(h[0, :, 6:]).all()


def test_gated_scan_offsets_beyond_32_bits():
    import torch
    from oxitorch_b200 import functional as F
    x, gate, h0, _, _, _ = _scan_inputs(1, 3, 64, "bfloat16")
    apart = 1_200_000_000
    base = torch.empty(2 * apart + 64, dtype=torch.bfloat16, device="cuda")
    far = base.as_strided((1, 3, 64), (64, apart, 1))
    far.copy_(x)
    want, got = F.gated_scan(x, gate, h0), F.gated_scan(far, gate, h0)
    assert (want[0] == got[0]).all() and (want[1] == got[1]).all()


def test_gated_scan_empty_and_refusals():
    import torch
    from oxitorch_b200 import functional as F
    h0 = torch.ones(2, 8, device="cuda")
    e = torch.empty(2, 0, 8, device="cuda")
    h, last = F.gated_scan(e, e, h0)
    assert h.shape == (2, 0, 8) and (last == h0).all()
    assert (F.gated_scan(e, e)[1] == 0).all()
    leaf = h0.clone().requires_grad_()
    h, last = F.gated_scan(e, e, leaf)
    assert (torch.autograd.grad(last.sum(), leaf)[0] == 1).all()
    assert F.gated_scan(e[:0], e[:0])[1].shape == (0, 8)
    x = torch.zeros(2, 3, 8, device="cuda")
    for bad in (lambda: F.gated_scan(x, x[:1]), lambda: F.gated_scan(x, x.bfloat16()),
                lambda: F.gated_scan(x[0], x[0]), lambda: F.gated_scan(x, x, h0[:1]),
                lambda: F.gated_scan(x, x, h0.bfloat16()), lambda: F.gated_scan(x.half(), x.half()),
                lambda: F.gated_scan(x, x, starts=torch.zeros(2, 4, dtype=torch.bool, device="cuda")),
                lambda: F.gated_scan(x, x, starts=torch.zeros(2, 3, device="cuda")),
                lambda: F.gated_scan(x, x.cpu())):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,D", [(1, 1), (3, 130), (8, 4096), (300, 33)])
def test_gated_step_continues_a_scan(B, D, dtype):
    import torch
    from oxitorch_b200 import functional as F
    x, gate, h0, _, _, _ = _scan_inputs(B, 6, D, dtype)
    want, _, bound = R.gated_scan(_n(x), _n(gate), _n(h0))
    state, kept = h0.clone(), []
    for t in range(3):  # in place
        h = F.gated_step(x[:, t], gate[:, t], state)
        _check(h, want[:, t], bound[:, t], "h")
        _check(state, want[:, t], bound[:, t], "state")
    before = state.clone()
    out = torch.empty_like(state)
    h = F.gated_step(x[:, 3], gate[:, 3], state, out=out)
    assert (state == before).all()  # a rejected draft goes back to it
    _check(out, want[:, 3], bound[:, 3], "out")
    for bad in (lambda: F.gated_step(x[:, 0], gate[:, 0], state.bfloat16()),
                lambda: F.gated_step(x, gate, state), lambda: F.gated_step(x[:, 0], gate[:, 0], state, out=x[:, 0, :0]),
                lambda: F.gated_step(x[:, 0].clone().requires_grad_(), gate[:, 0], state)):
        with pytest.raises(ValueError):
            bad()
    pair = torch.zeros(2 * B * D, device="cuda")
    if B * D > 1:
        with pytest.raises(ValueError, match="overlap"):
            F.gated_step(x[:, 0], gate[:, 0], pair[:B * D].view(B, D), out=pair[1:B * D + 1].view(B, D))


def test_gradients_refuse_to_be_differentiated_again():
    import torch
    from oxitorch_b200 import functional as F
    x = torch.randn(2, 4, 8, device="cuda").requires_grad_()
    h, _ = F.gated_scan(x, x)
    y, _ = F.add_rms_norm(x, x, torch.ones(8, device="cuda"))
    loss = F.distill_loss(x, torch.zeros(2, 4, 1, device="cuda"), torch.zeros(2, 4, 1, dtype=torch.int64, device="cuda"))
    for out in (h.sum(), y.sum(), loss):
        (g,) = torch.autograd.grad(out, x, create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()


# ---- distill_loss ------------------------------------------------------------------------

def _distill_inputs(n, vocab, top, dtype, seed=0):
    g = np.random.default_rng(n * 7919 + vocab * 31 + top + seed)
    logits = 2 * g.standard_normal((n, vocab))
    ids = np.stack([g.permutation(vocab)[:top] for _ in range(n)])
    teacher = -np.sort(-(3 * g.standard_normal((n, top))), -1) + 5
    np.put_along_axis(logits, ids, teacher + g.standard_normal((n, top)), 1)
    kept = g.integers(1, 2 * top + 1, (n, 1))
    kept[g.random((n, 1)) < 0.2] = 0
    ids = np.where(np.arange(top) < kept, ids, -1)
    import torch
    return _t(logits, dtype), _t(teacher), torch.from_numpy(ids).cuda()


def _distill_check(logits, teacher, ids, tau, total_rows=None):
    import torch
    from oxitorch_b200 import functional as F
    leaf = logits.detach().requires_grad_()
    loss = F.distill_loss(leaf, teacher, ids, tau, total_rows)
    (grad,) = torch.autograd.grad(loss, leaf)
    want = R.distill(_n(logits), _n(teacher), ids.cpu().numpy(), tau, total_rows)
    _check(loss, want[0], want[2], "loss")
    _check(grad, want[1], want[3], "dlogits")
    with torch.no_grad():
        assert torch.equal(F.distill_loss(logits, teacher, ids, tau, total_rows), loss)
    return grad


@pytest.mark.parametrize("tau", [1.0, 2.0, 0.7])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,vocab,top", [(1, 1, 1), (3, 2, 2), (5, 33, 7), (9, 1000, 16), (4, 4099, 100), (70, 513, 3),
                                         (3, 32000, 64), (2, 60001, 512), (3, 131072, 20), (2, 262147, 33)])
def test_distill_loss(n, vocab, top, dtype, tau):
    _distill_check(*_distill_inputs(n, vocab, top, dtype), tau)


@pytest.mark.parametrize("dtype", DTYPES)
def test_distill_loss_strided_rows_and_leading_dims(dtype):
    import torch
    from oxitorch_b200 import functional as F
    logits, teacher, ids = _distill_inputs(6, 700, 9, dtype)
    wide = torch.full((6, 711), float("nan"), device="cuda", dtype=logits.dtype)
    for at in (0, 3):
        view = wide[:, at:at + 700]
        view.copy_(logits)
        _distill_check(view, teacher, ids, 1.0)
        wide.fill_(float("nan"))
    a = F.distill_loss(logits, teacher, ids, 1.5)
    b = F.distill_loss(logits.view(2, 3, 700), teacher.view(2, 3, 9), ids.view(2, 3, 9).int(), 1.5)
    assert a == b
    _distill_check(logits, teacher, ids, 1.0, total_rows=50)


@pytest.mark.parametrize("dtype", DTYPES)
def test_distill_loss_rows_without_a_teacher(dtype):
    """Their logits may hold anything; an absent entry's id is never followed."""
    import torch
    logits, teacher, ids = _distill_inputs(5, 300, 8, dtype)
    ids[0], ids[3] = -1, 2
    ids[3] = torch.arange(8, device="cuda")
    teacher[3] = float("-inf")
    logits[0], logits[3] = float("nan"), float("inf")
    clean = logits.clone()
    clean[0], clean[3] = 0.0, 0.0
    from oxitorch_b200 import functional as F
    leaf = logits.detach().requires_grad_()
    loss = F.distill_loss(leaf, teacher, ids)
    (grad,) = torch.autograd.grad(loss, leaf)
    want = R.distill(_n(clean), _n(teacher), ids.cpu().numpy(), 1.0)
    _check(loss, want[0], want[2], "loss")
    _check(grad, want[1], want[3], "dlogits")
    assert (grad[0] == 0).all() and (grad[3] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_distill_loss_masked_logits(dtype):
    """Student logits of -inf or the type's lowest value have probability 0; teacher
    entries of the lowest value too."""
    import torch
    logits, teacher, ids = _distill_inputs(4, 500, 6, dtype)
    ids[:] = torch.arange(6, device="cuda") * 3
    logits[:, 100:200] = float("-inf")
    logits[:, 300:400] = torch.finfo(logits.dtype).min
    teacher[1, 2:] = torch.finfo(torch.float32).min
    teacher[2, 1:] = float("-inf")
    for tau in (1.0, 0.5):
        grad = _distill_check(logits, teacher, ids, tau)
        assert (grad[:, 100:200] == 0).all() and (grad[:, 300:400] == 0).all()
    # a masked token that the teacher wants: infinitely wrong, its gradient is -p
    ids[0, 0] = 150
    from oxitorch_b200 import functional as F
    leaf = logits.detach().requires_grad_()
    loss = F.distill_loss(leaf, teacher, ids)
    assert torch.isposinf(loss)
    (grad,) = torch.autograd.grad(loss, leaf)
    assert torch.isfinite(grad.float()).all() and grad[0, 150] < 0


def test_distill_loss_repeated_ids_add_up():
    import torch
    logits, teacher, ids = _distill_inputs(6, 200, 40, "float32")
    g = np.random.default_rng(5)
    ids = torch.from_numpy(g.integers(0, 12, (6, 40))).cuda()
    _distill_check(logits, teacher, ids, 1.0)
    ids[:] = 7
    _distill_check(logits, teacher, ids, 1.0)


def test_distill_loss_bad_values():
    import torch
    from oxitorch_b200 import _native as N, functional as F
    logits, teacher, ids = _distill_inputs(4, 200, 5, "float32")
    ids[:, 0] = 3
    bad = ids.clone()
    bad[2, 1] = 200
    flag = torch.zeros(4, dtype=torch.int32, device="cuda")
    loss, grad = F.distill_loss_fwd(logits, teacher, bad, flag=flag)
    assert torch.isnan(loss).all() and torch.isnan(grad[2]).all() and torch.isfinite(grad[[0, 1, 3]]).all()
    with pytest.raises(RuntimeError, match="index 200 out of range for dim 1 of size 200"):
        N.check(N.load().oxc_check_error_flag(flag.data_ptr(), torch.cuda.current_stream().cuda_stream, 10000))
    t = teacher.clone()
    t[1, 0] = float("nan")
    loss, grad = F.distill_loss_fwd(logits, t, ids)
    assert torch.isnan(loss).all() and torch.isnan(grad[1]).all() and torch.isfinite(grad[[0, 2, 3]]).all()
    x = logits.clone()
    x[3, 17] = float("nan")
    loss, grad = F.distill_loss_fwd(x, teacher, ids)
    assert torch.isnan(loss).all() and torch.isnan(grad[3]).all() and torch.isfinite(grad[:3]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_distill_loss_scaled_and_twice(dtype):
    import torch
    from oxitorch_b200 import functional as F
    logits, teacher, ids = _distill_inputs(7, 900, 12, dtype)
    leaf = logits.detach().requires_grad_()
    loss = F.distill_loss(leaf, teacher, ids)
    (a,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    first = a.clone()
    (b,) = torch.autograd.grad(0.25 * loss, leaf, retain_graph=True)
    (c,) = torch.autograd.grad(loss, leaf)
    assert torch.equal(a, first) and torch.equal(c, first) and torch.equal(b, (first.float() * 0.25).to(b.dtype))
    (d,) = torch.autograd.grad(3.0 * F.distill_loss(leaf, teacher, ids), leaf)
    assert torch.equal(d, (first.float() * 3.0).to(d.dtype))


def test_distill_loss_no_rows_no_entries_and_refusals():
    import torch
    from oxitorch_b200 import functional as F
    x = torch.randn(3, 10, device="cuda").requires_grad_()
    none = torch.empty(3, 0, device="cuda")
    loss = F.distill_loss(x, none, none.long())
    (g,) = torch.autograd.grad(loss, x)
    assert loss == 0 and (g == 0).all()
    e = torch.empty(0, 10, device="cuda")
    assert F.distill_loss(e, e[:, :2], e[:, :2].long(), total_rows=4) == 0
    t, i = torch.zeros(3, 2, device="cuda"), torch.zeros(3, 2, dtype=torch.int64, device="cuda")
    for bad in (lambda: F.distill_loss(x, t, i[:2]), lambda: F.distill_loss(x, t[:, :1], i),
                lambda: F.distill_loss(x, t, i.float()), lambda: F.distill_loss(x, t, i, 0.0),
                lambda: F.distill_loss(x.half(), t, i), lambda: F.distill_loss(x, t, i, total_rows=2),
                lambda: F.distill_loss(x, t.cpu(), i), lambda: F.distill_loss(x[0], t[0], i[0]),
                lambda: F.distill_loss(x[:, :0], t, i)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        many = torch.zeros(3, 5000, device="cuda")
        F.distill_loss(x, many, many.long())


def test_distill_loss_rows_beyond_32_bits():
    import torch
    from oxitorch_b200 import functional as F
    logits, teacher, ids = _distill_inputs(3, 100, 5, "bfloat16")
    apart = 1_200_000_000
    far = torch.empty(2 * apart + 100, dtype=torch.bfloat16, device="cuda").as_strided((3, 100), (apart, 1))
    far.copy_(logits)
    a, b = F.distill_loss_fwd(logits, teacher, ids), F.distill_loss_fwd(far, teacher, ids)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ---- verify_draft -----------------------------------------------------------------------

def _verify_inputs(B, K, V, seed=0, near=0.6):
    g = np.random.default_rng(B * 101 + K * 11 + V + seed)

    def soft(z):
        e = np.exp(z - z.max(-1, keepdims=True))
        return (e / e.sum(-1, keepdims=True)).astype(np.float32)
    z = 2 * g.standard_normal((B, K + 1, V))
    p = soft(z)
    q = soft(z[:, :K] + near * g.standard_normal((B, K, V)))
    tokens = (q / g.exponential(size=(B, K, V))).argmax(-1).reshape(B, K)
    lengths = g.integers(0, K + 1, B)
    return p, q, tokens, g.random((B, K), np.float32), g.exponential(size=(B, V)).astype(np.float32), lengths


def _verify_check(p, q, tokens, u, e, lengths=None):
    import torch
    from oxitorch_b200 import functional as F
    dev = [None if a is None else torch.from_numpy(np.array(a)).cuda() for a in (p, q, tokens, u, e, lengths)]
    out, accepted = F.verify_draft(*dev)
    want, n = R.verify(p, q, tokens, u, e, lengths)
    assert np.array_equal(accepted.cpu().numpy(), n)
    assert np.array_equal(out.cpu().numpy(), want)
    return want, n


@pytest.mark.parametrize("B,K,V", [(1, 0, 7), (1, 1, 1), (3, 1, 5), (17, 4, 33), (5, 7, 4099), (64, 3, 1000),
                                   (2, 12, 50001), (300, 2, 40), (1, 40, 2000)])
def test_verify_draft(B, K, V):
    p, q, tokens, u, e, lengths = _verify_inputs(B, K, V)
    _verify_check(p, q, tokens, u, e, lengths)
    _verify_check(p, q, tokens, u, e)
    _verify_check(p, None, tokens, u, e, lengths)


@pytest.mark.parametrize("B,K,V", [(20, 2, 20001), (20, 2, 20004), (3, 1, 65536), (1, 2, 200003), (40, 1, 16388)])
def test_verify_draft_few_long_rows(B, K, V):
    """Larger CTAs, several of them to a sequence; rows aligned alike and not."""
    p, q, tokens, u, e, lengths = _verify_inputs(B, K, V)
    _verify_check(p, q, tokens, u, e, lengths)
    _verify_check(p, None, tokens, u, e)


def test_verify_draft_ties_equal_rows_and_zero_weights():
    p, q, tokens, u, e, _ = _verify_inputs(6, 3, 64)
    q[:] = p[:, :3]
    u[:] = 0.999
    want, n = _verify_check(p, q, tokens, u, e)  # p = q: all kept
    assert (n == 3).all()
    p[0, :3, :], q[0] = 0.0, 0.0
    p[0, 0, 5] = 1.0
    q[0, 0, 5] = 1.0
    tokens[0] = 9  # probability 0 on both sides: not kept, and p - q leaves nothing: p decides
    want, n = _verify_check(p, q, tokens, u, e)
    assert n[0] == 0 and want[0, 0] == 5
    e[:] = 1.0
    p[1, 3] = 0.0
    p[1, 3, [40, 20, 50]] = 0.25  # equal quotients: the lowest index
    want, n = _verify_check(p, q, tokens, u, e)
    assert want[1, 3] == 20
    p[2, :] = 0.0  # no positive probability anywhere
    want, n = _verify_check(p, q, tokens, u, e)
    assert n[2] == 0 and want[2, 0] == -1


def test_verify_draft_nan_infinite_race_and_bad_tokens():
    import torch
    from oxitorch_b200 import _native as N, functional as F
    p, q, tokens, u, e, _ = _verify_inputs(5, 2, 100)
    p[0, 0, tokens[0, 0]] = np.nan  # not kept
    p[0, 0, :50] = np.nan
    e[1, :10] = 0.0  # an infinite quotient: the first one wins
    e[2, 3:] = np.inf
    _verify_check(p, q, tokens, u, e)
    tokens[3, 0], tokens[4, 1] = 100, -1
    _verify_check(p, q, tokens, u, e)
    _verify_check(p, None, tokens, u, e)
    flag = torch.zeros(4, dtype=torch.int32, device="cuda")
    F.verify_draft(*[torch.from_numpy(np.array(a)).cuda() for a in (p, q, tokens[:, :], u, e)], flag=flag)
    with pytest.raises(RuntimeError, match="out of bounds"):
        N.check(N.load().oxc_check_error_flag(flag.data_ptr(), torch.cuda.current_stream().cuda_stream, 10000))
    lengths = np.array([-5, 9, 0, 1, 2])  # clamped to [0, drafted]
    _verify_check(p, q, np.clip(tokens, 0, 99), u, e, lengths)


def test_verify_draft_strided_probabilities_and_refusals():
    import torch
    from oxitorch_b200 import functional as F
    p, q, tokens, u, e, lengths = _verify_inputs(4, 3, 130)
    d = [torch.from_numpy(np.array(a)).cuda() for a in (p, q, tokens, u, e, lengths)]
    wide = torch.full((4, 7, 133), float("nan"), device="cuda")
    wide[:, :4, 1:131], wide[:, 4:, 1:131] = d[0], d[1]
    a = F.verify_draft(*d)
    b = F.verify_draft(wide[:, :4, 1:131], wide[:, 4:, 1:131], *d[2:])
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    t, q, tok, u, e, n = d
    for bad in (lambda: F.verify_draft(t[:, :3], q, tok, u, e), lambda: F.verify_draft(t, q, tok.int(), u, e),
                lambda: F.verify_draft(t.bfloat16(), q, tok, u, e), lambda: F.verify_draft(t, q, tok, u, e[:, :5]),
                lambda: F.verify_draft(t[0], q, tok, u, e), lambda: F.verify_draft(t, q.cpu(), tok, u, e),
                lambda: F.verify_draft(t, q, tok, u, e, n[:2])):
        with pytest.raises(ValueError):
            bad()
    assert F.verify_draft(t[:0], q[:0], tok[:0], u[:0], e[:0])[0].shape == (0, 4)


# ---- streams, repetition -------------------------------------------------------------------

def test_draft_ops_on_a_side_stream_and_repeated():
    """Results are the same bits on another stream and on every call."""
    import torch
    from oxitorch_b200 import functional as F
    x, gate, h0, dh, dlast, starts = _scan_inputs(2, 1000, 264, "bfloat16", starts=True)
    nx, nr, nw, ndy, ndr = _norm_inputs(500, 1032, "bfloat16")
    lg, te, ids = _distill_inputs(20, 3000, 30, "bfloat16")

    def everything():
        h, last, carry = F.gated_scan_fwd(x, gate, h0, starts)
        y, r, rstd = F.add_rms_norm_fwd(nx, nr, nw)
        return [h, last, *F.gated_scan_bwd(x, gate, carry, dh, dlast, starts), y, r,
                *F.add_rms_norm_bwd(r, nw, rstd, ndy, ndr, "exact"), *F.distill_loss_fwd(lg, te, ids)]
    want = everything()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), side):
        with torch.cuda.stream(stream):
            for _ in range(3):
                got = everything()
        stream.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert __import__("oxitorch_b200")._native.kernel_error_bits() == 0
