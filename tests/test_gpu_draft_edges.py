"""The recurrent draft model's operators where they can go wrong: ties of the
8-bit codes, the widest rows, variates of zero, NaN beside a sequence start,
long teacher lists, derivatives that there are none of, and operands that do not
fit each other.  Error bounds come from tests/draft_reference.py."""

import numpy as np
import pytest

import draft_reference as R
from test_gpu_draft import DTYPES, _check, _distill_inputs, _n, _norm_inputs, _scan_inputs, _t, _verify_inputs

pytestmark = pytest.mark.gpu


# ---- add_rms_norm --------------------------------------------------------------------

@pytest.mark.parametrize("block", [128, None])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,offset", [(24576, 1024, 0), (24576, 1001, 0), (24576, 1000, 1)])
def test_add_rms_norm_quant_codes_are_quotients(rows, cols, offset, dtype, block):
    """The code is y / scale, an f32 division, rounded to nearest even, with the y that
    add_rms_norm_fwd gives: bit for bit, by vectors, by shifted vectors and by single
    elements.  Of 24 million codes several lie within an f32 rounding of a tie."""
    import torch
    from oxitorch_b200 import functional as F
    g = torch.Generator(device="cuda")
    g.manual_seed(rows + cols + offset)

    def rows_at(t):  # `offset` elements after an aligned address
        wide = torch.empty(rows, cols + 4, device="cuda", dtype=t.dtype)
        wide[:, offset:offset + cols] = t
        return wide[:, offset:offset + cols]
    x = rows_at(torch.randn(rows, cols, device="cuda", generator=g).to(getattr(torch, dtype)))
    res = rows_at(torch.randn(rows, cols, device="cuda", generator=g) * 3)
    w = torch.rand(cols, device="cuda", generator=g) + 0.5
    q, scale, _ = F.add_rms_norm_quant(x, res, w, 1e-5, block=block)
    y, _, _ = F.add_rms_norm_fwd(rows_at(x.float()), res, w, 1e-5)
    b = block or cols
    largest = torch.stack([v.abs().amax(-1) for v in y.split(b, -1)], -1)
    want = (largest / torch.full_like(largest, R.E4M3_MAX)).clamp(min=2.0 ** -126)
    assert torch.equal(scale, want)
    codes = (y / want.repeat_interleave(b, -1)[:, :cols]).to(torch.float8_e4m3fn)
    off = int((codes.view(torch.uint8) != q.view(torch.uint8)).sum())
    assert off == 0, f"{off} codes of {codes.numel()}"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [32763, 32765, 32766, 32767])
def test_add_rms_norm_widest_rows(cols, dtype):
    """Just under the limit: a row that starts 3 elements after an aligned address
    touches 8193 vectors of 4."""
    import torch
    from oxitorch_b200 import functional as F
    x, res, w, dy, dr = _norm_inputs(6, cols, dtype, seed=5)
    want_y, _, _ = R.add_rms_norm(_n(x), _n(res), _n(w), 1e-5)
    y, r, rstd = F.add_rms_norm_fwd(x, res, w, 1e-5)
    _check(y, want_y, 56 * R.EPS * np.abs(want_y), "y")
    assert (r == x.float() + res).all()
    for mode in ("ref", "exact"):
        dx, dres, dw = F.add_rms_norm_bwd(r, w, rstd, dy, dr, mode)
        (d, want_dw), (bd, bdw) = R.add_rms_norm_grad(_n(x), _n(res), _n(w), 1e-5, _n(dy), _n(dr), mode == "exact")
        _check(dres, d, bd, "dresidual")
        _check(dx, d, bd, "dx")
        _check(dw, want_dw, bdw, "dweight")
    for block in (128, None):
        q, scale, r = F.add_rms_norm_quant(x, res, w, 1e-5, block=block)
        assert (r == x.float() + res).all()
        want = R.block_scales(want_y, block)
        _check(scale, want, 60 * R.EPS * want, "scale")
        z = want_y / np.repeat(want, block or cols, -1)[:, :cols]
        _check(q.to(torch.float32), z, R.e4m3_half_step(z) * (1 + 2.0 ** -10) + 120 * R.EPS * np.abs(z), "q")


# ---- verify_draft --------------------------------------------------------------------

@pytest.mark.parametrize("B,V", [(40, 50), (3, 40003), (200, 20004)])
def test_verify_draft_zero_variates_pick_no_token_without_weight(B, V):
    """A variate of zero gives a positive weight an infinite quotient and a weight of
    zero nothing: the token after the kept ones always has weight."""
    import torch
    from oxitorch_b200 import functional as F
    p, q, tokens, u, e, lengths = _verify_inputs(B, 2, V, seed=9)
    g = np.random.default_rng(B + V)
    e[g.random((B, V)) < 4 / V] = 0.0
    e[0], e[1, : V // 2] = 0.0, 0.0
    for draft in (q, None):
        dev = [None if a is None else torch.from_numpy(np.array(a)).cuda() for a in (p, draft, tokens, u, e, lengths)]
        out, accepted = (a.cpu().numpy() for a in F.verify_draft(*dev))
        for b in range(B):
            n, j = int(lengths[b]), int(accepted[b])
            w = p[b, j].copy()
            if j < n and draft is not None:
                w = p[b, j] - q[b, j]
            elif j < n:
                w[tokens[b, j]] = 0.0
            some = w > 0
            assert some.any()
            with np.errstate(divide="ignore", invalid="ignore"):
                score = np.where(some, w / e[b], -1.0)
            assert out[b, j] == score.argmax() and w[out[b, j]] > 0


# ---- gated_scan ----------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [72, 130, 256])
def test_gated_scan_starts_stop_a_nan_gate(D, dtype):
    """A NaN gate at a start or at one of the tokens after it, in the same warp's eight
    tokens, the same chunk or a later one, does not reach what lies before the start."""
    import torch
    from oxitorch_b200 import functional as F
    T = 300
    x, gate, h0, dh, dlast, _ = _scan_inputs(1, T, D, dtype)
    for new in (1, 64, 130, 255):
        starts = torch.zeros(1, T, dtype=torch.bool, device="cuda")
        starts[:, new] = True
        (wx, wg, w0), (bx, bg, b0) = R.gated_scan_grad(_n(x)[:, :new], _n(gate)[:, :new], _n(h0), None,
                                                       _n(dh)[:, :new], None)
        want, _, bound = R.gated_scan(_n(x)[:, :new], _n(gate)[:, :new], _n(h0))
        for after in (0, 1, 2, 5, 6, 7, 11, 40):
            bad = gate.clone()
            bad[:, new + after] = float("nan")
            leaves = [t.clone().requires_grad_() for t in (x, bad, h0)]
            h, last = F.gated_scan(*leaves, starts)
            dx, dg, dh0 = torch.autograd.grad((h, last), leaves, (dh, dlast))
            where = f"NaN {after} after the start at {new}"
            _check(h[:, :new], want, bound, "h, " + where)
            assert torch.isnan(h[:, new + after:].float()).all() and torch.isnan(last).all()
            _check(dx[:, :new], wx, bx, "dx, " + where)
            _check(dg[:, :new], wg, bg, "dgate, " + where)
            _check(dh0, w0, b0, "dh0, " + where)


# ---- distill_loss --------------------------------------------------------------------

def _distill_against_reference(logits, teacher, ids, tau):
    import torch
    from oxitorch_b200 import functional as F
    leaf = logits.detach().requires_grad_()
    loss = F.distill_loss(leaf, teacher, ids, tau)
    (grad,) = torch.autograd.grad(loss, leaf)
    want = R.distill(_n(logits), _n(teacher), ids.cpu().numpy(), tau)
    _check(loss, want[0], want[2], "loss")
    _check(grad, want[1], want[3], "dlogits")


@pytest.mark.parametrize("dtype,vocab", [("float32", 290000), ("float32", 300000), ("float32", 320000),
                                         ("float32", 327680), ("bfloat16", 600000), ("bfloat16", 650000)])
def test_distill_loss_long_teacher_lists_beside_wide_rows(dtype, vocab):
    """The longest lists take 80 KB of shared memory beside a row's part of up to 160 KB."""
    for top in (2900, 4096):
        _distill_against_reference(*_distill_inputs(2, vocab, top, dtype), 1.0)


# ---- derivatives ---------------------------------------------------------------------

def test_forward_mode_derivatives_are_refused():
    """A tangent that would be dropped is an error, whether or not the tensor also wants
    a gradient."""
    import torch
    import torch.autograd.forward_ad as fwAD
    from oxitorch_b200 import functional as F
    x, t = torch.randn(2, 4, 8, device="cuda"), torch.randn(2, 4, 8, device="cuda")
    h0, ones = torch.zeros(2, 8, device="cuda"), torch.ones(8, device="cuda")
    tl, ti = torch.zeros(2, 4, 2, device="cuda"), torch.arange(2, device="cuda").expand(2, 4, 2)
    with fwAD.dual_level():
        d, d0, dl = fwAD.make_dual(x, t), fwAD.make_dual(h0, h0.clone()), fwAD.make_dual(tl, tl.clone())
        for call in (lambda: F.gated_scan(d, x), lambda: F.gated_scan(x, d), lambda: F.gated_scan(x, x, d0),
                     lambda: F.distill_loss(d, tl, ti), lambda: F.distill_loss(x, dl, ti),
                     lambda: F.gated_step(d[:, 0], x[:, 0], h0), lambda: F.gated_step(x[:, 0], x[:, 0], d0),
                     lambda: F.add_rms_norm(d, x, ones), lambda: F.add_rms_norm_quant(x, d, ones)):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises((RuntimeError, ValueError)):
                    call()
        # without a tangent nothing is refused inside a level
        F.gated_scan(x, x, h0)
        F.distill_loss(x, tl, ti)
        F.gated_step(x[:, 0], x[:, 0], h0)


def test_add_rms_norm_quant_refuses_to_cut_a_gradient():
    """Its outputs have no gradient, the residual stream among them."""
    import torch
    from oxitorch_b200 import functional as F
    x, w = torch.randn(3, 8, device="cuda"), torch.ones(8, device="cuda")
    for at in range(3):
        args = [x, x, w]
        args[at] = args[at].clone().requires_grad_()
        with pytest.raises(ValueError, match="gradient"):
            F.add_rms_norm_quant(*args)
        with torch.no_grad():
            q, scale, r = F.add_rms_norm_quant(*args)
        assert not r.requires_grad


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("factor", [3.0, 0.1, -0.7])
def test_distill_loss_gradient_is_the_same_whichever_backward_asks(dtype, factor):
    """The factor on the loss gives the same bits in the first backward and in later
    ones, within its own rounding of the gradient for a factor of 1."""
    import torch
    from oxitorch_b200 import functional as F
    logits, teacher, ids = _distill_inputs(9, 1003, 12, dtype)
    leaf = logits.detach().requires_grad_()
    loss = F.distill_loss(leaf, teacher, ids, 2.0)
    (first,) = torch.autograd.grad(factor * loss, leaf, retain_graph=True)
    (second,) = torch.autograd.grad(factor * loss, leaf, retain_graph=True)
    (one,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    (third,) = torch.autograd.grad(factor * loss, leaf)
    assert torch.equal(first, second) and torch.equal(first, third)
    _, want, _, bound = R.distill(_n(logits), _n(teacher), ids.cpu().numpy(), 2.0)
    _check(one, want, bound, "factor 1")
    f = float(np.float32(factor))
    # the rounding for a factor of 1, times the factor, and (in _check) the second one
    once = 2.0 ** -8 * (np.abs(want) + bound) if dtype == "bfloat16" else R.EPS * np.abs(want)
    _check(first, f * want, abs(f) * (bound + once + 2.0 ** -133), "factor")


# ---- operands that do not fit each other ---------------------------------------------

def test_gated_scan_bwd_refuses_operands_that_do_not_fit():
    import torch
    from oxitorch_b200 import functional as F
    x = torch.randn(2, 130, 8, device="cuda")
    gate = torch.randn_like(x)
    _, _, carry = F.gated_scan_fwd(x, gate)
    _, _, short = F.gated_scan_fwd(x[:, :64], gate[:, :64])
    F.gated_scan_bwd(x, gate, carry)
    for bad in (lambda: F.gated_scan_bwd(x, gate[:, :129], carry), lambda: F.gated_scan_bwd(x, gate[:1], carry),
                lambda: F.gated_scan_bwd(x, gate.bfloat16(), carry), lambda: F.gated_scan_bwd(x, gate.cpu(), carry),
                lambda: F.gated_scan_bwd(x, gate, short), lambda: F.gated_scan_bwd(x, gate, carry.bfloat16()),
                lambda: F.gated_scan_bwd(x, gate, carry.repeat_interleave(2)[::2]),
                lambda: F.gated_scan_bwd(x, gate, carry.cpu()), lambda: F.gated_scan_bwd(x[0], gate[0], carry)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        F.gated_scan_bwd(x, gate, None)


def test_add_rms_norm_bwd_refuses_operands_that_do_not_fit():
    import torch
    from oxitorch_b200 import functional as F
    x, w = torch.randn(5, 3, 16, device="cuda"), torch.ones(16, device="cuda")
    _, r, rstd = F.add_rms_norm_fwd(x, x, w)
    want = F.add_rms_norm_bwd(r, w, rstd, x)
    for bad in (lambda: F.add_rms_norm_bwd(r, w[:8], rstd, x), lambda: F.add_rms_norm_bwd(r, w.bfloat16(), rstd, x),
                lambda: F.add_rms_norm_bwd(r, w, rstd[:2], x), lambda: F.add_rms_norm_bwd(r, w, rstd.double(), x),
                lambda: F.add_rms_norm_bwd(r, w.cpu(), rstd, x), lambda: F.add_rms_norm_bwd(r, w, rstd.cpu(), x),
                lambda: F.add_rms_norm_bwd(r[0], w, rstd, x), lambda: F.add_rms_norm_bwd(r, w, rstd, x, grad_mode="half"),
                lambda: F.add_rms_norm_bwd(r[0, 0, 0], w, rstd, x[0, 0, 0])):
        with pytest.raises(ValueError):
            bad()
    # strided ones are read where they are
    apart = torch.full((5, 3, 2), float("nan"), device="cuda")
    apart[..., 0] = rstd
    twice = torch.stack([w, w * 9], -1)
    got = F.add_rms_norm_bwd(r, twice[:, 0], apart[..., 0], x)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_flags_and_factors_that_do_not_fit_are_refused():
    import torch
    from oxitorch_b200 import functional as F
    p = torch.softmax(torch.randn(2, 2, 10, device="cuda"), -1)
    tok, u, e = torch.zeros(2, 1, dtype=torch.int64, device="cuda"), torch.rand(2, 1, device="cuda"), torch.ones(2, 10, device="cuda")
    x, tl, ti = torch.randn(3, 10, device="cuda"), torch.zeros(3, 2, device="cuda"), torch.zeros(3, 2, dtype=torch.int64, device="cuda")
    flag = torch.zeros(8, dtype=torch.int32, device="cuda")
    F.verify_draft(p, p[:, :1], tok, u, e, flag=flag[:4])
    F.distill_loss_fwd(x, tl, ti, grad_loss=torch.ones(1, device="cuda"), flag=flag[4:])
    F.distill_loss_fwd(x, tl, ti, grad_loss=torch.ones((), device="cuda"))
    for bad in (flag[::2], flag, flag[:4].long(), flag[:4].cpu()):
        with pytest.raises(ValueError):
            F.verify_draft(p, p[:, :1], tok, u, e, flag=bad)
        with pytest.raises(ValueError):
            F.distill_loss_fwd(x, tl, ti, flag=bad)
    for bad in (torch.ones(2, device="cuda"), torch.ones(1, device="cuda").double(), torch.ones(1),
                torch.ones(0, device="cuda")):
        with pytest.raises(ValueError):
            F.distill_loss_fwd(x, tl, ti, grad_loss=bad)


# ---- distill_loss: many rows to a cluster, and the kernel for any width ------------------

def _mixed_rows(n, vocab, top, dtype):
    """Rows as in training, among them ones without a teacher, with an entry of -inf,
    with ids listed twice or more, and with masked logits."""
    import torch
    logits, teacher, ids = _distill_inputs(n, vocab, top, dtype)
    ids[::5, top // 2:] = ids[::5, :top - top // 2]
    ids[1::7] = -1
    teacher[2::9, 0] = float("-inf")
    logits[3::11, vocab // 3:vocab // 2] = float("-inf")
    keep = torch.zeros_like(ids, dtype=torch.bool)
    keep[3::11] = (ids[3::11] >= vocab // 3) & (ids[3::11] < vocab // 2)
    ids[keep] = 0
    return logits, teacher, ids


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,vocab,top", [(9001, 1003, 40), (1501, 32001, 64), (333, 131073, 300)])
def test_distill_loss_many_rows_to_a_cluster(n, vocab, top, dtype):
    """Several rows in turn through each cluster of 1, 2, 4 or 8 CTAs, not the same
    number for each."""
    _distill_against_reference(*_mixed_rows(n, vocab, top, dtype), 1.5)


@pytest.mark.parametrize("dtype,vocab", [("float32", 330001), ("bfloat16", 660001)])
def test_distill_loss_rows_wider_than_a_cluster_holds(dtype, vocab):
    import torch
    from oxitorch_b200 import functional as F
    logits, teacher, ids = _mixed_rows(13, vocab, 50, dtype)
    for tau in (1.0, 0.7):
        _distill_against_reference(logits, teacher, ids, tau)
    ids[:, 0] = 3
    clean = ids.clone()
    ids[4, 1] = vocab
    t = teacher.clone()
    t[6, 0] = float("nan")
    x = logits.clone()
    x[8, 17] = float("nan")
    x[10] = float("-inf")
    flag = torch.zeros(4, dtype=torch.int32, device="cuda")
    loss, grad = F.distill_loss_fwd(x, t, ids, flag=flag)
    assert torch.isnan(loss).all() and flag.tolist() == [2, vocab, 0, vocab]
    bad = [4, 6, 8, 10]
    assert torch.isnan(grad[bad]).all()
    good = [i for i in range(13) if i not in bad]
    _, want = F.distill_loss_fwd(logits, teacher, clean)
    assert torch.equal(grad[good], want[good])


# ---- graphs --------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
def test_draft_ops_captured_in_a_graph(dtype):
    """A replay on new inputs in the captured buffers gives the bits of an eager call."""
    import torch
    from oxitorch_b200 import functional as F
    scan, norm = _scan_inputs(2, 700, 264, dtype, starts=True), _norm_inputs(300, 1032, dtype)
    dist = _distill_inputs(40, 33000, 30, dtype)
    ver = [torch.from_numpy(np.array(a)).cuda() for a in _verify_inputs(9, 3, 20003)]

    def everything():
        x, gate, h0, dh, dlast, starts = scan
        h, last, carry = F.gated_scan_fwd(x, gate, h0, starts)
        nx, nr, nw, ndy, ndr = norm
        y, r, rstd = F.add_rms_norm_fwd(nx, nr, nw)
        q, scale, _ = F.add_rms_norm_quant(nx, nr, nw)
        out = torch.empty_like(h0)
        step = F.gated_step(x[:, 3], gate[:, 3], h0, out=out)
        p, d, tokens, u, e, lengths = ver
        return [h, last, *F.gated_scan_bwd(x, gate, carry, dh, dlast, starts), y, r,
                *F.add_rms_norm_bwd(r, nw, rstd, ndy, ndr, "exact"), q.view(torch.uint8), scale, step, out,
                *F.distill_loss_fwd(*dist), *F.verify_draft(p, d, tokens, u, e, lengths)]
    everything()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = everything()
    for seed in (1, 2):
        for t, s in zip(scan[:5], _scan_inputs(2, 700, 264, dtype, seed)[:5]):
            t.copy_(s)
        for t, s in zip(norm, _norm_inputs(300, 1032, dtype, seed)):
            t.copy_(s)
        for t, s in zip(dist, _distill_inputs(40, 33000, 30, dtype, seed)):
            t.copy_(s)
        for t, s in zip(ver, _verify_inputs(9, 3, 20003, seed)):
            t.copy_(torch.from_numpy(np.array(s)))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in got]
        assert all(torch.equal(a, b) for a, b in zip(kept, everything()))
    assert __import__("oxitorch_b200")._native.kernel_error_bits() == 0
