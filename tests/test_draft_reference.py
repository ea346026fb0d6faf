"""The 64-bit references of the draft model's operators against differences of
their own forward passes, and the refusals that need no device."""

import numpy as np
import pytest

import draft_reference as R


def _differences(f, a, step=1e-6):
    g = np.zeros_like(a)
    for i in np.ndindex(a.shape):
        keep = a[i]
        a[i] = keep + step
        up = f()
        a[i] = keep - step
        down = f()
        a[i] = keep
        g[i] = (up - down) / (2 * step)
    return g


# central differences of a function of size ~10 with step 1e-6 in 64 bits: the
# rounding 10 * 1e-16 / 1e-6 and the third derivative's 1e-12 stay below 1e-7
TOL = dict(rtol=1e-6, atol=1e-7)


def test_add_rms_norm_gradient_is_the_difference_quotient():
    g = np.random.default_rng(1)
    x, res, w = g.standard_normal((3, 7)), g.standard_normal((3, 7)), g.uniform(0.5, 1.5, 7)
    dy, dr = g.standard_normal((3, 7)), g.standard_normal((3, 7))

    def f():
        y, r, _ = R.add_rms_norm(x, res, w, 1e-3)
        return (y * dy).sum() + (r * dr).sum()
    (d, dw), _ = R.add_rms_norm_grad(x, res, w, 1e-3, dy, dr)
    np.testing.assert_allclose(d, _differences(f, x), **TOL)
    np.testing.assert_allclose(d, _differences(f, res), **TOL)
    np.testing.assert_allclose(dw, _differences(f, w), **TOL)


@pytest.mark.parametrize("packed", [False, True])
def test_gated_scan_gradient_is_the_difference_quotient(packed):
    g = np.random.default_rng(2)
    x, gate, dh = (g.standard_normal((2, 5, 3)) for _ in range(3))
    h0, dlast = g.standard_normal((2, 3)), g.standard_normal((2, 3))
    starts = np.array([[0, 0, 1, 0, 0], [1, 0, 0, 0, 1]], bool) if packed else None

    def f():
        h, last, _ = R.gated_scan(x, gate, h0, starts)
        return (h * dh).sum() + (last * dlast).sum()
    (dx, dg, dh0), _ = R.gated_scan_grad(x, gate, h0, starts, dh, dlast)
    np.testing.assert_allclose(dx, _differences(f, x), **TOL)
    np.testing.assert_allclose(dg, _differences(f, gate), **TOL)
    np.testing.assert_allclose(dh0, _differences(f, h0), **TOL)


@pytest.mark.parametrize("tau", [1.0, 2.5])
def test_distill_gradient_is_the_difference_quotient(tau):
    g = np.random.default_rng(3)
    logits, teacher = g.standard_normal((4, 6)), g.standard_normal((4, 3))
    ids = np.array([[0, 3, 5], [2, -1, 4], [-1, -1, -1], [1, 1, 2]])

    def f():
        return R.distill(logits, teacher, ids, tau)[0]
    np.testing.assert_allclose(R.distill(logits, teacher, ids, tau)[1], _differences(f, logits), **TOL)


def test_verified_tokens_follow_the_target():
    """Drafting from q and verifying against p samples from p: the frequencies
    of the first token over many given random numbers are p's."""
    g = np.random.default_rng(4)
    n, p, q = 40000, np.array([0.5, 0.3, 0.2]), np.array([0.1, 0.3, 0.6])
    target = np.broadcast_to(p.astype(np.float32), (n, 2, 3))
    draft = np.broadcast_to(q.astype(np.float32), (n, 1, 3))
    tokens = g.choice(3, size=(n, 1), p=q)
    out, accepted = R.verify(target, draft, tokens, g.random((n, 1), np.float32),
                             g.exponential(size=(n, 3)).astype(np.float32))
    counts = np.bincount(out[:, 0], minlength=3) / n
    # five standard deviations of a frequency, sqrt(0.25 / n) each at most
    np.testing.assert_allclose(counts, p, atol=5 * np.sqrt(0.25 / n))
    assert abs(accepted.mean() - np.minimum(p, q).sum()) < 5 * np.sqrt(0.25 / n)


def test_refusals_without_a_device():
    import torch
    from oxitorch_b200 import functional as F
    x = torch.zeros(2, 4)
    for call in (lambda: F.add_rms_norm_fwd(x, x, torch.ones(4)),
                 lambda: F.add_rms_norm_quant(x, x, torch.ones(4)),
                 lambda: F.gated_scan(x[None], x[None]),
                 lambda: F.gated_step(x, x, x),
                 lambda: F.distill_loss(x, x, torch.zeros(2, 4, dtype=torch.int64)),
                 lambda: F.verify_draft(x[None], None, None, None, None)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(TypeError):
        F.gated_scan([1.0], [1.0])
    with pytest.raises(ValueError, match="grad mode"):
        F.add_rms_norm(x, x, torch.ones(4), grad_mode="half")


def test_abi_refusals_and_sizes():
    from oxitorch_b200 import _native as N
    L = N.load(require_device=False)
    assert L.oxc_add_rms_norm_bwd_workspace_size(0, 8) == 0
    assert L.oxc_gated_scan_carry_size(2, 0, 8) == 0
    assert L.oxc_gated_scan_carry_size(2, 1, 8) == 16
    bad = N.ERR_INVALID_ARGUMENT
    assert L.oxc_add_rms_norm_fwd(None, 0, None, 0, None, None, None, None, 2, 4, 7, 1e-6, None) == bad
    assert "dtype" in N.last_error()
    assert L.oxc_add_rms_norm_fwd(None, 0, None, 0, None, None, None, None, 2, 4, 0, 1e-6, None) == bad
    assert L.oxc_add_rms_norm_fwd(None, 0, None, 0, None, None, None, None, 2, 40000, 0, 1e-6, None) \
        == N.ERR_NOT_IMPLEMENTED
    assert L.oxc_add_rms_norm_quant(None, 0, None, 0, None, None, None, None, 2, 4, 64, 0, 1e-6, None) == bad
    assert "block" in N.last_error()
    assert L.oxc_add_rms_norm_bwd(None, None, None, None, 0, None, 0, None, None, None, 2, 4, 0, 5, None,
                                  0, None) == bad
    assert L.oxc_add_rms_norm_bwd(None, None, None, None, 0, None, 0, None, None, None, 2, 4, 0, 1, None,
                                  0, None) == bad
    assert "workspace" in N.last_error()
    zeros = [0] * 2
    assert L.oxc_gated_scan_fwd(None, *zeros, None, *zeros, None, None, None, None, None, 2, 3, 4, 0, None, 0,
                                None) == bad
    assert L.oxc_gated_scan_fwd(None, *zeros, None, *zeros, None, None, None, None, None, -1, 3, 4, 0, None, 0,
                                None) == bad
    assert L.oxc_gated_step(None, 0, None, 0, None, None, None, 2, 4, 9, None) == bad
    for tau in (0.0, -1.0, float("nan"), float("inf")):
        assert L.oxc_distill_loss(None, 0, None, None, 1, tau, None, None, None, None, 2, 4, 2, 0, None, None) == bad
        assert "temperature" in N.last_error()
    assert L.oxc_distill_loss(None, 0, None, None, 1, 1.0, None, None, None, None, 4, 4, 2, 0, None, None) == bad
    assert "total_rows" in N.last_error()
    assert L.oxc_scale_by(None, 4, 0, None, None) == bad
    assert L.oxc_verify_draft(None, 0, 0, None, 0, 0, None, None, None, None, 2, 3, 4, None, None, None, None) == bad
    # nothing to do is no error
    assert L.oxc_gated_step(None, 0, None, 0, None, None, None, 0, 4, 0, None) == N.OK
    assert L.oxc_scale_by(None, 0, 0, None, None) == N.OK
    assert L.oxc_verify_draft(None, 0, 0, None, 0, 0, None, None, None, None, 0, 3, 4, None, None, None, None) == N.OK
