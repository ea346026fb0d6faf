"""The 64-bit references of the selective state space model's operators against
differences of their own forward passes, and the refusals that need no device."""

import numpy as np
import pytest

import selective_reference as R
from test_draft_reference import TOL, _differences


@pytest.mark.parametrize("silu", [True, False])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("width", [1, 2, 4])
def test_causal_conv_gradient_is_the_difference_quotient(width, packed, silu):
    g = np.random.default_rng(width)
    x, dy = g.standard_normal((2, 6, 3)), g.standard_normal((2, 6, 3))
    w, bias = g.standard_normal((3, width)), g.standard_normal(3)
    x0, dlast = g.standard_normal((2, width - 1, 3)), g.standard_normal((2, width - 1, 3))
    starts = np.array([[0, 0, 1, 0, 0, 1], [1, 0, 0, 0, 1, 0]], bool) if packed else None

    def f():
        y, last, _ = R.causal_conv(x, w, bias, x0, starts, silu)
        return (y * dy).sum() + (last * dlast).sum()
    got, _ = R.causal_conv_grad(x, w, bias, x0, starts, silu, dy, dlast)
    for d, a in zip(got, (x, w, bias, x0)):
        np.testing.assert_allclose(d, _differences(f, a), **TOL)


@pytest.mark.parametrize("packed", [False, True])
def test_causal_conv_of_packed_rows_is_that_of_their_sequences(packed):
    g = np.random.default_rng(5)
    x, w = g.standard_normal((1, 9, 2)), g.standard_normal((2, 4))
    starts = np.zeros((1, 9), bool)
    starts[0, [0, 2, 3]] = True
    y, last, _ = R.causal_conv(x, w, None, None, starts)
    for lo, hi in ((0, 2), (2, 3), (3, 9)):
        np.testing.assert_array_equal(y[:, lo:hi], R.causal_conv(x[:, lo:hi], w)[0])
    np.testing.assert_array_equal(last, R.causal_conv(x[:, 3:], w)[1])


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("packed", [False, True])
def test_selective_scan_gradient_is_the_difference_quotient(packed, gated):
    g = np.random.default_rng(7)
    b, T, d, n = 2, 5, 3, 2
    args = {"x": g.standard_normal((b, T, d)), "delta": g.standard_normal((b, T, d)),
            "A": -g.uniform(0.2, 2.0, (d, n)), "B": g.standard_normal((b, T, n)), "C": g.standard_normal((b, T, n)),
            "D": g.standard_normal(d), "z": g.standard_normal((b, T, d)) if gated else None,
            "delta_bias": g.standard_normal(d), "h0": g.standard_normal((b, d, n))}
    starts = np.array([[0, 0, 1, 0, 0], [1, 0, 0, 0, 1]], bool) if packed else None
    dy, dlast = g.standard_normal((b, T, d)), g.standard_normal((b, d, n))

    def f():
        s = R.Scan(**args, starts=starts)
        return (s.out()[0] * dy).sum() + (s.last * dlast).sum()
    got, _ = R.Scan(**args, starts=starts).grad(dy, dlast)
    for k, a in args.items():
        if a is not None:
            np.testing.assert_allclose(got[k], _differences(f, a), err_msg=k, **TOL)


@pytest.mark.parametrize("kl,tau", [(0.0, 1.0), (0.3, 1.0), (0.1, 2.5)])
def test_policy_gradient_is_the_difference_quotient(kl, tau):
    g = np.random.default_rng(3)
    logits, adv = g.standard_normal((6, 5)), np.array([1.0, -1.0, 2.0, -0.5, 1.0, 0.7])
    tokens = np.array([0, 3, 4, 2, -1, 1])
    logp = R.policy(logits, tokens, adv, adv, tau=tau)[0][1]
    old, ref = logp - np.array([0.5, 0.5, -0.5, -0.5, 0.0, 0.1]), logp + 0.3 * g.standard_normal(6)

    def f():
        return R.policy(logits, tokens, old, adv, ref, (0.2, 0.3), kl, tau)[0][0]
    grad = R.policy(logits, tokens, old, adv, ref, (0.2, 0.3), kl, tau)[0][2]
    np.testing.assert_allclose(grad, _differences(f, logits), **TOL)
    assert not grad[4].any()
    if kl == 0:
        assert not grad[0].any() and not grad[3].any()  # clipped from above, and from below


def test_sizes_that_are_refused():
    """Statuses that come before anything touches the device."""
    from oxitorch_b200 import _native as N
    L = N.load(require_device=False)
    z = [0] * 2
    conv = lambda w, dt=0, b=1: L.oxc_causal_conv_fwd(16, *z, 16, None, None, None, 16, None, b, 1, 4, w, 1, dt, None)  # noqa: E731
    assert conv(9) == N.ERR_NOT_IMPLEMENTED and conv(0) == N.ERR_INVALID_ARGUMENT
    assert conv(4, dt=7) == N.ERR_INVALID_ARGUMENT and conv(4, b=-1) == N.ERR_INVALID_ARGUMENT
    assert L.oxc_causal_conv_fwd(16, *z, None, None, None, None, 16, None, 1, 1, 4, 4, 1, 0, None) == N.ERR_INVALID_ARGUMENT
    assert L.oxc_causal_conv_fwd(16, *z, 16, None, None, None, 16, None, 2 ** 20, 2 ** 20, 2 ** 20, 4, 1, 0,
                                 None) == N.ERR_NOT_IMPLEMENTED
    assert L.oxc_causal_conv_bwd(16, *z, 16, None, None, None, None, *z, None, 16, None, 16, 1, 1, 4, 4, 1, 0, None, 0,
                                 None) == N.ERR_INVALID_ARGUMENT  # no workspace
    assert L.oxc_causal_conv_step(16, 0, 16, None, None, None, 16, 1, 4, 4, 1, 0, None) == N.ERR_INVALID_ARGUMENT
    scan = lambda n, length=1, b=1, d=4: L.oxc_selective_scan_fwd(  # noqa: E731
        16, *z, 16, *z, 16, 16, *z, 16, *z, None, None, *z, None, None, None, None, None, None, b, length, d, n, 0, None, 0,
        None)
    assert scan(129) == N.ERR_NOT_IMPLEMENTED and scan(0) == N.ERR_INVALID_ARGUMENT
    assert scan(16) == N.ERR_INVALID_ARGUMENT  # no y
    assert scan(16, length=2 ** 35) == N.ERR_NOT_IMPLEMENTED
    assert scan(16, b=2 ** 20, d=2 ** 20) == N.ERR_NOT_IMPLEMENTED
    assert L.oxc_selective_scan_bwd(16, *z, 16, *z, 16, 16, *z, 16, *z, None, None, *z, None, None, 16, None, *z, None, 16,
                                    16, 16, 16, 16, None, None, 1, 1, 4, 16, 0, None, 0, None) == N.ERR_INVALID_ARGUMENT
    loss = lambda rows=1, vocab=8, total=1, clip=0.2, kl=0.0, tau=1.0: L.oxc_policy_loss(  # noqa: E731
        None, 0, None, None, 16, None, clip, clip, kl, tau, None, 16, None, None, None, rows, vocab, total, 0, None, None)
    assert loss() == N.ERR_INVALID_ARGUMENT and loss(vocab=2 ** 31) == N.ERR_NOT_IMPLEMENTED
    assert loss(vocab=0) == N.ERR_INVALID_ARGUMENT and loss(total=0) == N.ERR_INVALID_ARGUMENT
    for bad in ({"clip": -0.1}, {"kl": -1.0}, {"kl": float("nan")}, {"tau": 0.0}, {"tau": float("inf")}):
        assert loss(**bad) == N.ERR_INVALID_ARGUMENT


def test_clipping_refuses_tensors_that_overlap():
    """Two gradients on the same memory, one listed twice, an output on another's
    input: refused before anything is launched."""
    from array import array

    from oxitorch_b200 import _native as N
    L = N.load(require_device=False)

    def call(ptrs, sizes, out=None, dtypes=None, max_norm=1.0):
        p, n, d = array("q", ptrs), array("q", sizes), array("i", dtypes or [0] * len(ptrs))
        o = None if out is None else array("q", out)
        need = L.oxc_clip_global_norm_workspace_size(len(ptrs))
        return L.oxc_clip_global_norm(p.buffer_info()[0], None if o is None else o.buffer_info()[0], n.buffer_info()[0],
                                      d.buffer_info()[0], len(ptrs), max_norm, 16, 16, need, None)
    assert call([4096, 4096], [4, 4]) == N.ERR_INVALID_ARGUMENT
    assert "overlap" in N.last_error()
    assert call([4096, 4100], [4, 4]) == N.ERR_INVALID_ARGUMENT
    assert call([4096, 8192], [4, 4], out=[8192, 4096]) == N.ERR_INVALID_ARGUMENT
    assert call([4096, 8192], [4, 4], out=[16384, 16392]) == N.ERR_INVALID_ARGUMENT
    assert call([4096], [4], dtypes=[5]) == N.ERR_INVALID_ARGUMENT
    assert call([4096], [-4]) == N.ERR_INVALID_ARGUMENT
    assert call([0], [4]) == N.ERR_INVALID_ARGUMENT
    for bad in (-1.0, float("nan")):
        assert call([4096], [4], max_norm=bad) == N.ERR_INVALID_ARGUMENT
