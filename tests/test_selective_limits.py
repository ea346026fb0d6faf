"""Limits of the operators of a selective state space model that are checked before
anything touches the device."""


def test_policy_loss_divisors():
    """Any positive divisor passes, also one below the rows of the call (what is refused
    here are the missing operands behind it); zero and negative ones do not."""
    from oxitorch_b200 import _native as N
    L = N.load(require_device=False)

    def call(total, rows=3):
        return L.oxc_policy_loss(None, 0, None, None, 16, None, 0.2, 0.2, 0.0, 1.0, None, 16, None, None, None, rows, 8, total,
                                 0, None, None)
    for total in (1, 2, 3, 2 ** 40):
        assert call(total) == N.ERR_INVALID_ARGUMENT and "null pointer" in N.last_error()
    for rows in (0, 3):
        for total in (0, -1, -2 ** 40):
            assert call(total, rows) == N.ERR_INVALID_ARGUMENT and "total_rows" in N.last_error()


def test_policy_loss_temperatures():
    """Those whose reciprocal, or they themselves, f32 does not hold are refused."""
    from oxitorch_b200 import _native as N
    L = N.load(require_device=False)
    for tau in (0.0, -1.0, 1e-50, 1e-39, 1e39, float("inf"), float("nan")):
        assert L.oxc_policy_loss(None, 0, None, None, 16, None, 0.2, 0.2, 0.0, tau, None, 16, None, None, None, 1, 8, 1, 0,
                                 None, None) == N.ERR_INVALID_ARGUMENT
        assert "temperature" in N.last_error()
