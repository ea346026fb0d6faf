"""The operators of a selective state space model where they can go wrong: rates
without bound in a single step.  Error bounds come from tests/selective_reference.py."""

import numpy as np
import pytest

import selective_reference as R
from test_gpu_draft import DTYPES, _check, _n, _t
from test_gpu_selective import _scan_inputs

pytestmark = pytest.mark.gpu


# ---- selective_step ------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rate", [-float("inf"), -3e38])
@pytest.mark.parametrize("N", [4, 7, 16, 33])
def test_selective_step_keeps_its_state_beside_unbounded_rates(N, rate, dtype):
    """A rate that forgets at once (one is beyond f32 only after the product with
    log2(e)) times a step of 0, as of a padded token, leaves the state as it is: token by
    token and in the scan.  In 64 bits a rate of -1e30 does the same."""
    import torch
    from oxitorch_b200 import functional as F
    B, T, D = 2, 6, 10
    args, _, _, _ = _scan_inputs(B, T, D, N, dtype, False)
    args["delta"][:, 1::2] = -200.0
    args["delta"][1, 2] = -200.0
    args["A"][:, N // 2], args["A"][3] = rate, rate
    ref = R.Scan(**{k: _n(t) for k, t in args.items() if k != "A"}, A=np.maximum(_n(args["A"]), -1e30))
    want, bound = ref.out()
    y, last = F.selective_scan(**args)
    _check(y, want, bound, "scan")
    _check(last, ref.last, ref.last_bound, "last")
    state = args["h0"].clone()
    for t in range(T):
        at = {k: args[k][:, t] for k in ("x", "delta", "B", "C", "z")}
        y = F.selective_step(**at, A=args["A"], D=args["D"], delta_bias=args["delta_bias"], state=state)
        _check(y, want[:, t], bound[:, t], f"y {t}")
        _check(state, ref.h[:, t], ref.e[:, t], f"state {t}")
