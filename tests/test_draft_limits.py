"""Sizes that the recurrent draft model's operators refuse because an index of their
kernels would pass 31 bits; no device is needed."""

import pytest


@pytest.fixture(scope="module")
def lib():
    from oxitorch_b200 import _native as N
    return N.load(require_device=False)


@pytest.mark.parametrize("vocab", [2 ** 31 - 1, 2 ** 31 - 500, 2 ** 31])
def test_distill_loss_vocabulary(lib, vocab):
    """A thread's index steps by the CTA's size past the last token."""
    from oxitorch_b200 import _native as N
    for dtype in (N.F32, N.BF16):
        assert lib.oxc_distill_loss(None, 0, None, None, 1, 1.0, None, 16, None, None, 1, vocab, 1, dtype, None,
                                    None) == N.ERR_NOT_IMPLEMENTED


@pytest.mark.parametrize("dim", [2 ** 31 - 1, 2 ** 31 - 100, 2 ** 31, 2 ** 33])
def test_gated_scan_channels(lib, dim):
    """A tile's channels are counted from its first one, past the last channel."""
    from oxitorch_b200 import _native as N
    zeros = [0] * 2
    for length in (1, 100):
        assert lib.oxc_gated_scan_fwd(None, *zeros, None, *zeros, None, None, None, None, None, 1, length, dim, 0,
                                      None, 0, None) == N.ERR_NOT_IMPLEMENTED
        assert lib.oxc_gated_scan_bwd(None, *zeros, None, *zeros, None, None, None, *zeros, None, None, None, None,
                                      1, length, dim, 0, None, 0, None) == N.ERR_NOT_IMPLEMENTED
