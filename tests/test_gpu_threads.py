"""Calls from several threads at once, each on a stream of its own, on sizes that need
different amounts of one kernel's shared memory."""

import threading

import pytest

pytestmark = pytest.mark.gpu


def _at_once(makes, calls):
    """Runs each of the functions that `makes` return `calls` times in a thread of its own;
    returns their last results and what they raised."""
    import torch
    found, failed = [None] * len(makes), []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                call = makes[i]()
                for _ in range(calls):
                    found[i] = call()
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # shown by the assertion on them
            failed.append(repr(e))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(makes))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return found, failed


def _policy(vocab):
    """The C entry itself: as little as possible between a call's requests to the driver."""
    import torch
    from oxitorch_b200 import _native as N
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn(2, vocab, device="cuda", generator=g)
    tokens, v = torch.tensor([0, vocab - 1], device="cuda"), torch.ones(2, device="cuda")
    old, loss, logp, rows, d = -10 * v, v[:1].clone(), v.clone(), v.clone(), torch.empty_like(x)
    args = (x.data_ptr(), vocab, tokens.data_ptr(), old.data_ptr(), v.data_ptr(), None, 0.2, 0.2, 0.0, 1.0, None,
            loss.data_ptr(), logp.data_ptr(), rows.data_ptr(), d.data_ptr(), 2, vocab, 2, 0, None,
            torch.cuda.current_stream().cuda_stream)
    entry = N.load().oxc_policy_loss

    def call():
        N.check(entry(*args), "policy_loss")
        return x, tokens, old, loss, logp, d  # (x to old: kept alive)
    return call


@pytest.mark.parametrize("make,sizes", [(_policy, (98304, 200000, 320000))], ids=["policy_loss"])
def test_threads_with_different_shared_memory(make, sizes):
    import torch
    found, failed = _at_once([lambda n=n: make(n) for n in 2 * sizes], 4000)
    assert not failed
    for n, got in zip(2 * sizes, found):
        for a, b in zip(got, make(n)()):
            assert torch.equal(a, b)
