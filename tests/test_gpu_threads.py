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


def _distill(vocab):
    import torch
    from oxitorch_b200 import _native as N
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x, teacher = (torch.randn(2, n, device="cuda", generator=g) for n in (vocab, 8))
    ids = torch.arange(16, device="cuda").view(2, 8)
    loss, rows, d = x.new_empty(1), x.new_empty(2 * N.DISTILL_PARTS), torch.empty_like(x)
    args = (x.data_ptr(), vocab, teacher.data_ptr(), ids.data_ptr(), 8, 1.0, None, loss.data_ptr(), rows.data_ptr(),
            d.data_ptr(), 2, vocab, 2, 0, None, torch.cuda.current_stream().cuda_stream)
    entry = N.load().oxc_distill_loss

    def call():
        N.check(entry(*args), "distill_loss")
        return x, teacher, ids, loss, rows[:2], d
    return call


def _add_rms_norm(cols):
    import torch
    from oxitorch_b200 import _native as N
    g = torch.Generator(device="cuda").manual_seed(cols)
    r, dy, dr = (torch.randn(16, cols, device="cuda", generator=g) for _ in range(3))
    w, rstd = torch.randn(cols, device="cuda", generator=g), torch.rand(16, device="cuda", generator=g) + 0.5
    dx, dw = torch.empty_like(r), torch.empty_like(w)
    L = N.load()
    ws = torch.empty(L.oxc_add_rms_norm_bwd_workspace_size(16, cols), dtype=torch.uint8, device="cuda")
    args = (r.data_ptr(), w.data_ptr(), rstd.data_ptr(), dy.data_ptr(), cols, dr.data_ptr(), cols, dx.data_ptr(),
            dx.data_ptr(), dw.data_ptr(), 16, cols, 0, 0, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)

    def call():
        N.check(L.oxc_add_rms_norm_bwd(*args), "add_rms_norm backward")
        return r, w, rstd, dy, dr, dx, dw
    return call


def _layer_norm(cols):
    import torch
    from oxitorch_b200 import _native as N
    g = torch.Generator(device="cuda").manual_seed(cols)
    x, dy = (torch.randn(16, cols, device="cuda", generator=g) for _ in range(2))
    w, b = (torch.randn(cols, device="cuda", generator=g) for _ in range(2))
    mean, rstd = x.mean(1), 1 / x.std(1)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
    L = N.load()
    ws = torch.empty(L.oxc_layer_norm_bwd_workspace_size(16, cols), dtype=torch.uint8, device="cuda")
    args = (x.data_ptr(), w.data_ptr(), b.data_ptr(), mean.data_ptr(), rstd.data_ptr(), dy.data_ptr(), dx.data_ptr(),
            dw.data_ptr(), db.data_ptr(), 16, cols, 0, 0, ws.data_ptr(), ws.numel(),
            torch.cuda.current_stream().cuda_stream)

    def call():
        N.check(L.oxc_layer_norm_bwd(*args), "layer_norm backward")
        return x, w, b, mean, rstd, dy, dx, dw, db
    return call


@pytest.mark.parametrize("make,sizes", [(_policy, (98304, 200000, 320000)), (_distill, (98304, 200000, 280000)),
                                        (_add_rms_norm, (18000, 24576, 32768)), (_add_rms_norm, (8704, 10000, 12288)),
                                        (_layer_norm, (3104, 3200, 4096))],
                         ids=["policy_loss", "distill_loss", "add_rms_norm", "add_rms_norm, narrower", "layer_norm"])
def test_threads_with_different_shared_memory(make, sizes):
    import torch
    found, failed = _at_once([lambda n=n: make(n) for n in 2 * sizes], 4000)
    assert not failed
    for n, got in zip(2 * sizes, found):
        for a, b in zip(got, make(n)()):
            assert torch.equal(a, b)
