"""The operators of a selective state space model where they can go wrong: rates
without bound in a single step, factors below the smallest normal f32, ratios next to
where they are clipped, divisors of the policy loss, derivatives that there are none
of, and rows cut into segments in every layout of the states.  Error bounds come from
tests/selective_reference.py."""

import threading

import numpy as np
import pytest

import selective_reference as R
from test_gpu_draft import DTYPES, _check, _n, _t
from test_gpu_selective import _clip_check, _gradients, _policy_check, _policy_inputs, _scan_check, _scan_inputs

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


# ---- clip_global_norm_ ---------------------------------------------------------------

def test_global_norm_beyond_32_bits():
    """Squares that f32 does not hold, a norm that it holds, and one that it does not."""
    import torch
    from oxitorch_b200 import tensor_ops as T
    grads = _gradients([1000, 77], ["float32"], 1e37)
    norm, _ = R.clip([_n(g) for g in grads], 1.0)
    assert norm < 2.0 ** 128
    got = T.global_norm(grads).item()
    assert abs(got - norm) <= 2.0 ** -23 * norm  # finite, and the 64-bit value
    assert torch.isinf(T.global_norm(grads * 2000))
    assert torch.isfinite(T.global_norm([g.bfloat16() for g in grads]))


@pytest.mark.parametrize("dtypes", [["float32"], ["bfloat16"], ["float32", "bfloat16"]])
@pytest.mark.parametrize("max_norm", [1.0, 1e-3, 1e-6, 1e-20])
def test_clip_global_norm_by_factors_below_the_smallest_normal(max_norm, dtypes):
    """Gradients of 1e36 clipped to norms down to 1e-20: the factor, 6e-39 to 6e-59, is
    one that f32 holds with few bits or not at all; the clipped values are ordinary."""
    import torch
    sizes = [1000, 77, 5, 4096, 20001]
    _clip_check(_gradients(sizes, dtypes, 1e36), max_norm)
    grads = _gradients(sizes, dtypes, 1e36)
    _clip_check(grads, max_norm, out=[torch.full_like(g, float("nan")) for g in grads])
    wide = torch.zeros(20010, device="cuda", dtype=grads[-1].dtype)
    wide[3:20004] = grads[-1]
    _clip_check([wide[3:20004]], max_norm)  # rows off their 16 bytes
    assert not wide[:3].any() and not wide[20004:].any()


def test_clip_global_norm_where_the_norm_is_beyond_32_bits():
    """The norm returned is infinite, the factor is not zero: it comes from the 64-bit norm."""
    import torch
    from oxitorch_b200 import tensor_ops as T
    grads = _gradients([4001] * 500, ["float32"], 1e37)
    norm, want = R.clip([_n(g) for g in grads], 2.0)
    assert norm > 2.0 ** 128
    assert torch.isinf(T.clip_global_norm_(grads, 2.0))
    for g, w in zip(grads, want):
        _check(g, w, 2.0 ** -23 * np.abs(w), "clipped")


def test_global_norm_refuses_what_it_has_no_gradient_for():
    import torch
    from torch.autograd import forward_ad
    from oxitorch_b200 import tensor_ops as T
    a, b = _gradients([12, 20], ["float32"])
    want = T.global_norm([a, b])
    for bad in ([a.clone().requires_grad_(), b], [b, a.clone().requires_grad_() * 2], [torch.nn.Parameter(a.clone())]):
        with pytest.raises(ValueError, match="gradient"):
            T.global_norm(bad)
        with torch.no_grad():
            T.global_norm(bad)
    assert torch.equal(T.global_norm([a, None, torch.nn.Parameter(b, requires_grad=False)]), want)
    for bad in ([a.clone().requires_grad_(), b], [b, a.clone().requires_grad_() * 2]):
        with pytest.raises(ValueError, match="gradient"):  # also beside an output of its own
            T.clip_global_norm_(bad, 1.0, out=[torch.empty_like(g) for g in bad])
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(a, torch.ones_like(a))
        for call in (T.global_norm, lambda g: T.clip_global_norm_(g, 1.0)):
            with pytest.raises(ValueError, match="gradient"):
                call([b, dual])
        assert torch.equal(T.global_norm([a, b]), want)


# ---- policy_loss ---------------------------------------------------------------------

def _edge_rows(vocab, far, tau, clip, seed):
    """Rows of `vocab` logits, the first c of them 0 and the token's `far`, the others
    -inf, whose sum of exponentials is c in f32 (exp(far / tau) is below 2^-40) and off by
    less than 1e-12 in truth; old log-probabilities with which the ratio lies within 1e-6 of
    where it is clipped, but no nearer than 2e-8, on either side."""
    g = np.random.default_rng(seed)
    rows = []
    for c in g.permutation(np.arange(500, vocab)):
        at = c - 1 if far == 0 else c
        if at >= vocab:
            continue
        logp = far / tau - np.log(float(c))
        for edge in (1 - clip[0], 1 + clip[1]):
            old = np.float32(logp - np.log(edge))
            for old in (old, np.nextafter(old, np.float32(0)), np.nextafter(old, np.float32(-1e9))):
                off = np.exp(logp - np.float64(old)) / edge - 1
                if 2e-8 < abs(off) < 1e-6:
                    rows.append((c, at, old, logp, edge, off))
        if len(rows) > 600:
            break
    return rows


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [2000, 20011])
@pytest.mark.parametrize("far,tau,clip", [(0.0, 1.0, (0.2, 0.28)), (-30.0, 1.0, (0.2, 0.2)), (-30.0, 0.7, (0.2, 0.28)),
                                          (-30.0, 0.9, (0.3, 0.1))])
def test_policy_loss_ratios_next_to_where_they_are_clipped(far, tau, clip, vocab, dtype):
    """Whether a row is clipped decides whether it has a gradient.  A log-probability of
    -7 to -50 in f32 is off by 5e-7 to 4e-6, more than these ratios lie from the edge: the
    side has to be the one that 64 bits say.  Rows of -inf beside 0 have an exact sum."""
    import torch
    from oxitorch_b200 import functional as F
    rows = _edge_rows(vocab, far, tau, clip, vocab)
    assert len(rows) > 300
    c, at, old, logp, edge, off = (np.array(v) for v in zip(*rows))
    assert (off > 0).any() and (off < 0).any() and len(set(edge)) == 2
    n = len(rows)
    x = torch.arange(vocab, device="cuda") < torch.from_numpy(c).cuda()[:, None]
    x = torch.where(x, 0.0, -float("inf"))
    x[torch.arange(n), torch.from_numpy(at).cuda()] = far
    x = x.to(getattr(torch, dtype))
    old_t = torch.from_numpy(old.astype(np.float32)).cuda()
    tokens = torch.from_numpy(at).cuda()
    for sign in (1.0, -1.0):
        adv = torch.full((n,), sign, device="cuda")
        _, got, d = F.policy_loss_fwd(x, tokens, old_t, adv, clip=clip, temperature=tau, total_rows=n)
        # with z = (logit - max) / tau: the difference, 1 / tau and their product are off by
        # 2^-24 |z| each, logf by 2^-23 of log c, the sum by 2^-24 |logp|; |logp| = |z| + log c
        _check(got, logp, 2.0 ** -22 * np.abs(logp) + 1e-10, "logp")
        r = np.exp(logp - old.astype(np.float64))
        clipped = r > 1 + clip[1] if sign > 0 else r < 1 - clip[0]
        have = d.float().abs().sum(1).cpu().numpy() > 0
        assert np.array_equal(have, ~clipped), f"{(have == clipped).sum()} of {n} rows on the wrong side"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,vocab", [(64, 1003), (7, 32001), (5, 330001)])
def test_policy_loss_mean_over_the_tokens_that_count(n, vocab, dtype):
    """total_rows as the number of rows that are no padding: below the rows of the call."""
    if vocab == 330001 and dtype == "bfloat16":
        vocab = 660001  # beyond what a cluster holds
    logits, tokens, old, ref, adv = _policy_inputs(n, vocab, dtype)
    tokens[::3] = -1
    count = int((tokens >= 0).sum())
    assert 0 < count < n
    _policy_check(logits, tokens, old, adv, ref, kl=0.1, total=count)
    _policy_check(logits, tokens, old, adv, total=count)
    _policy_check(logits, tokens, old, adv, ref, kl=0.1, tau=0.7, total=count + 1)


def test_policy_loss_mean_over_the_tokens_that_count_twice_backward_and_captured():
    """The gradient computed again has the same divisor; a captured call takes it as given."""
    import torch
    from oxitorch_b200 import functional as F
    logits, tokens, old, ref, adv = _policy_inputs(40, 1003, "float32")
    tokens[::4] = -1
    count = int((tokens >= 0).sum())
    dev = lambda a: torch.from_numpy(np.asarray(a)).cuda()  # noqa: E731
    x, rest = logits.requires_grad_(), [dev(v) for v in (tokens, old, adv, ref)]
    loss, _ = F.policy_loss(x, *rest, kl_coef=0.1, total_rows=count)
    a, = torch.autograd.grad(loss, x, retain_graph=True)
    b, = torch.autograd.grad(loss, x)
    assert torch.equal(a, b)
    x = x.detach()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        F.policy_loss_fwd(x, *rest, kl_coef=0.1, total_rows=count)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got, _, d = F.policy_loss_fwd(x, *rest, kl_coef=0.1, total_rows=count)
    torch.cuda.current_stream().wait_stream(side)
    graph.replay()
    assert torch.equal(got.reshape(()), loss.detach()) and torch.equal(d, a)


def test_policy_loss_divisors():
    """No rows with the default divisor, a batch of padding alone, and the divisors that
    are refused: 0, negative ones, and fewer than the tokens that count."""
    import torch
    from oxitorch_b200 import functional as F
    x = torch.zeros(0, 5, device="cuda", requires_grad=True)
    none, no = torch.zeros(0, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda")
    loss, logp = F.policy_loss(x, no, none, none)
    assert loss == 0 and logp.shape == (0,)
    assert torch.autograd.grad(loss, x)[0].shape == (0, 5)
    assert F.policy_loss(x.detach(), no, none, none)[0] == 0
    x, v = torch.randn(4, 5, device="cuda"), torch.ones(4, device="cuda")
    pad = torch.full((4,), -1, device="cuda")
    loss, _, d = F.policy_loss_fwd(x, pad, v, v, total_rows=1)
    assert loss == 0 and not d.any()
    tokens = torch.tensor([1, -1, 3, 0], device="cuda")
    F.policy_loss(x, tokens, -v, v, total_rows=3)
    for args in ((x, tokens), (x[:0], tokens[:0])):
        n = len(args[0])
        for bad in (0, -1, -3):
            with pytest.raises(ValueError):
                F.policy_loss(*args, v[:n], v[:n], total_rows=bad)
    for total in (2, 1):
        with pytest.raises(ValueError, match="total_rows"):
            F.policy_loss(x, tokens, v, v, total_rows=total)
        with pytest.raises(ValueError, match="total_rows"):
            F.policy_loss(x.clone().requires_grad_(), tokens, v, v, total_rows=total)


@pytest.mark.parametrize("name", ["old_logp", "advantages", "ref_logp"])
def test_policy_loss_refuses_what_it_has_no_gradient_for(name):
    """Also where the logits need none: the loss would leave the graph without a word."""
    import torch
    from torch.autograd import forward_ad
    from oxitorch_b200 import functional as F
    x, tokens = torch.randn(3, 5, device="cuda"), torch.tensor([0, 4, -1], device="cuda")
    v = torch.ones(3, device="cuda")
    args = dict(old_logp=-v, advantages=v, ref_logp=-v, kl_coef=0.1)
    for logits in (x, x.clone().requires_grad_()):
        with pytest.raises(ValueError, match=name):
            F.policy_loss(logits, tokens, **{**args, name: args[name].clone().requires_grad_()})
        with torch.no_grad():
            F.policy_loss(logits, tokens, **{**args, name: args[name].clone().requires_grad_()})
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(args[name], torch.ones_like(v))
            with pytest.raises(ValueError, match=name):
                F.policy_loss(logits, tokens, **{**args, name: dual})
            F.policy_loss(logits, tokens, **args)


def test_token_logprobs_over_no_classes():
    """Refused where there are rows, as policy_loss refuses it; no rows are no matter."""
    import torch
    from oxitorch_b200 import functional as F
    for lead in ((3,), (2, 3), (1,)):
        tokens = torch.zeros(lead, dtype=torch.int64, device="cuda")
        with pytest.raises(ValueError, match="zero classes"):
            F.token_logprobs(torch.zeros(*lead, 0, device="cuda"), tokens)
        with pytest.raises(ValueError, match="zero classes"):
            F.policy_loss(torch.zeros(*lead, 0, device="cuda"), tokens, tokens.float(), tokens.float())
    for vocab in (0, 5):
        none = torch.zeros(0, dtype=torch.int64, device="cuda")
        assert F.token_logprobs(torch.zeros(0, vocab, device="cuda"), none).shape == (0,)
        assert F.policy_loss(torch.zeros(0, vocab, device="cuda"), none, none.float(), none.float())[0] == 0


# ---- selective_scan ------------------------------------------------------------------

# the channels of a CTA of the VJP
_BACKWARD_CHANNELS = ((8, 128), (16, 128), (32, 64), (64, 32), (128, 16))


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("T,D,N", [(300, 20, 7), (260, 21, 8), (300, 20, 10), (230, 19, 12), (290, 140, 16), (300, 20, 24),
                                   (211, 17, 23), (300, 36, 31), (260, 20, 40), (300, 19, 48), (260, 20, 64), (200, 33, 57),
                                   (260, 12, 90), (200, 15, 96), (260, 20, 128), (300, 13, 101)])
def test_selective_scan_of_segments_in_every_layout(T, D, N, gated, dtype, packed):
    """One row, cut into segments in both directions, for every number of states a lane
    and of lanes a channel, at widths that vectors fit and that they do not."""
    from oxitorch_b200 import _native
    size = _native.load().oxc_selective_scan_workspace_size
    channels = next(c for n, c in _BACKWARD_CHANNELS if N <= n)
    one = 4 * (D * (N + 2) + -(-D // channels) * T * 2 * N)
    assert size(1, T, D, N, 0) > 0 and size(1, T, D, N, 1) > one
    _scan_check(*_scan_inputs(1, T, D, N, dtype, packed, gated=gated))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,D,N", [(1, 40, 300, 64), (2, 33, 150, 128), (1, 35, 515, 40), (2, 20, 260, 96)])
def test_selective_scan_many_states_over_many_channels(B, T, D, N, dtype):
    """dB and dC summed over several tiles of channels where a CTA holds few of them.

    With rates of -128 some decays lie below 2^-126, where the exponential gives 0: what is
    lost of a gradient is below 2^-126 times one of a token (below 2^9: two normal variates,
    a gate and another), the states (2^6), rates (2^8) and tokens (2^6) that it is summed
    over; with 2^-126 for the states themselves, 2^-90 covers all."""
    import torch
    from oxitorch_b200 import functional as F
    args, starts, dy, dlast = _scan_inputs(B, T, D, N, dtype, True)
    leaves = [t.requires_grad_() for t in args.values()]
    y, last = F.selective_scan(**args, starts=torch.from_numpy(starts).cuda())
    ref = R.Scan(**{k: _n(t) for k, t in args.items()}, starts=starts)
    want, bound = ref.out()
    _check(y, want, bound + 2.0 ** -90, "y")
    _check(last, ref.last, ref.last_bound + 2.0 ** -90, "last")
    got = torch.autograd.grad((y, last), leaves, (dy, dlast))
    want, bound = ref.grad(_n(dy), _n(dlast))
    for k, d in zip(args, got):
        _check(d, want[k], bound[k] + 2.0 ** -90, "d" + k)


def test_selective_scan_backward_in_two_threads():
    """Two threads that call the VJP at once, each on a stream of its own."""
    import torch
    from oxitorch_b200 import functional as F
    args, _, dy, dlast = _scan_inputs(1, 200, 24, 16, "float32", False)
    carry = F.selective_scan_fwd(**args)[2]
    del args["h0"]
    want = F.selective_scan_bwd(**args, carry=carry, dy=dy, dlast=dlast)
    torch.cuda.synchronize()
    found, failed = {}, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    found[i] = F.selective_scan_bwd(**args, carry=carry, dy=dy, dlast=dlast)
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # shown by the assertion below
            failed.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for got in found.values():
        for a, b in zip(got, want):
            assert torch.equal(a, b)
