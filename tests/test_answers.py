"""Log-probabilities of drawn tokens, the clipped policy loss and the preference loss against float64.

What the kernels round.  Of a row: the exponentials, 2^-23 for the instruction and 2^-22 |z - max| / tau for the three roundings of their
argument, and a sum of V / 512 additions and some forty more, 2^-24 each: a relative error
  rel = 2^-22 (1 + spread) + 2^-24 (V / 512 + 40), spread = largest |z - max| / tau
of the sum and of a probability.  A log-probability is off by rel, by two ulps of the logarithm and by the roundings of its two terms
and their difference: d_lp = rel + 2^-22 (|z_x - max| / tau + log sum + 1).  A ratio and e^d by that, relative, and by two ulps.  A gradient:
half a step of f16, 2^-11 |g| (2^-25 below its normal range), the coefficient's error and, of the probability, rel twice."""
import numpy as np
import pytest

from cacti_amd import ffi

GPU = pytest.mark.gpu
LOGP = dict(N=2, V=64, logit=64, ld=64, tok=64, mask=None, temp=1.0, logp=64, stats=64, status=None, stream=None)
ADJ = dict(N=2, V=64, logit=0x1000, ld=64, tok=64, stats=64, dlogp=64, temp=1.0, d=0x8000, ldd=64, acc=0, stream=None)
POLICY = dict(N=2, V=64, logit=0x1000, ld=64, tok=64, mask=None, old=64, adv=64, ref=None, scale=64, lo=0.2, hi=0.2, beta=0.1, temp=1.0, loss=64,
              logp=64, d=0x8000, ldd=64, acc=0, status=None, stream=None)
PAIRS = dict(N=8, pairs=2, logp=64, ref=None, mask=None, starts=64, scale=64, beta=0.1, smoothing=0.0, mean=0, loss=64, reward=64, dlogp=64,
             status=None, stream=None)
ROWS = [(dict(N=0), "empty"), (dict(V=0), "empty"), (dict(V=65537, ld=65537, ldd=65537), "65536"), (dict(N=1 << 23), "2^23"), (dict(ld=63), "pitch"),
        (dict(logit=None), "null"), (dict(tok=None), "null"), (dict(temp=0.0), "temperature"), (dict(temp=float("nan")), "temperature"),
        (dict(logit=65), "misaligned"), (dict(tok=65), "misaligned")]
GRAD = [(dict(d=None), "null"), (dict(ldd=63), "pitch"), (dict(d=0x8001), "misaligned"), (dict(d=0x1002), "place"), (dict(d=0x1000, ldd=65), "place")]
REFUSED = [("cacti_hip_token_logp_fwd", LOGP, c) for c in ROWS + [(dict(logp=None), "null"), (dict(stats=66), "misaligned"), (dict(status=66), "misaligned")]] + \
          [("cacti_hip_token_logp_bwd", ADJ, c) for c in ROWS + GRAD + [(dict(stats=None), "null"), (dict(dlogp=66), "misaligned")]] + \
          [("cacti_hip_policy_loss", POLICY, c) for c in ROWS + GRAD + [
              (dict(old=None), "null"), (dict(adv=None), "null"), (dict(scale=None), "null"), (dict(loss=None), "null"), (dict(logp=None), "null"),
              (dict(ref=66), "misaligned"), (dict(lo=-0.1), "clip"), (dict(lo=1.1), "clip"), (dict(hi=float("nan")), "clip"), (dict(beta=-1.0), "beta"),
              (dict(beta=float("inf")), "beta")]] + \
          [("cacti_hip_preference_loss", PAIRS, c) for c in [
              (dict(N=0), "empty"), (dict(pairs=0), "empty"), (dict(N=1 << 23), "2^23"), (dict(logp=None), "null"), (dict(starts=None), "null"),
              (dict(scale=None), "null"), (dict(reward=None), "null"), (dict(dlogp=66), "misaligned"), (dict(beta=-0.1), "beta"),
              (dict(smoothing=1.5), "smoothing"), (dict(smoothing=float("nan")), "smoothing")]]


@pytest.mark.parametrize("entry,args,change", REFUSED)
def test_refuses(entry, args, change):
    change, why = change
    L = ffi.lib()
    assert getattr(L, entry)(*dict(args, **{k: v for k, v in change.items() if k in args}).values()) < 0
    assert why in L.cacti_hip_last_error().decode()


def dev(x):
    import torch
    x = np.ascontiguousarray(x)
    return torch.from_numpy(x.astype(np.uint16).view(np.int16) if x.dtype == np.int64 else x).cuda()


def make(seed, N, V, std=3.0):
    r = np.random.default_rng(seed)
    z = (r.standard_normal((N, V)) * std).astype(np.float16)
    tok = r.integers(0, V, N)
    tok[: N // 2] = np.argsort(-z[: N // 2], 1)[np.arange(N // 2), r.integers(0, min(V, 8), N // 2)]        # some of them likely
    return r, z, tok


def rows64(z, tok, temp):
    """log-probabilities [N, V] and those of the tokens; rel and d_lp as above."""
    x = z.astype(np.float64) / temp
    mx = x.max(1, keepdims=True)
    s = np.exp(x - mx).sum(1, keepdims=True)
    logs = x - mx - np.log(s)
    at = np.arange(len(tok)), tok
    spread = (mx - np.where(np.isfinite(x), x, mx).min(1, keepdims=True))[:, 0]
    rel = 2.0 ** -22 * (1 + spread) + 2.0 ** -24 * (z.shape[1] / 512 + 40)
    d_lp = rel + 2.0 ** -22 * (np.abs((x - mx)[at]) + np.log(s)[:, 0] + 1)
    return logs, logs[at], rel, d_lp


def gradient64(logs, tok, c, d_c, rel):
    """c (one-hot - p) and its error for a coefficient that is off by d_c."""
    hot = np.zeros_like(logs)
    hot[np.arange(len(tok)), tok] = 1
    p = np.exp(logs)
    g = c[:, None] * (hot - p)
    # (where the one-hot's 1 meets a p near it the difference is off by that of p and by one rounding)
    tol = d_c[:, None] * (hot + p) + np.abs(c)[:, None] * (p * (2 * rel + 2.0 ** -22)[:, None] + 2.0 ** -23 * hot) + 2.0 ** -11 * np.abs(g) + 2.0 ** -25
    return g, tol


def near(got, want, tol, what):
    got = np.asarray(got.cpu() if hasattr(got, "cpu") else got).astype(np.float64)
    assert np.isfinite(got).all(), what
    off = np.abs(got - want) - tol
    assert (off <= 0).all(), "%s: %.3g beyond its bound" % (what, off.max())


SHAPES = [(1, 1, 1.0), (2, 2, 1.0), (5, 7, 0.7), (3, 8, 2.0), (4, 1021, 1.0), (3, 8191, 1.3), (2, 8200, 1.0), (3, 16385, 0.6), (2, 32000, 1.0), (2, 65536, 1.0)]


@GPU
@pytest.mark.parametrize("N,V,temp", SHAPES)
def test_logp_and_adjoint(N, V, temp):
    from cacti_amd import ops
    print("token_logp", N, V, temp, flush=True)
    for std in (3.0, 0.1):
        r, z, tok = make(V + N, N, V, std)
        d = r.standard_normal(N).astype(np.float32)
        logp, stats = ops.token_logp_fwd(dev(z), dev(tok), temp)
        grad = ops.token_logp_bwd(dev(z), dev(tok), stats, dev(d), temp)
        logs, lp, rel, d_lp = rows64(z, tok, temp)
        near(logp, lp, d_lp, "logp")
        c = d.astype(np.float64) / temp
        near(grad, *gradient64(logs, tok, c, np.abs(c) * 2.0 ** -22, rel), "gradient")


def policy64(z, tok, old, adv, ref, scale, lo, hi, beta, temp):
    logs, lp, rel, d_lp = rows64(z, tok, temp)
    old, adv, scale = (x.astype(np.float64) for x in (old, adv, scale))
    ratio = np.exp(lp - old)
    d_r = ratio * (d_lp + 2.0 ** -22 * (1 + np.abs(lp - old)))
    assert (np.abs(ratio - (1 - lo)) > d_r).all() and (np.abs(ratio - (1 + hi)) > d_r).all()      # no draw on a border
    free, bound = ratio * adv, np.clip(ratio, 1 - lo, 1 + hi) * adv
    loss, slope = -np.minimum(free, bound), np.where(free <= bound, -free, 0)
    d_loss, d_slope = np.abs(adv) * (d_r + 2.0 ** -22 * np.maximum(ratio, 1 + hi)), np.abs(adv) * (d_r + 2.0 ** -22 * ratio)
    if ref is not None:
        d = ref.astype(np.float64) - lp
        e = np.expm1(d)
        loss, slope = loss + beta * (e - d), slope - beta * e
        d_loss = d_loss + beta * (np.abs(e) * d_lp + 2.0 ** -21 * (np.abs(e) + np.abs(d)))
        d_slope = d_slope + beta * (np.exp(d) * d_lp + 2.0 ** -21 * np.abs(e))
    c = slope * scale / temp
    d_c = np.abs(scale) / temp * (d_slope + 2.0 ** -22 * np.abs(slope))
    return loss, d_loss + 2.0 ** -22 * np.abs(loss), lp, d_lp, *gradient64(logs, tok, c, d_c, rel)


def policy_inputs(r, z, tok, temp):
    N = len(tok)
    lp = rows64(z, tok, temp)[1]
    near_by = lambda x: (lp + x * r.standard_normal(N)).astype(np.float32)
    return near_by(0.3), r.standard_normal(N).astype(np.float32), near_by(0.5), (r.standard_normal(N) * 4).astype(np.float32)


@GPU
@pytest.mark.parametrize("N,V,temp", SHAPES)
@pytest.mark.parametrize("with_ref", [True, False])
def test_policy(N, V, temp, with_ref):
    from cacti_amd import ops
    print("policy_loss", N, V, temp, flush=True)
    r, z, tok = make(3 * V + N, N, V)
    old, adv, ref, scale = policy_inputs(r, z, tok, temp)
    ref = ref if with_ref else None
    loss, logp, grad = ops.policy_loss(dev(z), dev(tok), dev(old), dev(adv), dev(scale), ref=None if ref is None else dev(ref), clip=(0.2, 0.3),
                                       beta=0.05, temperature=temp)
    wl, tl, wp, tp, wg, tg = policy64(z, tok, old, adv, ref, scale, 0.2, 0.3, 0.05, temp)
    near(loss, wl, tl, "loss")
    near(logp, wp, tp, "logp")
    near(grad, wg, tg, "gradient")


@GPU
@pytest.mark.parametrize("V", [65, 2048, 2055, 2056, 8199, 8200, 10247, 10248, 16391, 16392, 32775, 32776])
def test_widths_on_either_side_of_what_threads_hold(V):
    test_logp_and_adjoint(9, V, 0.9)
    test_policy(9, V, 1.0, True)


@GPU
def test_gradients_against_differences():
    """Central differences of the float64 loss at the kernels' own gradients."""
    from cacti_amd import ops
    r, z, tok = make(5, 4, 40)
    old, adv, ref, scale = policy_inputs(r, z, tok, 1.4)
    ones = np.ones(4, np.float32)
    grad = ops.policy_loss(dev(z), dev(tok), dev(old), dev(adv), dev(ones), ref=dev(ref), beta=0.3, temperature=1.4)[2].cpu().numpy().astype(np.float64)
    f = lambda x: policy64(x, tok, old, adv, ref, ones, 0.2, 0.2, 0.3, 1.4)[0]
    h, z64 = 1e-4, z.astype(np.float64)
    for d in [np.eye(40)[j][None] * np.ones((4, 1)) for j in (0, int(tok[0]), int(tok[1]), 39)] + [r.standard_normal((4, 40))]:
        num, got = (f(z64 + h * d) - f(z64 - h * d)) / (2 * h), (grad * d).sum(1)
        # differences: h^2 times a third derivative below 40 sum |d|^3 (a ratio and e^d below 8); the gradient: half a step of f16 and fp32's share
        tol = 40 * h * h * (np.abs(d) ** 3).sum(1) + (np.abs(d) * (np.abs(grad) * 2.0 ** -11 + 2.0 ** -16)).sum(1) + 1e-8
        assert (np.abs(num - got) <= tol).all(), (num, got)


@GPU
def test_rows_that_the_mask_left_out_have_no_gradient_whatever_theirs_is():
    import torch
    from cacti_amd import ops
    for V in (40, 2056, 20001):
        r, z, tok = make(V, 6, V)
        mask = np.array([True, False, True, False, False, True])
        z[1], z[3], d = np.nan, 60000, np.ones(6, np.float32)
        logp, stats = ops.token_logp_fwd(dev(z), dev(tok), mask=dev(mask))
        grad = ops.token_logp_bwd(dev(z), dev(tok), stats, dev(d))
        want = ops.token_logp_bwd(dev(z), dev(tok), stats, dev(d * mask))
        assert torch.equal(grad, want) and not bool(grad[dev(~mask)].any()) and not bool(logp[dev(~mask)].any())
        into = torch.full_like(grad, 3.0)
        ops.token_logp_bwd(dev(z), dev(tok), stats, dev(d), acc=into)
        assert bool((into[dev(~mask)] == 3).all()) and torch.isfinite(into).all()


@GPU
def test_rows_that_are_left_out_are_not_read():
    """Masked rows, tokens beyond the vocabulary, coefficients of 0: nothing of them, whatever their logits are; added to: left as it is."""
    import torch
    from cacti_amd import ops
    for V in (200, 203):
        r, z, tok = make(6, 6, V)
        old, adv, ref, scale = policy_inputs(r, z, tok, 1.0)
        clean = [x.cpu().numpy() for x in ops.policy_loss(dev(z), dev(tok), dev(old), dev(adv), dev(scale), ref=dev(ref), beta=0.1)]
        mask = np.array([True, False, True, True, False, True])
        z[1], z[4, 3], z[2] = np.nan, np.inf, np.nan
        tok[2] = V
        scale[3] = 0
        skipped = [1, 2, 4]
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = ops.policy_loss(dev(z), dev(tok), dev(old), dev(adv), dev(scale), ref=dev(ref), mask=dev(mask), beta=0.1, status=status)
        assert int(status) == 3
        for got, was in zip(out, clean):
            got = got.cpu().numpy()
            assert not got[skipped].any() and np.array_equal(got[[0, 5]], was[[0, 5]])
        assert not out[2][3].cpu().numpy().any()
        status.zero_()
        logp, stats = ops.token_logp_fwd(dev(z), dev(tok), mask=dev(mask), status=status)
        assert int(status) == 3 and not logp.cpu().numpy()[skipped].any() and np.array_equal(logp.cpu().numpy()[[0, 3, 5]], clean[1][[0, 3, 5]])
        d = np.array([1, 0, 1, -2, 0, 0.5], np.float32)
        grad = ops.token_logp_bwd(dev(z), dev(tok), stats, dev(d))
        assert not grad[skipped].cpu().numpy().any() and bool(grad[0].any())
        into = torch.full((6, V), 3.0, dtype=torch.float16, device="cuda")
        assert ops.token_logp_bwd(dev(z), dev(tok), stats, dev(d), acc=into) is into
        want = np.where(d[:, None] == 0, 0, grad.cpu().numpy()).astype(np.float32) + 3
        assert np.array_equal(into.cpu().numpy(), want.astype(np.float16))


@GPU
def test_logits_that_are_no_numbers_stay_visible():
    import torch
    from cacti_amd import ops
    r, z, tok = make(7, 5, 100)
    old, adv, ref, scale = policy_inputs(r, z, tok, 1.0)
    adv = np.abs(adv) + 0.1
    clean = [x.cpu().numpy() for x in ops.policy_loss(dev(z), dev(tok), dev(old), dev(adv), dev(scale))]
    z[0, 3], z[2], old[3] = np.nan, -np.inf, np.nan
    z[1, tok[1]] = -np.inf
    loss, logp, grad = (x.cpu().numpy() for x in ops.policy_loss(dev(z), dev(tok), dev(old), dev(adv), dev(scale)))
    for n in (0, 2):
        assert np.isnan(loss[n]) and np.isnan(logp[n]) and np.isnan(grad[n]).all()
    assert np.isnan(loss[3]) and np.isnan(grad[3]).all() and np.isfinite(logp[3])
    # a token that the model rules out: ratio 0, no loss, no gradient
    assert np.isneginf(logp[1]) and loss[1] == 0 and not grad[1].any()
    assert loss[4] == clean[0][4] and np.array_equal(grad[4], clean[2][4])
    # other tokens may be ruled out
    z[4, np.arange(100) != tok[4]] = -np.inf
    loss, logp, grad = (x.cpu().numpy() for x in ops.policy_loss(dev(z[4:]), dev(tok[4:]), dev(old[4:]), dev(adv[4:]), dev(scale[4:])))
    assert logp[0] == 0 and not grad.any()


@GPU
def test_the_ratio_of_a_policy_that_has_not_moved_is_one():
    from cacti_amd import ops
    for V in (1000, 1003, 32000):
        r, z, tok = make(8, 9, V)
        adv = r.standard_normal(9).astype(np.float32)
        old, _ = ops.token_logp_fwd(dev(z), dev(tok))
        loss, logp, _ = ops.policy_loss(dev(z), dev(tok), old, dev(adv), dev(adv))
        assert np.array_equal(loss.cpu().numpy(), -adv) and np.array_equal(logp.cpu().numpy(), old.cpu().numpy())


@GPU
def test_rows_may_be_strided_and_lie_anywhere_also_in_the_logits_place():
    import torch
    from cacti_amd import ops
    for V in (1000, 1003, 9001):
        r, z, tok = make(10, 5, V)
        old, adv, ref, scale = policy_inputs(r, z, tok, 1.0)
        args = [dev(x) for x in (tok, old, adv, scale)]
        wl, tl, wp, tp, wg, tg = policy64(z, tok, old, adv, ref, scale, 0.2, 0.2, 0.1, 1.0)
        for ld, off, ldo, offo in ((V, 0, V + 5, 3), (V + 3, 1, V, 0), (V + 8, 8, V + 8, 0), (2 * V, 5, V + 1, 2)):
            big = torch.zeros(5 * ld + 16, dtype=torch.float16, device="cuda")
            rows = big[off:off + 5 * ld].view(5, ld)[:, :V]
            into = torch.full((5 * ldo + 16,), 7.0, dtype=torch.float16, device="cuda")
            out = into[offo:offo + 5 * ldo].view(5, ldo)[:, :V]
            for place in (out, rows):
                rows.copy_(dev(z))
                out.zero_()
                before = place.cpu().numpy().astype(np.float32)
                loss, logp, grad = ops.policy_loss(rows, *args, ref=dev(ref), beta=0.1, acc=place)
                assert grad is place
                near(loss, wl, tl, "loss")
                # added to what was there: one more rounding of the sum
                near(place, before + wg, tg + 2.0 ** -11 * np.abs(before + wg), "gradient")
                kept = into.clone()
                kept[offo:offo + 5 * ldo].view(5, ldo)[:, :V] = 7
                assert bool((kept == 7).all())
            rows.copy_(dev(z))
            _, stats = ops.token_logp_fwd(rows, args[0])
            want = ops.token_logp_bwd(rows, args[0], stats, args[3])
            assert ffi.lib().cacti_hip_token_logp_bwd(5, V, rows.data_ptr(), ld, args[0].data_ptr(), stats.data_ptr(), args[3].data_ptr(), 1.0,
                                                      rows.data_ptr(), ld, 0, torch.cuda.current_stream().cuda_stream) == 0
            # (pieces of the gradient that begin elsewhere than the row's hold the same elements)
            assert torch.equal(rows, want)


# ---------------------------------------------------------------- pairs
def pairs64(logp, ref, starts, scale, beta, eps, mask, mean):
    P = len(scale)
    lp = logp.astype(np.float64) - (0 if ref is None else ref.astype(np.float64))
    m = np.ones(len(lp), bool) if mask is None else mask
    reward, each = np.zeros(2 * P), np.zeros(2 * P)
    for t in range(2 * P):
        at = slice(starts[t], starts[t + 1])
        each[t] = beta / (max(1, m[at].sum()) if mean else 1)
        reward[t] = each[t] * lp[at][m[at]].sum()
    h = reward[0::2] - reward[1::2]
    ls = lambda x: -np.logaddexp(0, -x)
    loss = -(1 - eps) * ls(h) - eps * ls(-h)
    slope = scale.astype(np.float64) * (eps * np.exp(ls(h)) - (1 - eps) * np.exp(ls(-h)))
    d = np.zeros(len(lp))
    for t in range(2 * P):
        at = slice(starts[t], starts[t + 1])
        d[at] = np.where(m[at], (1, -1)[t % 2] * slope[t // 2] * each[t], 0)
    return loss, reward, d


@GPU
@pytest.mark.parametrize("lens", [[1, 1], [3, 0, 0, 5], [0, 0], [300, 1, 17, 900, 256, 257], [2000, 1999], [1] * 200])
@pytest.mark.parametrize("eps,mean,with_ref,masked", [(0.0, False, True, True), (0.1, True, True, True), (0.3, False, False, False), (1.0, True, False, True)])
def test_preference(lens, eps, mean, with_ref, masked):
    from cacti_amd import ops
    r = np.random.default_rng(sum(lens))
    starts = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    N, P = int(starts[-1]) + 3, len(lens) // 2
    logp, ref = (-np.abs(r.standard_normal(N)) * 3).astype(np.float32), (-np.abs(r.standard_normal(N)) * 3).astype(np.float32)
    ref = ref if with_ref else None
    mask = r.random(N) < 0.6 if masked else None
    scale = r.standard_normal(P).astype(np.float32)
    out = ops.preference_loss(dev(logp), None if ref is None else dev(ref), dev(starts), dev(scale), 0.13, eps, None if mask is None else dev(mask), mean)
    for got, want in zip(out, pairs64(logp, ref, starts, scale, 0.13, eps, mask, mean)):
        # fp64 to the last rounding
        near(got, want, 2.0 ** -24 * np.abs(want) + 1e-12, "of a pair")


@GPU
def test_pairs_far_apart_and_pairs_that_there_are_not():
    import torch
    from cacti_amd import ops
    starts = np.array([0, 2, 4, 6, 8], np.int32)
    logp = np.array([-900, -900, 0, 0, 0, 0, -np.inf, -1], np.float32)
    scale = np.ones(2, np.float32)
    loss, reward, d = (x.cpu().numpy() for x in ops.preference_loss(dev(logp), None, dev(starts), dev(scale), 1.0))
    assert loss[0] == 1800 and np.array_equal(d[:4], [-1, -1, 1, 1])
    assert loss[1] == 0 and np.isneginf(reward[3]) and not d[4:].any()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for bad, which in (([0, 2, 1, 6, 8], 1), ([-1, 2, 4, 6, 8], 1), ([0, 2, 4, 6, 9], 2), ([0, 2, 4, 2 ** 31 - 1, 8], 2)):
        status.zero_()
        loss, reward, d = (x.cpu().numpy() for x in ops.preference_loss(dev(logp), None, dev(np.array(bad, np.int32)), dev(scale), 1.0, status=status))
        assert int(status) == which and loss[which - 1] == 0 and not reward[2 * which - 2:2 * which].any() and np.isfinite(d).all()


@GPU
def test_arguments_that_do_not_go_together():
    import torch
    from cacti_amd import ops
    r, z, tok = make(11, 4, 64)
    old, adv, ref, scale = (dev(x) for x in policy_inputs(r, z, tok, 1.0))
    z, tok = dev(z), dev(tok)
    mask = torch.ones(4, dtype=torch.bool, device="cuda")
    logp, stats = ops.token_logp_fwd(z, tok)
    for bad in ((z.float(), tok), (z, tok.int()), (z, tok[:2]), (z.cpu(), tok), (z.t(), tok), (z, None)):
        with pytest.raises(AssertionError):
            ops.token_logp_fwd(*bad)
    for more in (dict(mask=mask.int()), dict(mask=mask[:3]), dict(status=scale)):
        with pytest.raises(AssertionError):
            ops.token_logp_fwd(z, tok, **more)
    for bad in ((stats[:2], scale), (stats, scale[:1]), (stats, None), (stats, scale.double())):
        with pytest.raises(AssertionError):
            ops.token_logp_bwd(z, tok, *bad)
    for more in (dict(ref=ref[:2]), dict(acc=z[:2]), dict(acc=z.float()), dict(mask=mask.half())):
        with pytest.raises(AssertionError):
            ops.policy_loss(z, tok, old, adv, scale, **more)
    with pytest.raises(AssertionError):
        ops.policy_loss(z, tok, old, adv, None)
    with pytest.raises(ffi.CactiError):
        ops.policy_loss(z, tok, old, adv, scale, clip=(2.0, 0.1))
    with pytest.raises(ffi.CactiError):
        ops.token_logp_fwd(z, tok, 0.0)
    starts = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    for bad in ((logp, None, starts[:2], scale[:1]), (logp, None, starts, scale), (logp, None, starts.long(), scale[:1]), (logp, scale[:2], starts, scale[:1])):
        with pytest.raises(AssertionError):
            ops.preference_loss(*bad)
    # nothing to do
    assert [x.numel() for x in ops.policy_loss(z[:0], tok[:0], old[:0], adv[:0], scale[:0])] == [0, 0, 0]
    loss, reward, d = ops.preference_loss(logp, None, starts[:1], scale[:0])
    assert loss.numel() == 0 and reward.numel() == 0 and not bool(d.any())


@GPU
def test_captured_and_replayed():
    import torch
    from cacti_amd import ops
    r, z, tok = make(12, 30, 2000)
    old, adv, ref, scale = (dev(x) for x in policy_inputs(r, z, tok, 1.0))
    z, tok = dev(z), dev(tok)
    starts = torch.tensor([0, 7, 15, 22, 30], dtype=torch.int32, device="cuda")

    def step():
        logp, stats = ops.token_logp_fwd(z, tok)
        loss, reward, d = ops.preference_loss(logp, ref, starts, scale[:2])
        return [*ops.policy_loss(z, tok, old, adv, scale, ref=ref, beta=0.1), loss, reward, ops.token_logp_bwd(z, tok, stats, d)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for i in range(4):
        g.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        z.copy_(torch.roll(z, 3, 1))


@GPU
def test_a_reference_or_an_old_policy_far_off():
    """Ratios and e^d beyond fp32, which a coefficient brings back or makes nothing of: without a divergence term (beta 0) what ref is does not
    matter, an advantage of 0 has no loss, and what fp32 can hold is held (e^x's error is that of x, as bounded above)."""
    from cacti_amd import ops
    r, z, tok = make(13, 9, 64)
    old, adv, ref, scale = policy_inputs(r, z, tok, 1.0)
    scale[:] = 1
    z[0, tok[0]] = -np.inf                                                             # a token that the model rules out
    for n, d in ((1, 90), (2, 95), (3, 70)):
        z[n, tok[n]] = z[n].max() - d
    old[:4] = rows64(z, tok, 1.0)[1][:4]
    old[0], ref[:4], adv[:4] = 0, 0, 0.5
    lp = rows64(z, tok, 1.0)[1]
    old[4:8], adv[4:8] = lp[4:8] - [95, 92, 200, 95], [-1e-4, 0, 0, 0.3]
    args = [dev(x) for x in (z, tok, old, adv, scale)]
    bare, off = ops.policy_loss(*args), ops.policy_loss(*args, ref=dev(ref))
    for a, b in zip(bare, off):
        assert np.array_equal(a.cpu().numpy(), b.cpu().numpy(), equal_nan=True)
    at = np.arange(1, 9)                                                               # (the first row: no numbers to compare with)
    for out, beta in ((bare, 0.0), (ops.policy_loss(*args, ref=dev(ref), beta=0.01), 0.01)):
        loss, logp, grad = (x.cpu().numpy() for x in out)
        wl, tl, wp, tp, wg, tg = policy64(z[at], tok[at], old[at], adv[at], ref[at] if beta else None, scale[at], 0.2, 0.2, beta, 1.0)
        near(logp[at], wp, tp, "logp")
        # (the bound of a loss has the ratio's error also where the ratio is clipped; there it is that of adv = 0 and one product)
        clipped = np.where(at == 7, 0, adv[at]).astype(np.float32)
        tl[6] = policy64(z[at], tok[at], old[at], clipped, ref[at] if beta else None, scale[at], 0.2, 0.2, beta, 1.0)[1][6] + 2.0 ** -22
        # what fp32 cannot hold is infinite, and no number of its gradient one that could be taken for it
        fits32 = np.abs(wl) < 3.4e38
        assert np.array_equal(fits32, at != 2) if beta else fits32.all()
        assert np.isposinf(loss[at][~fits32]).all() and not np.isfinite(grad[at][~fits32]).any()
        near(loss[at][fits32], wl[fits32], tl[fits32], "loss")
        wg, tg, grad = wg[fits32], tg[fits32], grad[at][fits32]
        fits = np.abs(wg) < 60000                                                      # (beyond: infinite in f16)
        assert np.isinf(grad[np.abs(wg) > 70000]).all() and not np.isnan(grad).any()
        near(np.where(fits, grad, 0), np.where(fits, wg, 0), tg, "gradient")
        assert np.isneginf(logp[0]) and (np.isposinf(loss[0]) if beta else loss[0] == 0 and not bool(out[2][0].any()))
    assert bare[0][5] == 0 and bare[0][6] == 0 and not bare[2][5:8].any()
    # .. and none of an infinite slope
    scale[:2] = 0
    _, _, grad = ops.policy_loss(*args[:4], dev(scale), ref=dev(ref), beta=0.01)
    assert not grad[:2].any()
    old[6] = np.nan                                                                    # (what is no number stays one)
    loss, _, grad = ops.policy_loss(args[0], args[1], dev(old), *args[3:])
    assert bool(loss[6].isnan()) and bool(grad[6].isnan().all())


@GPU
@pytest.mark.parametrize("wrong", [{k: v} for k in range(9) for v in (-5, 100, 2 ** 31 - 1, -2 ** 31)] +
                         [{0: 24}, {8: 1}, {8: 0}, {3: 4}, {5: 3}, {2: 99, 5: -1}, {1: -1, 3: 99, 5: -1, 7: 99}, {0: 30, 8: -1}])
def test_a_wrong_number_costs_its_own_pairs_alone(wrong):
    """All rows that a good pair has hold what they do where all numbers are right, whatever the others are; all else is 0."""
    import torch
    from cacti_amd import ops
    r = np.random.default_rng(14)
    good = [2, 5, 7, 11, 12, 16, 19, 22, 25]
    logp, ref, scale = r.standard_normal(28).astype(np.float32), r.standard_normal(28).astype(np.float32), r.standard_normal(4).astype(np.float32)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    run = lambda s: [x.cpu().numpy() for x in ops.preference_loss(dev(logp), dev(ref), dev(np.array(s, np.int32)), dev(scale), 0.2, status=status)]
    want = run(good)
    bad = sorted({i for k in wrong for i in (k // 2, (k - 1) // 2) if 0 <= i < 4})
    for i in bad:
        want[0][i] = want[1][2 * i] = want[1][2 * i + 1] = 0
        want[2][good[2 * i]:good[2 * i + 2]] = 0
    assert int(status) == 0
    for _ in range(3):
        status.zero_()
        out = run([wrong.get(k, s) for k, s in enumerate(good)])
        assert int(status) == 1 + max(bad)
        for got, w in zip(out, want):
            assert np.array_equal(got, w)


@GPU
def test_many_pairs_that_there_are_not():
    """Runs of them longer than a workgroup looks at in one go, between pairs that there are."""
    from cacti_amd import ops
    r = np.random.default_rng(15)
    P, N = 1500, 6000
    good = 2 * np.arange(2 * P + 1)
    logp, scale = r.standard_normal(N + 5).astype(np.float32), r.standard_normal(P).astype(np.float32)
    for runs in ([(0, P)], [(3, 700), (701, 1490)], [(0, 256), (257, 300), (900, P)], [(1, 2)]):
        starts, ok = good.copy(), np.ones(P, bool)
        for lo, hi in runs:
            starts[2 * lo + 1:2 * hi:2] = -7
            ok[lo:hi] = False
        loss, reward, d = (x.cpu().numpy() for x in ops.preference_loss(dev(logp), None, dev(starts.astype(np.int32)), dev(scale), 0.3))
        wl, wr, wd = pairs64(logp, None, good, scale, 0.3, 0.0, None, False)
        wd[:N] *= np.repeat(ok, 4)
        for got, want in ((loss, wl * ok), (reward, wr * np.repeat(ok, 2)), (d, wd)):
            near(got, want, 2.0 ** -24 * np.abs(want) + 1e-12, "of a pair")
            assert not got[want == 0].any()
