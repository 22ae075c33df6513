"""Verification of drafted tokens: cacti_hip_verify_draft_f16 against a plain form in numpy's float64.

Results are whole numbers and have to be equal.  Both sides sum in 64 bits; a draw would differ only where r lies within the
sums' rounding of a border, some 65536 * 2^-50 of all draws, which the seeds here do not hit."""
import numpy as np
import pytest

from cacti_amd import ffi

GPU = pytest.mark.gpu
ARGS = dict(T=4, B=2, V=64, target=64, ldt=64, draft=64, ldd=64, tok=64, starts=64, u=64, r=64, temp=1.0, accepted=64, next=64, ws=64,
            ws_bytes=1 << 20, status=None, stream=None)


@pytest.mark.parametrize("change,why", [(dict(T=0), "empty"), (dict(B=0), "empty"), (dict(V=0), "empty"), (dict(V=65537, ldt=65537, ldd=65537), "65536"),
                                        (dict(T=1 << 18, ws_bytes=1 << 40), "2^18"), (dict(ldt=63), "pitch"), (dict(ldd=63), "pitch"),
                                        (dict(target=None), "null"), (dict(tok=None), "null"), (dict(starts=None), "null"), (dict(u=None), "null"),
                                        (dict(r=None), "null"), (dict(accepted=None), "null"), (dict(next=None), "null"), (dict(ws=None), "null"),
                                        (dict(ws_bytes=4), "workspace"), (dict(temp=-1.0), "temperature"), (dict(temp=float("nan")), "temperature"),
                                        (dict(temp=float("inf")), "temperature"), (dict(target=65), "misaligned"), (dict(u=66), "misaligned")])
def test_refuses(change, why):
    L = ffi.lib()
    assert L.cacti_hip_verify_draft_f16(*dict(ARGS, **change).values()) < 0
    assert why in L.cacti_hip_last_error().decode()


@pytest.mark.parametrize("change", [dict(), dict(next=66), dict(next=64 + 6), dict(next=64 - 6)])
def test_refuses_tokens_in_place(change):
    """A row's token is read by the lane of the row before it."""
    L = ffi.lib()
    assert L.cacti_hip_verify_draft_f16(*dict(ARGS, **change).values()) < 0
    assert "share memory" in L.cacti_hip_last_error().decode()


def probabilities(z, temp):
    z = np.where(np.isnan(z), -np.inf, z.astype(np.float64))
    if temp == 0:
        return (np.arange(len(z)) == z.argmax()).astype(np.float64)
    with np.errstate(invalid="ignore"):
        d = np.where(z == z.max(), 0.0, z - z.max())
    w = np.exp(d / temp)
    return w / w.sum()


def reference(target, draft, tok, starts, u, r, temp):
    T, V = target.shape
    accepted, nxt = np.zeros(len(starts) - 1, np.int32), np.zeros(T, np.int64)
    for b in range(len(starts) - 1):
        s, e = starts[b], starts[b + 1]
        for i in range(s, e):
            p = probabilities(target[i], temp)
            w = p
            if i + 1 < e:
                x = tok[i + 1]
                if draft is None or temp == 0:
                    q = (np.arange(V) == x).astype(np.float64)
                else:
                    q = probabilities(draft[i], temp)
                if x < V and np.float64(u[i]) * q[x] < p[x]:
                    nxt[i] = x
                    accepted[b] += 1
                    continue
                w = np.maximum(p - q, 0)
                if w.sum() == 0:
                    w = p
            c = w.cumsum()
            nxt[i] = np.searchsorted(c, np.float64(r[b]) * c[-1], side="right")
            break
    return accepted, nxt


def make(seed, n, V, draft=True, temp=1.0, noise=1.0, spare=0):
    g = np.random.default_rng(seed)
    T = sum(n) + spare
    target = (g.standard_normal((T, V)) * 2.5).astype(np.float16)
    d = (target + g.standard_normal((T, V)) * noise).astype(np.float16)
    tok = np.zeros(T, np.int64)
    for i in range(T - 1):
        if draft:
            tok[i + 1] = g.choice(V, p=probabilities(d[i], temp or 0.1))
        else:
            tok[i + 1] = target[i].astype(np.float64).argmax() if g.random() < 0.7 else g.integers(V)
    starts = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    return [target, d if draft else None, tok, starts, g.random(T).astype(np.float32), g.random(len(n)).astype(np.float32), temp]


def run(target, draft, tok, starts, u, r, temp, **more):
    import torch
    from cacti_amd import ops
    d = lambda x: None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda()
    a, nxt = ops.verify_draft(d(target), d(draft), d(tok.astype(np.uint16).view(np.int16)), d(starts), d(u), d(r), temperature=temp, **more)
    return a.cpu().numpy(), nxt.cpu().numpy().view(np.uint16).astype(np.int64)


def check(args):
    a, nxt = run(*args)
    wa, wn = reference(*args)
    rows = args[3][-1]
    assert np.array_equal(a, wa), (a, wa)
    assert np.array_equal(nxt[:rows], wn[:rows]), np.argwhere(nxt[:rows] != wn[:rows])[:4]
    return a


@GPU
@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("temp", [1.0, 0.6, 0.0])
@pytest.mark.parametrize("n,V", [([5], 32000), ([1, 4, 0, 8, 2], 8192), ([3, 3], 1000), ([4, 1], 1021), ([2], 7), ([3], 1), ([2, 2], 65536),
                                 ([1] * 70 + [3], 130)])
def test_verify(n, V, temp, draft):
    print("verify_draft", n[:6], V, temp, draft, flush=True)
    check(make(V + len(n), n, V, draft, temp))
    check(make(V + len(n) + 1, n, V, draft, temp, noise=0.05, spare=2))


@GPU
def test_every_outcome_is_met():
    """Over one large batch: sequences that keep none, some and all of what was drafted."""
    a = check(make(9, [5] * 60, 500))
    assert set(a) >= {0, 1, 2, 3, 4}


@GPU
def test_the_same_probabilities_keep_everything():
    args = make(10, [6, 6], 3000)
    args[1] = args[0].copy()
    args[4][:] = np.float32(1 - 2.0 ** -24)
    assert check(args).tolist() == [5, 5]


@GPU
def test_draws_follow_the_target():
    """What comes out in place of one drafted token has the target's distribution whatever the drafting model's is: 4096
    independent sequences over 4 tokens, each count within five standard deviations."""
    g = np.random.default_rng(12)
    V, B = 4, 4096
    p, q = np.array([0.1, 0.5, 0.15, 0.25]), np.array([0.4, 0.1, 0.3, 0.2])
    target, draft = (np.tile(np.log(x).astype(np.float16), (2 * B, 1)) for x in (p, q))
    p = probabilities(target[0], 1.0)
    q = probabilities(draft[0], 1.0)
    tok = np.zeros(2 * B, np.int64)
    tok[1::2] = g.choice(V, size=B, p=q)
    args = [target, draft, tok, np.arange(0, 2 * B + 1, 2, dtype=np.int32), g.random(2 * B).astype(np.float32), g.random(B).astype(np.float32), 1.0]
    check(args)
    _, nxt = run(*args)
    seen = np.bincount(nxt[::2], minlength=V)
    assert (np.abs(seen - B * p) <= 5 * np.sqrt(B * p * (1 - p))).all(), (seen, B * p)


@GPU
def test_random_numbers_at_the_ends():
    for u, r in ((0.0, 0.0), (1 - 2.0 ** -24, 1 - 2.0 ** -24)):
        args = make(13, [4, 3, 1], 777)
        args[4][:], args[5][:] = u, r
        check(args)


@GPU
def test_logits_that_are_no_numbers():
    """-inf and NaN are never chosen, +inf always is; several of them share; a row without a finite logit is even; of equal
    ones the first is the arg max."""
    for temp in (1.0, 0.0):
        for draft in (True, False):
            args = make(14, [3, 3, 2, 2, 2], 300, draft, temp)
            t = args[0]
            t[0, ::2], t[1, 5:9], t[3, 7] = np.nan, -np.inf, np.inf
            t[4, [9, 30, 31]], t[6, :] = np.inf, -np.inf
            t[8, :] = np.nan
            t[10, :] = 1.0
            if draft:
                args[1][2, ::3], args[1][0, 1::5], args[1][6, :] = np.nan, -np.inf, -np.inf
            check(args)


@GPU
def test_ids_beyond_the_vocabulary():
    """Never kept, and named."""
    import torch
    args = make(15, [3, 3], 100)
    args[1] = args[0].copy()
    args[2][4] = 100
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    a, nxt = run(*args, status=status)
    assert a.tolist()[1] == 0 and int(status) == 1 + 4 and nxt[3] < 100
    args[3][2] = 9                                            # rows beyond T
    status.zero_()
    a, _ = run(*args, status=status)
    assert a[1] == 0 and int(status) >= 1


@GPU
def test_rows_may_be_strided_and_lie_anywhere():
    import torch
    from cacti_amd import ops
    for V in (1000, 1001):
        args = make(16, [4, 2, 3], V)
        want = reference(*args)
        d = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()
        for ld, off in ((V + 3, 1), (V + 8, 8), (2 * V, 5)):
            big = [torch.zeros(9 * ld + 16, dtype=torch.float16, device="cuda") for _ in range(2)]
            rows = [x[off:off + 9 * ld].view(9, ld)[:, :V] for x in big]
            for x, y in zip(rows, args[:2]):
                x.copy_(d(y))
            a, nxt = ops.verify_draft(rows[0], rows[1], d(args[2].astype(np.int16)), d(args[3]), d(args[4]), d(args[5]))
            assert np.array_equal(a.cpu().numpy(), want[0]) and np.array_equal(nxt.cpu().numpy(), want[1])


@GPU
def test_arguments_that_do_not_go_together():
    import torch
    from cacti_amd import ops
    z = torch.zeros((4, 16), dtype=torch.float16, device="cuda")
    tok, starts = torch.zeros(4, dtype=torch.int16, device="cuda"), torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    u, r = torch.zeros(4, device="cuda"), torch.zeros(1, device="cuda")
    for bad in ((z.float(), None, tok, starts, u, r), (z, z[:2], tok, starts, u, r), (z, None, tok.int(), starts, u, r),
                (z, None, tok, starts.long(), u, r), (z, None, tok, starts, u[:3], r), (z, None, tok, starts, u, u), (z.cpu(), None, tok, starts, u, r),
                (z, None, tok[:3], starts, u, r), (z.t(), None, tok, starts, u, r)):
        with pytest.raises(AssertionError):
            ops.verify_draft(*bad)
    with pytest.raises(ffi.CactiError):
        ops.verify_draft(z, None, tok, starts, u, r, temperature=-1.0)
    a, nxt = ops.verify_draft(z[:0], None, tok[:0], torch.zeros(3, dtype=torch.int32, device="cuda"), u[:0], u[:2])
    assert a.tolist() == [0, 0] and nxt.numel() == 0


@GPU
def test_captured_and_replayed():
    import torch
    from cacti_amd import ops
    args = make(17, [5, 3, 1], 2000)
    d = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()
    dev = [d(args[0]), d(args[1]), d(args[2].astype(np.int16)), d(args[3]), d(args[4]), d(args[5])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.verify_draft(*dev)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ops.verify_draft(*dev)
    for i in range(4):
        g.replay()
        want = ops.verify_draft(*dev)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        dev[4].copy_(torch.rand_like(dev[4]))
        dev[5].copy_(torch.rand_like(dev[5]))
        dev[0].copy_(torch.roll(dev[0], 1, 1))
