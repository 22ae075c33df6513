"""Low-rank adapters of many requests, forward and adjoint, against float64.

What the kernels round.  h: a sum of K exact products in fp32, at most K 2^-24 sum |x A| (K steps in any order); dh the same over N.  Of
either, f16 takes two terms, scaled by the power of two that brings the largest of a row to 2^10 .. 2^11: what is left is 2^-22 of it, or half a
step of the second term's subnormal range, 2^-25 for a largest of 2^10, of which 2^-25 is far more than that.  For dA and dB a row's scale is
made that of the largest row so far: a row 2^-25 and less of that scale, whose largest is below 2^-24 of that row's, is lost.  y: R products of those and two
terms each, 2 R 2^-24 sum |h B|, the scale and the base in fp32 (2^-22 of either), and half a step of f16: 2^-11 |y|, 2^-25 below its normal
range.  dA and dB: 2 T + T / 64 additions.  In what follows each product carries the errors of both factors."""
import numpy as np
import pytest

from cacti_amd import ffi

GPU = pytest.mark.gpu
P0, STEP = 0x100000, 0x10000
FWD = dict(T=4, S=2, K=64, N=64, R=16, n=2, max_new=4, x=P0, ldx=64, A=P0 + STEP, B=P0 + 2 * STEP, starts=64, ids=64, scale=64, base=P0 + 3 * STEP, ldb=64,
           y=P0 + 4 * STEP, ldy=64, h=P0 + 5 * STEP, ws=None, ws_bytes=0, status=None, stream=None)
BWD = dict(T=4, S=2, K=64, N=64, R=16, n=2, max_new=4, x=P0, ldx=64, A=P0 + STEP, B=P0 + 2 * STEP, starts=64, ids=64, scale=64, h=P0 + 3 * STEP,
           dy=P0 + 4 * STEP, lddy=64, dx=P0 + 5 * STEP, lddx=64, dx_acc=0, dA=P0 + 6 * STEP, dA_acc=0, dB=P0 + 7 * STEP, dB_acc=0, ws=P0 + 8 * STEP,
           ws_bytes=1 << 30, status=None, stream=None)
COMMON = [(dict(T=0), "empty"), (dict(S=0), "empty"), (dict(K=0), "empty"), (dict(R=0), "empty"), (dict(n=0), "empty"), (dict(max_new=0), "empty"),
          (dict(x=None), "null"), (dict(A=None), "null"), (dict(B=None), "null"), (dict(starts=None), "null"), (dict(ids=None), "null"),
          (dict(scale=None), "null"), (dict(R=12), "R %"), (dict(R=136), "R <="), (dict(K=60, ldx=64), "multiples"), (dict(N=60), "multiples"),
          (dict(n=1025), "1024"), (dict(T=(1 << 24) + 1), "2^24"), (dict(ldx=56), "pitch"), (dict(ldx=68), "multiple"), (dict(x=P0 + 8), "aligned"),
          (dict(A=P0 + STEP + 2), "aligned"), (dict(starts=66), "aligned"), (dict(status=66), "aligned")]
REFUSED = [("cacti_hip_adapter_fwd", FWD, c) for c in COMMON + [
    (dict(y=None), "null"), (dict(h=None), "null"), (dict(ldy=56), "pitch"), (dict(ldb=66), "multiple"), (dict(base=P0 + 3 * STEP + 8), "aligned"),
    (dict(y=P0), "shares"), (dict(y=P0 + 128), "shares"), (dict(y=P0 + 3 * STEP, ldy=72), "place"), (dict(y=P0 + 3 * STEP + 16), "place"),
    (dict(T=100, max_new=100, K=8192, R=64, ldx=8192, x=1 << 30), "workspace")]] + \
          [("cacti_hip_adapter_bwd", BWD, c) for c in COMMON + [
              (dict(h=None), "null"), (dict(dy=None), "null"), (dict(dx=None), "null"), (dict(dA=None), "null"), (dict(dB=None), "null"), (dict(ws=None), "null"),
              (dict(lddy=56), "pitch"), (dict(lddx=68), "multiple"), (dict(dx=P0), "shares"), (dict(dx=P0 + 4 * STEP + 16), "shares"),
              (dict(ws_bytes=4096), "workspace"), (dict(dB=P0 + 7 * STEP + 8), "aligned")]]


REFUSED += [("cacti_hip_adapter_bwd", BWD, c) for c in [
    (dict(dB=P0 + 6 * STEP + 1024), "dA shares"), (dict(dA=P0 + 7 * STEP), "dA shares"),
    (dict(T=1 << 24, max_new=1 << 24, K=1 << 16, ldx=1 << 16, lddx=1 << 16, dy=1 << 44, dx=1 << 46, dB=1 << 47, ws_bytes=1 << 60), "too many tiles")]]


@pytest.mark.parametrize("entry,args,change", REFUSED)
def test_refuses(entry, args, change):
    change, why = change
    L = ffi.lib()
    assert getattr(L, entry)(*dict(args, **{k: v for k, v in change.items() if k in args}).values()) < 0
    assert why in L.cacti_hip_last_error().decode()


def test_workspace_holds_a_block_for_each_adapter():
    ws = ffi.lib().cacti_hip_adapter_bwd_workspace
    assert ws(0, 64, 64, 16, 1) == 0
    for T in (1, 64, 1000, 100000):
        for n in (1, 7, 1000):
            assert ws(T, 256, 128, 16, n) >= T * 16 * 4 + T * 4 + n * 16 * 384 * 4


def dev(x):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


class Case:
    def __init__(self, seed, counts, ids, K, N, R, n, behind=0):
        r = np.random.default_rng(seed)
        self.counts, self.K, self.N, self.R, self.n = counts, K, N, R, n
        self.starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.ids = np.array(ids, np.int32)
        self.T = int(self.starts[-1]) + behind
        h = lambda *s, std=1.0: (r.standard_normal(s) * std).astype(np.float16)
        self.x, self.A, self.B = h(self.T, K), h(n, R, K, std=K ** -0.5), h(n, N, R, std=0.2)
        self.base, self.dy = h(self.T, N), h(self.T, N, std=0.3)
        self.dx0, self.dA0, self.dB0 = h(self.T, K), h(n, R, K), h(n, N, R)
        self.scale = (2.0 ** r.integers(-2, 2, n) * r.choice([-1, 1], n)).astype(np.float32)
        self.scale[0] = 0.7

    def of(self, names):
        return [dev(getattr(self, x)) for x in names.split()]

    def rows(self, a):
        return np.concatenate([np.arange(self.starts[s], self.starts[s + 1]) for s in range(len(self.ids)) if self.ids[s] == a] + [np.zeros(0, int)]).astype(int)

    def forward(self, based):
        """y, h and their bounds (rows of an adapter or none alone)."""
        y = self.base.astype(np.float64) if based else np.zeros((self.T, self.N))
        h, th, ty = np.zeros((self.T, self.R)), np.zeros((self.T, self.R)), np.zeros((self.T, self.N))
        for a in range(self.n):
            at = self.rows(a)
            x, A, B, s = self.x[at].astype(np.float64), self.A[a].astype(np.float64), self.B[a].astype(np.float64), float(self.scale[a])
            h[at] = x @ A.T
            th[at] = self.K * 2.0 ** -24 * (np.abs(x) @ np.abs(A).T)
            left = th[at] + 2.0 ** -22 * np.abs(h[at]) + 2.0 ** -25 * np.abs(h[at]).max(1, keepdims=True)
            d = s * (h[at] @ B.T)
            ty[at] = abs(s) * ((left + 2 * self.R * 2.0 ** -24 * np.abs(h[at])) @ np.abs(B).T) + 2.0 ** -22 * (np.abs(d) + np.abs(y[at]))
            y[at] += d
            ty[at] += 2.0 ** -11 * np.abs(y[at]) + 2.0 ** -25
        return y, ty, h, th

    def adjoint(self, h, acc):
        """dx, dA, dB and their bounds, for the h that the kernel has."""
        dx, dA, dB = ((x.astype(np.float64) if acc else np.zeros(x.shape)) for x in (self.dx0, self.dA0, self.dB0))
        tx, tA, tB = (2.0 ** -22 * np.abs(x) for x in (dx, dA, dB))
        h = h.astype(np.float64)
        for a in range(self.n):
            at = self.rows(a)
            x, dy, A, B, s = self.x[at].astype(np.float64), self.dy[at].astype(np.float64), self.A[a].astype(np.float64), self.B[a].astype(np.float64), float(self.scale[a])
            dh = dy @ B
            own = self.N * 2.0 ** -24 * (np.abs(dy) @ np.abs(B)) + 2.0 ** -22 * np.abs(dh)
            left = own + 2.0 ** -25 * np.abs(dh).max(1, keepdims=True)
            most = lambda v: 2.0 ** -24 * np.abs(v).max() if len(at) else 0.0
            adds = (2 * len(at) + len(at) / 64 + 4) * 2.0 ** -24
            d = s * (dh @ A)
            dx[at] += d
            tx[at] += abs(s) * ((left + 2 * self.R * 2.0 ** -24 * np.abs(dh)) @ np.abs(A)) + 2.0 ** -22 * np.abs(d)
            dA[a] += s * (dh.T @ x)
            tA[a] += abs(s) * ((own + most(dh) + adds * np.abs(dh)).T @ np.abs(x))
            dB[a] += s * (dy.T @ h[at])
            tB[a] += abs(s) * (np.abs(dy).T @ ((2.0 ** -22 + adds) * np.abs(h[at]) + most(h[at])))
        return [(v, t + 2.0 ** -11 * np.abs(v) + 2.0 ** -25) for v, t in ((dx, tx), (dA, tA), (dB, tB))]


def near(got, want, tol, what):
    got = np.asarray(got.cpu() if hasattr(got, "cpu") else got).astype(np.float64)
    assert got.shape == want.shape and np.isfinite(got).all(), what
    off = np.abs(got - want) - tol
    assert (off <= 0).all(), "%s: %.3g beyond its bound" % (what, off.max())


def check(c, max_new=None, seed=0):
    from cacti_amd import ops
    x, A, B, starts, ids, scale, base, dy = c.of("x A B starts ids scale base dy")
    used = slice(0, int(c.starts[-1]))
    for b in (None, base):
        y, h = ops.adapter_fwd(x, A, B, starts, ids, scale, base=b, max_new=max_new)
        wy, ty, wh, th = c.forward(b is not None)
        near(h[used], wh[used], th[used], "h")
        near(y[used], wy[used], ty[used], "y")
    for acc in (False, True):
        into = c.of("dx0 dA0 dB0") if acc else [None] * 3
        got = ops.adapter_bwd(x, A, B, starts, ids, scale, h, dy, *into, max_new=max_new)
        hh = h.cpu().numpy()
        hh[c.starts[-1]:] = 0
        for g, i, (want, tol), what in zip(got, into, c.adjoint(hh, acc), ("dx", "dA", "dB")):
            assert i is None or g is i
            rows = used if what == "dx" else slice(None)
            near(g[rows], want[rows], tol[rows], what)
    return y, h, got


@GPU
@pytest.mark.parametrize("counts,ids", [([1], [0]), ([1] * 9, [0, 2, -1, 2, 1, 0, 0, -1, 2]), ([3, 0, 16, 17, 1], [1, 0, -1, 1, 2]), ([0, 0], [0, 1]),
                                        ([70, 5, 129], [2, 2, 0]), ([333], [1])])
@pytest.mark.parametrize("K,N,R", [(8, 8, 8), (64, 40, 16), (40, 136, 24), (264, 72, 64), (136, 520, 128), (1000, 1032, 8)])
def test_adapter(counts, ids, K, N, R):
    print("adapter", counts, ids, K, N, R, flush=True)
    check(Case(K + N + R + len(counts), counts, ids, K, N, R, 3, behind=1))
    check(Case(K + N + R, counts, ids, K, N, R, 3), max_new=max(max(counts), 1))


@GPU
@pytest.mark.parametrize("counts,ids,K,N,R,n", [([1] * 40, [i % 7 - 1 for i in range(40)], 3200, 3200, 16, 6), ([700, 41], [0, 0], 1024, 2816, 32, 1),
                                                ([1500], [0], 688, 256, 16, 1), ([9] * 70, [i % 50 for i in range(70)], 256, 688, 16, 64)])
def test_adapter_of_a_models_widths(counts, ids, K, N, R, n):
    print("adapter", len(counts), K, N, R, flush=True)
    check(Case(K + N + R, counts, ids, K, N, R, n), max_new=max(counts))


TWO = [([1] * 9, [0, 2, -1, 2, 1, 0, 0, -1, 2], 8640, 264, 32), ([3, 0, 16, 33, 1], [1, 0, -1, 1, 2], 8640, 1032, 64), ([70], [1], 4104, 520, 128),
       ([1] * 140, [i % 4 - 1 for i in range(140)], 4000, 264, 64), ([17] * 70, [i % 3 for i in range(70)], 2000, 72, 128),
       ([5000, 7, 3400], [2, -1, 0], 72, 40, 16), ([8200], [1], 264, 136, 24)]


@pytest.mark.parametrize("counts,ids,K,N,R", TWO)
def test_parts_of_two_launches_have_a_workspace(counts, ids, K, N, R):
    ws = ffi.lib().cacti_hip_adapter_fwd_workspace
    T = sum(counts)
    assert ws(T, len(ids), K, N, R, max(counts)) % (T * R * 4) == 0
    if K > 4096:
        assert ws(T, len(ids), K, N, R, max(counts)) >= 2 * T * R * 4


@GPU
@pytest.mark.parametrize("counts,ids,K,N,R", TWO)
def test_in_two_launches(counts, ids, K, N, R):
    """Sizes whose h is formed first: a long K, tiles between half the device and all of it, many rows; with the base's place, numbers that do
    not fit, and adapters of NaN that nobody has."""
    import torch
    from cacti_amd import ops
    print("adapter", len(counts), sum(counts), K, N, R, flush=True)
    c = Case(K + N + R, counts, ids, K, N, R, 4, behind=3)
    c.A[3], c.B[3] = np.nan, np.inf
    x, A, B, starts, scale, base = c.of("x A B starts scale base")
    c.n = 3
    used, most = int(c.starts[-1]), max(counts)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    wy, ty, wh, th = c.forward(True)
    bare, _ = ops.adapter_fwd(x, A, B, starts, dev(c.ids), scale, max_new=most)
    near(bare[:used], *[v[:used] for v in c.forward(False)[:2]], "y alone")
    got, h = ops.adapter_fwd(x, A, B, starts, dev(c.ids), scale, base=base, max_new=most, status=status)
    near(h[:used], wh[:used], th[:used], "h")
    near(got[:used], wy[:used], ty[:used], "y")
    own = base.clone()
    ops.adapter_fwd(x, A, B, starts, dev(c.ids), scale, base=own, out=own, max_new=most)
    assert torch.equal(own[:used], got[:used]) and torch.equal(own[used:], base[used:]) and int(status) == 0
    bad = c.ids.copy()
    bad[-1] = 4
    y, _ = ops.adapter_fwd(x, A, B, starts, dev(bad), scale, base=base, max_new=most, status=status)
    last = slice(int(c.starts[-2]), used)
    assert int(status) == len(ids) and torch.equal(y[last], base[last]) and torch.equal(y[:last.start], got[:last.start])


@GPU
@pytest.mark.parametrize("S,n,most,R", [(1500, 1024, 1, 8), (700, 700, 2, 16), (130, 900, 7, 24), (2100, 3, 1, 8), (65, 2, 9, 72)])
def test_many_sequences_and_many_adapters(S, n, most, R):
    """Lists of rows by several waves, adapters without rows, with one block of them and with more."""
    r = np.random.default_rng(S)
    check(Case(S + n, [int(x) for x in r.integers(0, most + 1, S)], [int(x) for x in r.integers(-1, n, S)], 24, 40, R, n, behind=2), max_new=most)


@GPU
def test_gradient_against_differences():
    """Differences of sum(dy y) in float64 along random directions, at the kernel's gradients: y is linear in each of x, A and B, so a
    central difference is exact but for its own rounding."""
    from cacti_amd import ops
    c = Case(3, [5, 20, 2], [1, 0, 1], 32, 48, 16, 2)
    x, A, B, starts, ids, scale, dy = c.of("x A B starts ids scale dy")
    _, h = ops.adapter_fwd(x, A, B, starts, ids, scale)
    grads = [g.cpu().numpy().astype(np.float64) for g in ops.adapter_bwd(x, A, B, starts, ids, scale, h, dy)]
    bounds = [t for _, t in c.adjoint(h.cpu().numpy(), False)]
    r = np.random.default_rng(4)

    def f():
        return sum(float(c.scale[a]) * (c.dy[at].astype(np.float64) * (c.x[at].astype(np.float64) @ c.A[a].astype(np.float64).T @ c.B[a].astype(np.float64).T)).sum()
                   for a in range(2) for at in [c.rows(a)])

    # (dB is that of the h which the kernel rounded: bounded by its own error times |dy|)
    _, _, _, th = c.forward(False)
    slack = sum((np.abs(c.dy[c.rows(a)]).astype(np.float64) @ np.ones((48, 1)) * th[c.rows(a)]).sum() * abs(c.scale[a]) for a in range(2)) * 4
    for name, g, t in zip(("x", "A", "B"), grads, bounds):
        for _ in range(3):
            was = getattr(c, name)
            d = r.standard_normal(was.shape)
            setattr(c, name, was.astype(np.float64) + 0.5 * d)
            up = f()
            setattr(c, name, was.astype(np.float64) - 0.5 * d)
            num = up - f()
            setattr(c, name, was)
            assert abs(num - (g * d).sum()) <= (t * np.abs(d)).sum() + slack + 1e-9 * abs(up)


@GPU
def test_in_the_bases_place_strided_rows_and_what_is_beside_them():
    import torch
    from cacti_amd import ops
    c = Case(5, [4, 18, 1], [0, -1, 1], 72, 88, 16, 2, behind=2)
    x, A, B, starts, ids, scale, base, dy = c.of("x A B starts ids scale base dy")
    want, h0 = ops.adapter_fwd(x, A, B, starts, ids, scale, base=base)
    dx0, dA0, dB0 = ops.adapter_bwd(x, A, B, starts, ids, scale, h0, dy)
    used = int(c.starts[-1])

    def wide(t, left, right, fill):
        big = torch.full((t.shape[0], left + t.shape[1] + right), fill, dtype=t.dtype, device="cuda")
        v = big[:, left:left + t.shape[1]]
        v.copy_(t)
        return big, v

    (_, xs), (bb, bs), (_, ds) = wide(x, 8, 16, 3.0), wide(base, 16, 0, 5.0), wide(dy, 0, 8, 2.0)
    keep = bs.clone()
    got, h = ops.adapter_fwd(xs, A, B, starts, ids, scale, base=bs, out=bs)
    assert got is bs and torch.equal(bs[:used], want[:used]) and torch.equal(h[:used], h0[:used])
    assert torch.equal(bs[used:], keep[used:]) and bool((bb[:, :16] == 5).all())
    out, o = wide(torch.full_like(base, 7.0), 8, 8, 9.0)
    ops.adapter_fwd(xs, A, B, starts, ids, scale, base=base, out=o)
    assert torch.equal(o[:used], want[:used]) and bool((o[used:] == 7).all()) and bool((out[:, :8] == 9).all()) and bool((out[:, -8:] == 9).all())
    into, v = wide(torch.full_like(x, 0.0), 8, 8, 4.0)
    dx, dA, dB = ops.adapter_bwd(xs, A, B, starts, ids, scale, h, ds, dx_acc=v)
    assert dx is v and torch.equal(v[:used], dx0[:used]) and torch.equal(dA, dA0) and torch.equal(dB, dB0)
    assert not bool(v[used:].any()) and bool((into[:, :8] == 4).all()) and bool((into[:, -8:] == 4).all())
    # rows without an adapter
    assert torch.equal(want[4:22], base[4:22]) and not bool(dx0[4:22].any()) and not bool(h0[4:22].any())


@GPU
def test_adapters_without_rows_and_values_that_are_no_numbers():
    import torch
    from cacti_amd import ops
    c = Case(6, [5, 7], [2, 2], 64, 64, 8, 4)
    x, A, B, starts, ids, scale, base, dy = c.of("x A B starts ids scale base dy")
    A[0], B[1], A[3] = float("nan"), float("inf"), float("nan")              # of adapters that nobody has
    y, h = ops.adapter_fwd(x, A, B, starts, ids, scale, base=base)
    _, dA, dB = ops.adapter_bwd(x, A, B, starts, ids, scale, h, dy)
    assert bool(torch.isfinite(y).all()) and bool(torch.isfinite(dA).all()) and bool(torch.isfinite(dB).all())
    assert not bool(dA[[0, 1, 3]].any()) and not bool(dB[[0, 1, 3]].any()) and bool(dA[2].any())
    old = dA.clone().fill_(1.5)
    ops.adapter_bwd(x, A, B, starts, ids, scale, h, dy, dA_acc=old)
    assert bool((old[[0, 1, 3]] == 1.5).all())
    # a row's NaN is its own
    x[6, 3] = float("nan")
    y2, h2 = ops.adapter_fwd(x, A, B, starts, ids, scale, base=base)
    rows = torch.arange(12, device="cuda") != 6
    assert bool(torch.isnan(y2[6]).all()) and torch.equal(y2[rows], y[rows])
    # an h beyond f16's range is what it is; y is beyond it too
    x[6] = 60000.0
    A[2, 1] = 100.0
    y3, h3 = ops.adapter_fwd(x, A, B, starts, ids, scale, base=base)
    assert float(h3[6, 1]) == 60000.0 * 64 * 100 or abs(float(h3[6, 1]) / 384e6 - 1) < 1e-3
    assert bool(torch.isinf(y3[6]).all()) and bool(torch.isfinite(y3[rows]).all())


@GPU
def test_numbers_that_do_not_fit():
    import torch
    from cacti_amd import ops
    c = Case(7, [4, 3, 5, 6], [0, 1, 1, 0], 64, 64, 16, 2)
    x, A, B, scale, base, dy = c.of("x A B scale base dy")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    good, h = ops.adapter_fwd(x, A, B, dev(c.starts), dev(c.ids), scale, base=base)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    # an id that is none: no adapter
    for bad in (2, -2, 2 ** 31 - 1):
        status.zero_()
        y, _ = ops.adapter_fwd(x, A, B, dev(c.starts), i32([0, bad, 1, 0]), scale, base=base, status=status)
        assert int(status) == 2 and torch.equal(y[4:7], base[4:7]) and torch.equal(y[7:], good[7:]) and torch.equal(y[:4], good[:4])
        status.zero_()
        dx, _, _ = ops.adapter_bwd(x, A, B, dev(c.starts), i32([0, bad, 1, 0]), scale, h, dy, status=status)
        assert int(status) == 2 and not bool(dx[4:7].any())
    # rows that there are not, or more than was said: none of them
    for starts, which, most in (([0, 4, 7, 12, 19], 4, None), ([0, 4, 7, 12, 18], 4, 5), ([-1, 4, 7, 12, 18], 1, None), ([0, 4, 7, 12, -2 ** 31], 4, None)):
        for call in ("fwd", "bwd"):
            status.zero_()
            out = torch.full_like(base if call == "fwd" else x, 7.0)
            if call == "fwd":
                ops.adapter_fwd(x, A, B, i32(starts), dev(c.ids), scale, base=base, out=out, max_new=most, status=status)
                want = good
            else:
                out.zero_()
                ops.adapter_bwd(x, A, B, i32(starts), dev(c.ids), scale, h, dy, dx_acc=out, max_new=most, status=status)
                want = ops.adapter_bwd(x, A, B, dev(c.starts), dev(c.ids), scale, h, dy)[0]
            assert int(status) == which
            gone = slice(12, 18) if which == 4 else slice(0, 4)
            keep = torch.ones(18, dtype=torch.bool, device="cuda")
            keep[gone] = False
            assert torch.equal(out[keep], want[keep]) and bool((out[gone] == (7 if call == "fwd" else 0)).all())


@GPU
def test_arguments_that_do_not_go_together():
    import torch
    from cacti_amd import ops
    c = Case(8, [4, 3], [0, 1], 64, 40, 16, 2)
    x, A, B, starts, ids, scale, base, dy = c.of("x A B starts ids scale base dy")
    _, h = ops.adapter_fwd(x, A, B, starts, ids, scale)
    good = (x, A, B, starts, ids, scale)
    for i, bad in ((0, x.float()), (0, x[:, :32]), (0, x.cpu()), (1, A[:1]), (1, A[:, :8].contiguous()), (1, A.transpose(1, 2)), (2, B[0]), (3, starts.long()),
                   (3, starts[:2]), (4, ids[:1]), (4, None), (5, scale[:1]), (5, scale.half())):
        args = list(good)
        args[i] = bad
        with pytest.raises(AssertionError):
            ops.adapter_fwd(*args)
    for more in (dict(base=base[:3]), dict(base=base.float()), dict(out=base[:, :32]), dict(max_new=0), dict(status=scale)):
        with pytest.raises(AssertionError):
            ops.adapter_fwd(*good, **more)
    for bad in ((h[:3], dy), (h.half(), dy), (h, dy[:, :32])):
        with pytest.raises(AssertionError):
            ops.adapter_bwd(*good, *bad)
    for more in (dict(dx_acc=x[:3]), dict(dA_acc=A[:1]), dict(dB_acc=B.float())):
        with pytest.raises(AssertionError):
            ops.adapter_bwd(*good, h, dy, **more)
    with pytest.raises(ffi.CactiError):
        ops.adapter_fwd(*good, out=x[:, :40])
    # no rows, no sequences
    y, h = ops.adapter_fwd(x[:0], A, B, starts * 0, ids, scale)
    assert y.shape == (0, 40) and h.shape == (0, 16)
    dx, dA, dB = ops.adapter_bwd(x[:0], A, B, starts * 0, ids, scale, h, dy[:0])
    assert dx.shape == (0, 64) and not bool(dA.any()) and not bool(dB.any())


@GPU
def test_captured_and_replayed():
    """A step follows ids that change between replays; its gradients are captured too."""
    import torch
    from cacti_amd import ops
    c = Case(9, [1, 30, 7, 2], [0, 1, -1, 2], 136, 264, 16, 3)
    x, A, B, starts, ids, scale, base, dy = c.of("x A B starts ids scale base dy")

    def step():
        y, h = ops.adapter_fwd(x, A, B, starts, ids, scale, base=base, max_new=30)
        return [y, h, *ops.adapter_bwd(x, A, B, starts, ids, scale, h, dy, max_new=30)]

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
        ids.copy_(torch.roll(ids, 1))
        x.copy_(torch.roll(x, 5, 1))


# Results over what is read or written beside them.  (Places far enough apart for each operand's size.)
APART = [("cacti_hip_adapter_fwd", FWD, c) for c in [
    (dict(y=P0 + STEP), "y or h"), (dict(y=P0 + 2 * STEP - 496), "y or h"), (dict(h=P0 + 4 * STEP + 128), "y or h"), (dict(h=P0), "y or h"),
    (dict(h=P0 + 3 * STEP + 384), "y or h"), (dict(h=P0 + 2 * STEP - 240), "y or h"), (dict(h=P0 + 2 * STEP + 4080), "y or h")]] + \
        [("cacti_hip_adapter_bwd", BWD, c) for c in [
            (dict(dx=P0 + STEP + 4080), "dx shares"), (dict(dx=P0 + 2 * STEP), "dx shares"), (dict(dx=P0 + 3 * STEP + 240), "dx shares")] +
         [({w: P0 + i * STEP + o}, "dA or dB") for w in ("dA", "dB") for i, o in ((0, 0), (0, 496), (1, 0), (2, 4080), (3, 240), (4, -4080), (5, 496), (5, -4080))]]


@pytest.mark.parametrize("entry,args,change", APART)
def test_refuses_results_over_operands(entry, args, change):
    test_refuses(entry, args, change)


@pytest.mark.parametrize("T,K,N,R,n", [(512, 3200, 8640, 128, 1024), (64, 3200, 8640, 128, 64), (1, 3200, 3200, 128, 1024), (2048, 8640, 3200, 64, 1000),
                                       (4096, 3200, 3200, 16, 3), (9600, 256, 256, 8, 1024)])
def test_workspace_goes_by_the_rows(T, K, N, R, n):
    """No more parts of gradients than adapters with more than a block of 64 rows may have, or 32 MB of them."""
    rest = T * 2 * 64 * 8 + 3 * 4 * T + 8 * (n + 1) + (1 << 13)
    assert ffi.lib().cacti_hip_adapter_bwd_workspace(T, K, N, R, n) <= rest + max(2 * T // 65 * R * (K + N) * 4, 32 << 20)


@GPU
@pytest.mark.parametrize("counts", [[65] * 40, [129] * 21, [64, 65] * 20, [1, 200, 64, 0, 65, 66, 3] * 6])
def test_adapters_of_several_blocks_among_others(counts):
    """As many parts as there can be (65 rows: two blocks), and adapters with and without between them."""
    print("adapter", counts[:2], len(counts), flush=True)
    n = len(counts)
    ids = [(7 * i) % n for i in range(n)]
    assert len(set(ids)) == n or n % 7 == 0
    check(Case(n, counts, ids, 24, 40, 16, n), max_new=max(counts))


def rows_by_powers_of_two(c, order, top=2):
    """Rows of dy and x by powers of two of 2^-20 .. 2^2 and 2^-12 .. 2^2, so that the largest row so far changes from step to step."""
    r = np.random.default_rng(c.T)
    e = np.linspace(-20, top, c.T).round()
    e = dict(rising=e, falling=e[::-1], mixed=r.permutation(e))[order]
    c.dy = (c.dy * 2.0 ** e[:, None]).astype(np.float16)
    c.x = (c.x * 2.0 ** ((e[::-1, None] - top) * 14 / 22 + top).round()).astype(np.float16)


STEPS = [([1001, 5, 697], [0, 1, 0], 3200, 3200, 16, 2), ([300, 813], [0, 0], 3200, 3200, 128, 1), ([900, 1131], [1, 0], 3200, 3200, 64, 3),
         ([129, 1, 1500], [0, 2, 2], 1024, 8640, 24, 3)]


@pytest.mark.parametrize("counts,ids,K,N,R,n", STEPS)
def test_blocks_of_more_than_a_step(counts, ids, K, N, R, n):
    """The cases below have blocks of more than 64 rows: their parts are fewer than blocks of 64."""
    T, terms = sum(counts), 2 * 64 * (1 if R <= 16 else 2 if R <= 32 else 4 if R <= 64 else 8)
    assert (ffi.lib().cacti_hip_adapter_bwd_workspace(T, K, N, R, n) - T * terms) // (R * (K + N) * 4) < T // 64


@GPU
@pytest.mark.parametrize("counts,ids,K,N,R,n", STEPS)
@pytest.mark.parametrize("order", ["rising", "falling", "mixed", None])
def test_gradients_in_several_steps(counts, ids, K, N, R, n, order):
    print("adapter", counts, K, N, R, order, flush=True)
    c = Case(K + N + R, counts, ids, K, N, R, n, behind=1)
    if order:
        rows_by_powers_of_two(c, order)
    check(c, max_new=max(counts))


TURNS = [([8200], [1], 264, 1032, 24), ([600, 33, 800, 667], [2, -1, 0, 1], 264, 4104, 64)]


@GPU
@pytest.mark.parametrize("counts,ids,K,N,R", TURNS)
def test_columns_in_several_turns(counts, ids, K, N, R):
    """A second launch whose waves have more than one block of 32 columns each: 8 waves to a workgroup, at most two workgroups to a compute unit."""
    T, units = sum(counts), sum(counts) // 64 + len(counts)
    assert T >= 8192 or ffi.lib().cacti_hip_adapter_fwd_workspace(T, len(ids), K, N, R, max(counts)) > 0
    assert -(-N // 32) > 8 * max(1, 512 // units)
    print("adapter", counts, K, N, R, flush=True)
    c = Case(K + N + R, counts, ids, K, N, R, 3, behind=2)
    check(c, max_new=max(counts))
    rows_by_powers_of_two(c, "mixed")
    check(c, max_new=max(counts))


@GPU
def test_infinite_values_reach_what_they_meet_and_nothing_else():
    """(Infinite there or no number: the two terms of a value may be of different signs.)"""
    from cacti_amd import ops
    c = Case(16, [5, 70, 7], [2, 0, 2], 72, 88, 16, 3)
    x, A, B, starts, ids, scale, base, dy = c.of("x A B starts ids scale base dy")
    own, every = np.array([i < 5 or i >= 75 for i in range(82)]), slice(None)

    def run():
        y, h = ops.adapter_fwd(x, A, B, starts, ids, scale, base=base)
        return dict(zip("y h dx dA dB".split(), (y, h, *ops.adapter_bwd(x, A, B, starts, ids, scale, h, dy))))

    clean = run()["h"].cpu().numpy()
    wy, ty, wh, th = c.forward(True)
    want = dict(zip("y h dx dA dB".split(), [(wy, ty), (wh, th), *c.adjoint(clean, False)]))
    for t, at, hit in ((B, (2, 5, 3), dict(y=[(own, 5)], dx=[(own, every)], dA=[(2, 3)])),
                       (A, (2, 1, 4), dict(h=[(own, 1)], y=[(own, every)], dx=[(own, 4)], dB=[(2, every, 1)])),
                       (x, (3, 9), dict(h=[(3, every)], y=[(3, every)], dA=[(2, every, 9)], dB=[(2, every)])),
                       (dy, (40, 7), dict(dx=[(40, every)], dA=[(0, every)], dB=[(0, 7)]))):
        was = t.clone()
        t[at] = float("inf")
        for k, got in run().items():
            got = got.cpu().numpy()
            where = np.zeros(got.shape, bool)
            for place in hit.get(k, []):
                where[place] = True
            assert not np.isfinite(got[where]).any(), (k, at)
            near(got[~where], want[k][0][~where], want[k][1][~where], k)
        t.copy_(was)
