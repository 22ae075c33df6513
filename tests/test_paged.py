"""The paged key / value cache: cacti_hip_paged_append and cacti_hip_paged_attention_f16 against plain forms in numpy.

Appending is compared bit for bit: the rotation's products are exact in fp32 (11 by 11 bits), their sum is rounded once and
once more into the page, and the quotient by a power of two rounds nothing (the values stay clear of fp32's subnormals).

Attention is compared with float64.  What the kernel rounds: the output, half a step of f16, 2^-11 |o|; each weight once to
f16, w (1 + d) with |d| <= 2^-11, in the numerator and, prompts in 16 bits, in the sum of the weights, so that o is off by sum p d (v - o) (to
first order), at most 2^-11 (sum p |v| + |o|); a score, a sum of up to 128 products in fp32, 128 * 2^-24 A with A = max_j alpha sum_d |q_d k_jd|, and the exponent's own
rounding and the exponential's (2^-22 (1 + A)), a relative error of each weight in numerator and denominator.  Together
  2^-10 |o| + (2^-11 + 2 (2^-17 A + 2^-22 (1 + A))) sum p |v| + 2^-25 (half a step of f16's subnormals)
Against codes of 8 bits a query is the sum of three e4m3 terms, scaled to have its largest element between 224 and 448: an element
of 11 bits takes 4 + 5 + 5 of them exactly unless its lowest fall below half a step of e4m3's subnormals, 2^-10, which is 2^-17.8
of the largest; so a score is off by at most 2^-17.8 alpha max|q| sum_d |k_d| more.
and fp32 sums over up to 10^4 keys, 2^-24 per step of a chain of at most len / 32 additions, counted as 2^-15 sum p |v|."""
import math

import numpy as np
import pytest

from cacti_amd import ffi

GPU = pytest.mark.gpu
F32 = np.float32


# ---------------------------------------------------------------- refusals, before anything is launched
APPEND = dict(T=4, B=2, H=4, Hkv=2, Dh=8, max_new=4, q=64, ldq=32, k=64, ldk=16, v=64, ldv=16, cos=64, sin=64, n_pos=64, qr=64, ldqr=32, kp=64,
              vp=64, ks=64, vs=64, bits=8, P=4, page=16, table=64, ldt=2, W=2, starts=64, lens=64, status=None, stream=None)
ATTEND = dict(T=4, B=2, H=4, Hkv=2, Dh=8, max_new=4, alpha=1.0, q=64, ldq=32, kp=64, vp=64, ks=64, vs=64, bits=8, P=4, page=16, table=64,
              ldt=2, W=2, starts=64, lens=64, out=64, ldo=32, ws=64, ws_bytes=1 << 30, status=None, stream=None)
COMMON = [(dict(T=0), "empty"), (dict(B=0), "empty"), (dict(P=0), "empty"), (dict(W=0, ldt=0), "empty"), (dict(max_new=0), "empty"),
          (dict(table=None), "null"), (dict(starts=None), "null"), (dict(lens=None), "null"), (dict(kp=None), "null"), (dict(vp=None), "null"),
          (dict(bits=4), "8 or 16"), (dict(bits=16), "scales"), (dict(ks=None), "scales"), (dict(vs=None), "scales"), (dict(H=3), "heads"),
          (dict(Dh=6), "Dh"), (dict(Dh=132), "Dh"), (dict(page=8), "pages of"), (dict(page=272), "pages of"), (dict(page=24), "pages of"),
          (dict(ldt=1), "pitch"), (dict(kp=72), "16-byte"), (dict(vp=72), "16-byte"), (dict(q=68), "8-byte"), (dict(ldq=34), "multiples of 4"),
          (dict(ldq=28), "row")]


@pytest.mark.parametrize("change,why", COMMON + [(dict(k=None), "null"), (dict(cos=None), "null"), (dict(q=None), "null"), (dict(n_pos=0), "null"),
                                                 (dict(ldk=12), "row"), (dict(ldv=18), "multiples of 4"), (dict(ldqr=28), "row"), (dict(v=66), "8-byte")])
def test_append_refuses(change, why):
    L = ffi.lib()
    assert L.cacti_hip_paged_append(*dict(APPEND, **change).values()) < 0
    assert why in L.cacti_hip_last_error().decode()


@pytest.mark.parametrize("change,why", COMMON + [(dict(q=None), "null"), (dict(out=None), "null"), (dict(ldo=30), "multiples of 4"),
                                                 (dict(ws_bytes=64), "workspace"), (dict(ws=72), "workspace"),
                                                 (dict(ws=None), "workspace"), (dict(alpha=float("nan")), "alpha"),
                                                 (dict(alpha=float("-inf")), "alpha"), (dict(), "output")])
def test_attention_refuses(change, why):
    L = ffi.lib()
    assert L.cacti_hip_paged_attention_f16(*dict(ATTEND, **change).values()) < 0
    assert why in L.cacti_hip_last_error().decode()


def test_workspace_does_not_grow_with_the_positions():
    ws = ffi.lib().cacti_hip_paged_attention_workspace
    for T, B, H, Hkv, Dh, new in [(1, 1, 32, 32, 100, 1), (48, 48, 32, 32, 100, 1), (700, 3, 16, 4, 128, 600)]:
        assert 0 < ws(T, B, H, Hkv, Dh, new) < 128 << 20 and ws(T, B, H, Hkv, Dh, new) % 16 == 0
    assert ws(0, 1, 32, 32, 100, 1) == 0 and ws(1, 1, 3, 2, 100, 1) == 0


# ---------------------------------------------------------------- plain forms
def e4m3_values():
    v = np.empty(256)
    for c in range(256):
        s, e, m = -1.0 if c & 128 else 1.0, c >> 3 & 15, c & 7
        v[c] = s * (m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
    v[[127, 255]] = np.nan
    return v


E4M3 = e4m3_values()


def encode(x):
    """float32 -> e4m3 codes: to nearest, ties to even; |x| <= 448 or not finite."""
    x = np.asarray(x, F32)
    a = np.abs(x.astype(np.float64))
    grid = E4M3[:127]
    hi = np.searchsorted(grid, np.where(np.isfinite(a), a, 0.0)).clip(1, 126)
    lo = hi - 1
    dl, dh = a - grid[lo], grid[hi] - a
    with np.errstate(invalid="ignore"):
        code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = np.where(np.isfinite(a), code, 127).astype(np.uint8)
    return code | (np.signbit(x).astype(np.uint8) << 7)


class Batch:
    """A ragged batch over a cache, in numpy, with the pages of its sequences shuffled over it."""

    def __init__(self, seed, n, lens, H, Hkv, Dh, page, bits, spare_rows=0, kv_std=1.0):
        r = self.r = np.random.default_rng(seed)
        self.n, self.lens, self.H, self.Hkv, self.Dh, self.page, self.bits = list(n), list(lens), H, Hkv, Dh, page, bits
        self.B, self.T = len(n), sum(n) + spare_rows
        self.W = max(1, max(-(-l // page) for l in lens)) + 1
        self.P = self.B * self.W + 2
        self.Dp = (Dh + 15) // 16 * 16
        self.table = r.permutation(self.P)[:self.B * self.W].reshape(self.B, self.W).astype(np.int32)
        self.starts = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        self.qkv = r.standard_normal((self.T, (H + 2 * Hkv) * Dh)).astype(np.float16)
        self.qkv[:, H * Dh:] *= np.float16(kv_std)
        shape = (self.P, Hkv, page, self.Dp)
        if bits == 8:
            self.kp, self.vp = (encode((r.standard_normal(shape) * 48).clip(-448, 448)) for _ in range(2))
            self.ks, self.vs = (np.exp2(r.integers(-7, -4, (self.P, Hkv))).astype(F32) for _ in range(2))
        else:
            self.kp, self.vp = (r.standard_normal(shape).astype(np.float16) for _ in range(2))
            self.ks = self.vs = None
        self.kp[..., Dh:] = 0
        self.vp[..., Dh:] = 0
        S = self.W * page
        ang = np.arange(S)[:, None] * 10000.0 ** (-np.arange(0, Dh, 2) / Dh)
        self.cos, self.sin = (np.concatenate([f(ang)] * 2, 1).astype(np.float16) for f in (np.cos, np.sin))
        self.alpha = 1 / math.sqrt(Dh)

    def split(self):
        H, Hkv, Dh = self.H, self.Hkv, self.Dh
        return (self.qkv[:, :H * Dh].reshape(self.T, H, Dh), self.qkv[:, H * Dh:(H + Hkv) * Dh].reshape(self.T, Hkv, Dh),
                self.qkv[:, (H + Hkv) * Dh:].reshape(self.T, Hkv, Dh))

    def rotated(self, x, p):
        c, s, h = self.cos[p].astype(F32), self.sin[p].astype(F32), self.Dh // 2
        x = x.astype(F32)
        with np.errstate(invalid="ignore"):
            return np.concatenate([x[:, :h] * c[:h] - x[:, h:] * s[:h], x[:, h:] * c[h:] + x[:, :h] * s[h:]], 1)

    def append(self):
        """Into copies of the pages; returns q rotated (rows of no sequence zero) and the cache."""
        q, k, v = self.split()
        cache = [x if x is None else x.copy() for x in (self.kp, self.vp, self.ks, self.vs)]
        qo = np.zeros(q.shape, np.float16)
        for b in range(self.B):
            first = self.lens[b] - self.n[b]
            rows = {}
            for i in range(self.n[b]):
                p, row = first + i, self.starts[b] + i
                with np.errstate(over="ignore"):
                    qo[row] = self.rotated(q[row], p).astype(np.float16)
                rows.setdefault(p // self.page, []).append((p % self.page, self.rotated(k[row], p), v[row].astype(F32)))
            for pi, new in rows.items():
                pid, slot0 = self.table[b, pi], new[0][0]
                for which in (0, 1):
                    pages, scales = cache[which], cache[2 + which]
                    x = np.stack([e[1 + which] for e in new], 1)                   # [Hkv, m, Dh]
                    if self.bits == 16:
                        pages[pid, :, slot0:slot0 + len(new), :self.Dh] = x.astype(np.float16)
                        continue
                    for h in range(self.Hkv):
                        top = np.abs(np.where(np.isfinite(x[h]), x[h], 0)).max().astype(np.float64)
                        e = -32
                        while top > 448 * 2.0 ** e and e < 15:
                            e += 1
                        to = 2.0 ** e
                        if slot0:
                            was = float(scales[pid, h])
                            if was > to:
                                to = was
                            elif was < to:
                                pages[pid, h, :slot0] = encode(E4M3[pages[pid, h, :slot0]] * (was / to))
                        scales[pid, h] = to
                        pages[pid, h, slot0:slot0 + len(new), :self.Dh] = encode(x[h] / F32(to))
        return qo, cache

    def dense(self, b, cache):
        """K, V of sequence b in float64, [len, Hkv, Dh]."""
        out = []
        for which in (0, 1):
            ids = self.table[b, :-(-self.lens[b] // self.page)]
            x = cache[which][ids]
            x = E4M3[x] * cache[2 + which][ids].astype(np.float64)[..., None, None] if self.bits == 8 else x.astype(np.float64)
            out.append(x.transpose(0, 2, 1, 3).reshape(-1, self.Hkv, self.Dp)[:self.lens[b], :, :self.Dh])
        return out

    def attend(self, q, cache):
        """(o, bound) in float64; a row's sum is over what it sees, and nothing else is looked at."""
        o = np.zeros(q.shape)
        tol = np.full(q.shape, 2.0 ** -25)
        G = self.H // self.Hkv
        for b in range(self.B):
            K, V = self.dense(b, cache)
            for i in range(self.n[b]):
                row, seen = self.starts[b] + i, self.lens[b] - self.n[b] + i + 1
                for h in range(self.H):
                    qv, k, v = q[row, h].astype(np.float64), K[:seen, h // G], V[:seen, h // G]
                    s = self.alpha * (k @ qv)
                    with np.errstate(all="ignore"):
                        w = np.exp(s - s.max())
                        w /= w.sum()
                        o[row, h] = (w[:, None] * v).sum(0)
                        A = self.alpha * np.abs(k * qv).sum(1).max()
                        near = (w[:, None] * np.abs(v)).sum(0)
                        eps = 2.0 ** -17 * A + 2.0 ** -22 * (1 + A)
                        if self.bits == 8:
                            eps += 2.0 ** -17.8 * self.alpha * np.abs(qv).max() * np.abs(k).sum(1).max()
                    tol[row, h] += 2.0 ** -10 * np.abs(o[row, h]) + (2.0 ** -11 + 2.0 ** -15 + 2 * eps) * near
        return o, tol

    # ---- on the device
    def put(self):
        import torch
        d = lambda x: None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda()
        self.d = dict(table=d(self.table), starts=d(self.starts), lens=d(np.asarray(self.lens, np.int32)), cos=d(self.cos), sin=d(self.sin))
        qkv = d(self.qkv)
        H, Hkv, Dh = self.H, self.Hkv, self.Dh
        self.d["q"], self.d["k"] = qkv[:, :H * Dh].view(-1, H, Dh), qkv[:, H * Dh:(H + Hkv) * Dh].view(-1, Hkv, Dh)
        self.d["v"] = qkv[:, (H + Hkv) * Dh:].view(-1, Hkv, Dh)
        return self.put_cache((self.kp, self.vp, self.ks, self.vs))

    def put_cache(self, cache):
        import torch
        d = [None if x is None else torch.from_numpy(x.copy()).cuda() for x in cache]
        if self.bits == 8:
            d[:2] = [x.view(torch.float8_e4m3fn) for x in d[:2]]
        return tuple(d)

    def at(self):
        return self.d["table"], self.d["starts"], self.d["lens"]


def numpy_of(t):
    import torch
    return t.view(torch.uint8).cpu().numpy() if t.dtype is torch.float8_e4m3fn else t.cpu().numpy()


def same_bits(got, want, name):
    """Bit for bit; a NaN's sign is not laid down."""
    if got.dtype == np.uint8:
        got, want = (np.where(x == 0xff, np.uint8(0x7f), x) for x in (got, want))
    got, want = (x.view({1: np.uint8, 2: np.uint16, 4: np.uint32}[x.itemsize]) for x in (got, want))
    bad = np.argwhere(got != want)
    assert len(bad) == 0, "%s: %d of %d differ, first at %s: %#x, expected %#x" % (name, len(bad), got.size, bad[0], got[tuple(bad[0])], want[tuple(bad[0])])


def check_append(B, **more):
    """Runs the kernel on the batch and compares everything; returns the cache on the device."""
    import torch
    from cacti_amd import ops
    cache = B.put()
    out = torch.zeros((B.T, B.H, B.Dh), dtype=torch.float16, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = ops.paged_append(B.d["k"], B.d["v"], cache, *B.at(), B.d["cos"], B.d["sin"], q=B.d["q"], out=out, status=status, **more)
    assert got is out and int(status) == 0
    qo, want = B.append()
    same_bits(numpy_of(got), qo, "q")
    for name, g, w in zip(("k pages", "v pages", "k scale", "v scale"), cache, want):
        if w is not None:
            same_bits(numpy_of(g), w, name)
    return cache, want


# ---------------------------------------------------------------- appending
APPENDS = [
    # n, lens, H, Hkv, Dh, page
    ([1], [1], 4, 4, 64, 16),                                # the first token of all
    ([1], [701], 32, 32, 100, 64),
    ([1, 1, 1], [16, 17, 18], 8, 2, 64, 16),                 # last slot of a page, first, second
    ([0, 3, 0, 2, 0], [5, 33, 0, 2, 64], 4, 1, 36, 16),      # sequences without new rows
    ([70], [70], 4, 4, 4, 16),                               # a whole prompt, narrow heads
    ([130, 1, 47], [131, 900, 100], 8, 8, 100, 64),          # prompts that begin inside a page
    ([300], [777], 2, 1, 128, 256),
    ([40, 9], [50, 96], 6, 2, 80, 48),                       # pages that are no power of two
]


@GPU
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("n,lens,H,Hkv,Dh,page", APPENDS)
def test_append(n, lens, H, Hkv, Dh, page, bits):
    print("paged_append", n, lens, H, Hkv, Dh, page, bits, flush=True)
    check_append(Batch(sum(lens) + Dh + bits, n, lens, H, Hkv, Dh, page, bits))
    check_append(Batch(sum(lens) + Dh + bits + 1, n, lens, H, Hkv, Dh, page, bits, spare_rows=3), max_new=max(n))


@GPU
def test_append_many_sequences():
    """More of them than lanes of a wave, with and without a bound of the new rows."""
    r = np.random.default_rng(5)
    n = [int(x) for x in r.integers(0, 5, 150)]
    lens = [int(x) + a for x, a in zip(r.integers(0, 90, 150), n)]
    for bits in (8, 16):
        check_append(Batch(bits, n, lens, 4, 2, 64, 16, bits))
        check_append(Batch(bits, n, lens, 4, 2, 64, 16, bits), max_new=4)


@GPU
@pytest.mark.parametrize("std", [2.0 ** -12, 2.0 ** -3, 30.0, 2000.0])
def test_append_scales(std):
    """Values far below and above what the pages' scales hold: older codes are carried over, or the old scale stays."""
    check_append(Batch(int(std * 4096), [2, 5, 1, 20], [40, 69, 64, 20], 2, 2, 64, 32, 8, kv_std=std))


@GPU
def test_append_values_at_the_edge():
    """Zeros alone, subnormals, the largest f16, NaN and infinities."""
    B = Batch(3, [3, 2, 2, 2, 2], [3, 40, 7, 21, 2], 2, 2, 64, 16, 8)
    kv = B.qkv[:, 2 * 64:]
    kv[0:3] = 0
    kv[3] = np.float16(6e-8)
    kv[4] = np.float16(65504)
    kv[5, ::7], kv[5, 1::9] = np.nan, np.inf
    kv[6] = -np.inf
    kv[7:9] = np.nan
    check_append(B)


@GPU
@pytest.mark.parametrize("Dh", [4, 36, 100, 128])
def test_append_rotates_queries_in_place(Dh):
    import torch
    from cacti_amd import ops
    for n, lens in (([1, 1], [9, 70]), ([90, 3], [95, 16])):
        B = Batch(18 + Dh, n, lens, 8, 2, Dh, 64, 16)
        cache = B.put()
        want = ops.paged_append(B.d["k"], B.d["v"], cache, *B.at(), B.d["cos"], B.d["sin"], q=B.d["q"]).clone()
        got = ops.paged_append(B.d["k"], B.d["v"], cache, *B.at(), B.d["cos"], B.d["sin"], q=B.d["q"], out=B.d["q"])
        assert got is B.d["q"] and torch.equal(got, want)


@GPU
def test_append_leaves_the_rest_alone():
    """Slots behind the new ones, rows behind the last sequence and their queries; appending the same rows again changes nothing."""
    import torch
    from cacti_amd import ops
    for bits in (8, 16):
        B = Batch(11, [5, 2], [37, 18], 4, 2, 100, 16, bits, spare_rows=4)
        cache, want = check_append(B)
        out = torch.full((B.T, 4, 100), 7.0, dtype=torch.float16, device="cuda")
        ops.paged_append(B.d["k"], B.d["v"], cache, *B.at(), B.d["cos"], B.d["sin"], q=B.d["q"], out=out)
        assert bool((out[7:] == 7).all()) and not bool((out[:7] == 7).all())
        for g, w in zip(cache, want):
            if w is not None:
                same_bits(numpy_of(g), w, "appended again")
        assert ops.paged_append(B.d["k"], B.d["v"], cache, *B.at(), B.d["cos"], B.d["sin"]) is None


@GPU
@pytest.mark.parametrize("what", ["len too long", "more rows than positions", "rows beyond T", "more than max_new", "falling starts", "no rotation"])
def test_append_of_numbers_that_do_not_fit(what):
    """The sequence is left out and named, the others are as ever."""
    import torch
    from cacti_amd import ops
    B = Batch(21, [2, 3, 2], [30, 20, 19], 4, 2, 64, 16, 8)
    _, want = B.append()
    cache = B.put()
    starts, lens, cos, sin, more = B.starts.copy(), list(B.lens), B.d["cos"], B.d["sin"], {}
    bad = 2
    if what == "len too long":
        lens[2] = B.W * B.page + 1
    elif what == "more rows than positions":
        lens[2] = 1
    elif what == "rows beyond T":
        starts[3] = B.T + 5
    elif what == "falling starts":
        starts[3] = 1
    elif what == "no rotation":
        cos, sin, bad, lens[2] = cos[:30], sin[:30], 2, 31
    else:
        more, bad = dict(max_new=2), 1
    d = lambda x: torch.from_numpy(np.asarray(x, np.int32)).cuda()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.paged_append(B.d["k"], B.d["v"], cache, B.d["table"], d(starts), d(lens), cos, sin, status=status, **more)
    assert int(status) == bad + 1
    for b in range(3):
        w = want if b != bad else (B.kp, B.vp, B.ks, B.vs)
        for g, x in zip(cache, w):
            same_bits(numpy_of(g)[B.table[b]], x[B.table[b]], "sequence %d" % b)


@GPU
def test_append_to_a_page_that_is_not_there():
    import torch
    from cacti_amd import ops
    for wrong in (-1, 1 << 30, None):
        B = Batch(22, [20, 3], [20, 20], 4, 2, 64, 16, 8)
        _, want = B.append()
        cache = B.put()
        bad = B.table.copy()
        bad[0, 1] = B.P if wrong is None else wrong
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        ops.paged_append(B.d["k"], B.d["v"], cache, torch.from_numpy(bad).cuda(), B.d["starts"], B.d["lens"], B.d["cos"], B.d["sin"], status=status)
        assert int(status) == 1
        left = B.table[0, 1]
        for g, w, was in zip(cache, want, (B.kp, B.vp, B.ks, B.vs)):
            w = w.copy()
            w[left] = was[left]
            same_bits(numpy_of(g), w, "pages")


# ---------------------------------------------------------------- attention
def check_attention(B, cache=None, **more):
    import torch
    from cacti_amd import ops
    host = (B.kp, B.vp, B.ks, B.vs) if cache is None else cache
    dev = B.put()
    if cache is not None:
        dev = B.put_cache(cache)
    out = torch.full((B.T, B.H, B.Dh), 7.0, dtype=torch.float16, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = ops.paged_attention(B.d["q"], dev, *B.at(), B.alpha, out=out, status=status, **more)
    assert got is out and int(status) == 0
    got = got.cpu().numpy().astype(np.float64)
    want, tol = B.attend(B.split()[0], host)
    rows = sum(B.n)
    assert (got[rows:] == 7).all()
    fine = np.isfinite(want[:rows])
    assert np.array_equal(fine, np.isfinite(got[:rows]))
    off = np.abs(got[:rows] - want[:rows])[fine] / tol[:rows][fine]
    assert off.size == 0 or off.max() <= 1, "%.2f of the bound at most, %d beyond" % (off.max(), (off > 1).sum())
    return got


ATTENDS = [
    # n, lens, H, Hkv, Dh, page
    ([1], [1], 4, 4, 64, 16),
    ([1], [33], 2, 2, 4, 16),
    ([1], [701], 32, 32, 100, 64),
    ([1], [3000], 4, 4, 128, 64),                            # parts of a sequence, put together
    ([1, 1, 1], [1, 31, 2049], 8, 2, 64, 16),
    ([0, 3, 0, 2, 0], [5, 33, 0, 2, 64], 4, 1, 36, 16),
    ([17], [17], 4, 4, 64, 16),                              # a tile and a row
    ([5, 8, 1], [500, 8, 1290], 14, 2, 100, 32),             # seven heads to a key head
    ([3, 1], [140, 9], 16, 1, 128, 16),
    ([130, 1, 47], [131, 900, 100], 4, 4, 100, 64),          # prompts
    ([90], [777], 4, 2, 80, 48),
    ([3], [260], 2, 1, 128, 256),
    ([37, 5, 64], [37, 5, 64], 4, 2, 36, 16),                # up to 128 rows of a key head
    ([37, 5, 80], [37, 5, 80], 4, 2, 36, 16),                # prompts of narrow heads, pages of 16
    ([140, 33, 32], [300, 333, 90], 2, 2, 64, 16),
    ([100, 1, 70], [310, 400, 333], 2, 1, 4, 32),
    ([200, 2], [211, 130], 3, 1, 128, 16),
    ([1, 3], [300, 90], 72, 1, 64, 16),                      # a token's query heads fill more than a tile
    ([2], [70], 130, 1, 20, 16),
]


@GPU
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("n,lens,H,Hkv,Dh,page", ATTENDS)
def test_attention(n, lens, H, Hkv, Dh, page, bits):
    print("paged_attention", n, lens, H, Hkv, Dh, page, bits, flush=True)
    check_attention(Batch(sum(lens) + Dh + bits, n, lens, H, Hkv, Dh, page, bits))
    check_attention(Batch(sum(lens) + Dh + bits + 1, n, lens, H, Hkv, Dh, page, bits, spare_rows=3), max_new=max(n))


@GPU
def test_attention_many_sequences():
    r = np.random.default_rng(6)
    n = [int(x) for x in r.integers(0, 4, 140)]
    lens = [int(x) + a for x, a in zip(r.integers(0, 90, 140), n)]
    for bits in (8, 16):
        check_attention(Batch(bits, n, lens, 4, 2, 64, 16, bits))
        check_attention(Batch(bits, n, lens, 4, 2, 64, 16, bits), max_new=3)


@GPU
def test_attention_of_scales_far_apart():
    """Values of a page that are 2^40 larger than another's, in both: no weight overflows and none of the small page is lost
    where it has the probability.  Scores stay small: the keys' scales go down as their codes go up."""
    B = Batch(31, [2], [200], 4, 4, 64, 16, 8)
    for i, p in enumerate(B.table[0]):
        B.vs[p] = 2.0 ** (-30 + 40 * (i % 2))
        B.ks[p] = 2.0 ** -9
    check_attention(B)
    for i, p in enumerate(B.table[0]):                       # all probability on the small pages
        B.vs[p] = 2.0 ** (-20 + 18 * (i % 2))
        B.kp[p] = encode(np.zeros(B.kp[p].shape)) if i % 2 else B.kp[p]
        B.ks[p] = 2.0 ** -2
    check_attention(B)


@GPU
def test_attention_of_large_scores():
    """One key has all of it: scores in the hundreds."""
    for bits in (8, 16):
        B = Batch(32, [3, 1], [300, 77], 4, 2, 64, 16, bits)
        B.qkv *= np.float16(30)
        check_attention(B)


@GPU
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("last", [40, 70])                   # 70: a prompt
def test_attention_looks_at_nothing_hidden(last, bits):
    """NaN (and infinities) behind the last position, in other sequences' and in spare pages; rows that see a NaN have it,
    rows before it do not."""
    B = Batch(33, [6, 1, last], [70, 31, last], 4, 2, 64, 16, bits)
    clean = check_attention(B)
    poison = np.uint8(0x7f) if bits == 8 else np.float16(np.nan)
    kp, vp = B.kp.copy(), B.vp.copy()
    used = set()
    for b in range(B.B):
        for p in range(B.lens[b]):
            used.add((int(B.table[b, p // 16]), p % 16))
    for pid in range(B.P):
        for s in range(16):
            if (pid, s) not in used:
                kp[pid, :, s], vp[pid, :, s] = poison, poison
    got = check_attention(B, (kp, vp, B.ks, B.vs))
    assert np.array_equal(got, clean)
    # position 67 of sequence 0 is its row 3, position 20 of sequence 2 its row 20
    for which in (kp, vp):
        for v in ([poison] if bits == 8 else [poison, np.float16(np.inf), np.float16(-np.inf)]):
            was = which.copy()
            which[B.table[0, 67 // 16], 1, 67 % 16, 5] = v
            which[B.table[2, 20 // 16], 0, 20 % 16, 7:9] = v
            if which is vp or np.isnan(v) or bits == 8:
                check_attention(B, (kp, vp, B.ks, B.vs))
            which[:] = was


@pytest.mark.parametrize("G", [1, 2, 3, 4, 7, 8, 16, 40, 130])
@pytest.mark.parametrize("page", [16, 48, 160, 256])
def test_prompts_look_up_pages_that_there_are(G, page):
    """A prompt's tiles are counted by a line that is never below their steps, so a share may begin behind the last position that its
    tile sees: the kernel's lookup of the first pages, restated, stays within the table's row there, too."""
    for n in (1, 5, 40, 89, 217, 600):
        for first in (0, 1, 63, 64, 1000):
            W = -(-(first + n) // page)
            tokens = (128 + G - 1) // G
            base, slope = (first + 63) // 64, (tokens + 63) // 64 if tokens >= 64 else 0
            for t in range(-(-n * G // 128)):
                steps = base + slope * (t + 1) if slope else base + t // (64 // tokens) + 1
                end = first + min(n * G - 1, 128 * t + 127) // G + 1
                assert 0 < end <= 64 * steps                  # the line: nothing that is seen is left out
                for k in range(steps):
                    c0, c1 = 64 * k, end
                    at = min(c0, c1 - 1)                      # (c0 itself is behind the table's row in some of these)
                    p0 = at // page
                    most = (min(c1 - p0 * page, 64 * page) - 1) // page
                    assert 0 <= p0 and most >= 0 and p0 + min(63, most) < W


@GPU
@pytest.mark.parametrize("n,lens", [([70], [75]), ([70, 2], [75, 40])])
def test_attention_of_a_prompt_that_does_not_fit(n, lens):
    """A prompt with more positions than its row of the table has: zeros, and whoever stands beside it as ever."""
    import torch
    from cacti_amd import ops
    for bits in (8, 16):
        B = Batch(43, n, lens, 4, 2, 64, 16, bits)
        want, tol = B.attend(B.split()[0], (B.kp, B.vp, B.ks, B.vs))
        cache = B.put()
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        bad = torch.tensor([B.W * B.page + 1] + lens[1:], dtype=torch.int32, device="cuda")
        out = torch.full((B.T, 4, 64), 7.0, dtype=torch.float16, device="cuda")
        ops.paged_attention(B.d["q"], cache, B.d["table"], B.d["starts"], bad, B.alpha, out=out, status=status)
        assert int(status) == 1
        out = out.cpu().numpy().astype(np.float64)
        assert (out[:70] == 0).all() and (np.abs(out[70:] - want[70:]) <= tol[70:]).all()


@GPU
def test_attention_infinite_keys_of_a_prompt():
    """A key with an infinity of a prompt: rows that see it have no number where the score is +inf, no weight where it is -inf."""
    B = Batch(35, [140], [150], 2, 2, 100, 16, 16)
    B.kp[B.table[0, 1], 0, 3, 40] = np.inf
    q = B.split()[0]
    q[:, 0, 40] = -np.abs(q[:, 0, 40]) - np.float16(1)
    check_attention(B)
    q[:, 0, 40] *= np.float16(-1)
    import torch
    from cacti_amd import ops
    out = ops.paged_attention(torch.from_numpy(q.copy()).cuda(), B.put(), *B.at(), B.alpha).cpu().numpy()
    assert np.isfinite(out[:9]).all() and np.isnan(out[9:, 0]).all() and np.isfinite(out[:, 1]).all()


@GPU
def test_attention_infinite_keys():
    """A key with an infinity takes all of a row's probability or none of it."""
    B = Batch(34, [2], [50], 2, 2, 100, 16, 16)
    B.kp[B.table[0, 1], 0, 3, 40] = np.inf
    got_rows = B.split()[0][:, 0, 40]
    B.split()[0][:, 0, 40] = np.abs(got_rows) + np.float16(1)         # score +inf: NaN, as inf - inf has it
    import torch
    from cacti_amd import ops
    out = ops.paged_attention(torch.from_numpy(B.split()[0].copy()).cuda(), B.put(), *B.at(), B.alpha).cpu().numpy()
    assert np.isnan(out[:, 0]).all() and np.isfinite(out[:, 1]).all()
    B.split()[0][:, 0, 40] *= np.float16(-1)                          # score -inf: no weight
    B.d = None
    check_attention(B)


@GPU
@pytest.mark.parametrize("what", ["len too long", "more rows than positions", "more than max_new"])
def test_attention_of_numbers_that_do_not_fit(what):
    """Zeros for that sequence's rows (as far as max_new goes), the others as ever."""
    import torch
    from cacti_amd import ops
    B = Batch(41, [2, 3, 2], [30, 20, 19], 4, 2, 64, 16, 8)
    want, tol = B.attend(B.split()[0], (B.kp, B.vp, B.ks, B.vs))
    cache = B.put()
    lens, more, bad = list(B.lens), {}, 2
    if what == "len too long":
        lens[2] = B.W * B.page + 1
    elif what == "more rows than positions":
        lens[2] = 1
    else:
        more, bad = dict(max_new=2), 1
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full((B.T, 4, 64), 7.0, dtype=torch.float16, device="cuda")
    ops.paged_attention(B.d["q"], cache, B.d["table"], B.d["starts"], torch.tensor(lens, dtype=torch.int32, device="cuda"), B.alpha, out=out,
                        status=status, **more)
    assert int(status) == bad + 1
    out = out.cpu().numpy().astype(np.float64)
    for b in range(3):
        rows = slice(B.starts[b], B.starts[b + 1])
        if b == bad:
            assert ((out[rows] == 0) | (out[rows] == 7)).all() and (out[B.starts[b]] == 0).all()
        else:
            assert (np.abs(out[rows] - want[rows]) <= tol[rows]).all()


@GPU
def test_attention_with_a_page_that_is_not_there():
    """Named; the other sequences are as ever."""
    import torch
    from cacti_amd import ops
    B = Batch(42, [2, 3], [300, 20], 4, 2, 64, 16, 8)
    want, tol = B.attend(B.split()[0], (B.kp, B.vp, B.ks, B.vs))
    cache = B.put()
    for wrong in (-7, B.P, 1 << 30):
        bad = B.table.copy()
        bad[0, 2] = wrong
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = ops.paged_attention(B.d["q"], cache, torch.from_numpy(bad).cuda(), B.d["starts"], B.d["lens"], B.alpha, status=status)
        assert int(status) == 1
        assert (np.abs(out.cpu().numpy()[2:] - want[2:]) <= tol[2:]).all()


@GPU
@pytest.mark.parametrize("bits", [8, 16])
def test_a_cache_beyond_four_gigabytes(bits):
    """Page numbers whose offsets pass 32 bits, in bytes and in elements."""
    import torch
    from cacti_amd import ops
    B = Batch(51, [3, 1], [40, 33], 2, 2, 128, 64, bits)
    B.kp, B.vp = (x[:B.P].copy() for x in (B.kp, B.vp))
    qo, small = B.append()
    size = 2 * 64 * 128
    P = (1 << 32) // size + 64                               # 2^32 elements and some
    cache = ops.paged_cache(P, 2, 64, 128, dtype=torch.float8_e4m3fn if bits == 8 else torch.float16)
    dev = B.put()
    up = P - B.P
    for big, x in zip(cache, dev):
        if x is not None:
            (big.view(torch.uint8) if bits == 8 and big.dim() == 4 else big)[up:] = x.view(torch.uint8) if bits == 8 and x.dim() == 4 else x
    B.d["table"] = B.d["table"] + up
    q = ops.paged_append(B.d["k"], B.d["v"], cache, *B.at(), B.d["cos"], B.d["sin"], q=B.d["q"])
    for big, w in zip(cache, small):
        if w is not None:
            same_bits(numpy_of(big[up:]), w, "pages")
    out = ops.paged_attention(q, cache, *B.at(), B.alpha).cpu().numpy()
    want, tol = B.attend(qo, small)
    assert (np.abs(out - want) <= tol).all()


@GPU
def test_arguments_that_do_not_go_together():
    import torch
    from cacti_amd import ops
    B = Batch(61, [2], [20], 4, 2, 64, 16, 8)
    cache = B.put()
    q, k, v, cos, sin = (B.d[x] for x in ("q", "k", "v", "cos", "sin"))
    append = lambda **c: ops.paged_append(**dict(dict(k=k, v=v, cache=cache, table=B.d["table"], starts=B.d["starts"], lens=B.d["lens"], cos=cos,
                                                      sin=sin, q=q), **c))
    attend = lambda **c: ops.paged_attention(**dict(dict(q=q, cache=cache, table=B.d["table"], starts=B.d["starts"], lens=B.d["lens"],
                                                         alpha=1.0), **c))
    for f in (lambda: append(k=k.float()), lambda: append(v=v[:1]), lambda: append(k=k.cpu()), lambda: append(k=k.transpose(0, 1)),
              lambda: append(cos=cos[:, :32]), lambda: append(sin=sin[:3]), lambda: append(starts=B.d["starts"][:1]),
              lambda: append(lens=B.d["lens"].long()), lambda: append(table=B.d["table"].long()), lambda: append(cache=cache[:2] + (None, cache[3][:1])),
              lambda: append(cache=(cache[0], cache[1][:1], cache[2], cache[3])), lambda: append(q=q[:1]), lambda: append(max_new=-1),
              lambda: append(q=None, out=q), lambda: attend(q=q[:, :, :60]), lambda: attend(out=q[:1]), lambda: attend(q=q.cpu()),
              lambda: attend(status=torch.zeros(2, dtype=torch.int32, device="cuda"))):
        with pytest.raises(AssertionError):
            f()
    with pytest.raises(ffi.CactiError):
        append(cache=cache[:2] + (None, None))
    with pytest.raises(ffi.CactiError):
        attend(q=q[:, :3].contiguous())                      # three heads over two
    # nothing to do
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert attend(q=q[:0], starts=B.d["starts"] * 0).shape == (0, 4, 64)
    assert ops.paged_attention(q, cache, B.d["table"][:0], none, none[:0], 1.0).shape == q.shape
    assert append(k=k[:0], v=v[:0], q=q[:0]).shape == (0, 4, 64)


@GPU
def test_captured_and_replayed():
    """Append and attention of single tokens in a graph, the sequences growing between its replays, against eager calls on
    another cache; other work in between."""
    import torch
    from cacti_amd import ops
    for bits in (8, 16):
        B = Batch(71, [1, 1, 1], [63, 16, 500], 4, 2, 64, 16, bits)
        caches = [B.put(), B.put_cache((B.kp, B.vp, B.ks, B.vs))]
        q, k, v = (B.d[x] for x in "qkv")
        lens = B.d["lens"]

        def step(cache, qr):
            ops.paged_append(k, v, cache, *B.at(), B.d["cos"], B.d["sin"], q=q, out=qr, max_new=1)
            return ops.paged_attention(qr, cache, *B.at(), B.alpha, max_new=1)

        qr = [torch.empty((3, 4, 64), dtype=torch.float16, device="cuda") for _ in range(2)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(caches[0], qr[0])                           # (the same rows again in the first replay: no change)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(caches[0], qr[0])
        for i in range(5):
            g.replay()
            want = step(caches[1], qr[1])
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(qr[0], qr[1])
            for a, b in zip(*caches):
                if a is not None:
                    same_bits(numpy_of(a), numpy_of(b), "cache")
            lens += 1
            for x in (q, k, v):
                x.copy_(torch.roll(x, 1, 0) * 1.25)


@GPU
def test_on_another_stream():
    import torch
    B = Batch(81, [5, 1], [500, 1290], 8, 2, 100, 32, 8)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        check_append(B)
        check_attention(B)
