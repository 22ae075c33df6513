"""Pages of a cache that are handed out, shared, copied and packed, against a walk over lists.  Whole numbers and copies: everything
has to be equal."""
import random

import numpy as np
import pytest

from cacti_amd import ffi

GPU = pytest.mark.gpu
FORK = dict(P=9, B=2, W=4, page=16, refs=64, table=0x1000, ldt=4, lens=64, parent=64, new_table=0x2000, ldn=4, new_lens=0x3000, status=None, stream=None)
FIT = dict(P=9, B=2, W=4, page=16, refs=64, table=64, ldt=4, first=64, lens=64, src=64, dst=64, slots=64, ws=64, ws_bytes=1 << 20, status=None, stream=None)
COMPACT = dict(P=9, B=2, W=4, refs=64, table=64, ldt=4, src=64, dst=64, used=64, ws=64, ws_bytes=1 << 20, stream=None)
BOOK = [(dict(P=0), "empty"), (dict(B=0), "empty"), (dict(W=0), "empty"), (dict(refs=None), "null"), (dict(table=None), "null"), (dict(ldt=3), "pitch"),
        (dict(refs=66), "misaligned"), (dict(status=66), "misaligned"), (dict(P=(1 << 28) + 1), "too many"), (dict(B=(1 << 20) + 1), "too many")]
REFUSED = [("cacti_hip_paged_fork", FORK, c) for c in BOOK + [
    (dict(page=0), "empty"), (dict(W=1 << 27, ldt=1 << 27), "too many"), (dict(lens=None), "null"), (dict(parent=None), "null"), (dict(new_table=None), "null"),
    (dict(new_lens=66), "misaligned"), (dict(ldn=3), "pitch"), (dict(new_table=0x1000), "shares"), (dict(new_table=0x1000 + 28), "shares"),
    (dict(lens=0x3004), "share memory")]] + \
          [("cacti_hip_paged_fit", FIT, c) for c in BOOK + [
              (dict(page=0), "empty"), (dict(first=None), "null"), (dict(src=None), "null"), (dict(slots=66), "misaligned"), (dict(ws=None), "null"),
              (dict(ws_bytes=32), "workspace")]] + \
          [("cacti_hip_paged_compact", COMPACT, c) for c in [x for x in BOOK if "status" not in x[0]] + [
              (dict(src=None), "null"), (dict(used=None), "null"), (dict(used=66), "misaligned"), (dict(ws_bytes=32), "workspace")]]


REFUSED += [(e, a, (dict(W=1 << 11, B=1 << 20, ldt=1 << 11, ldn=1 << 11), "too many")) for e, a in (("cacti_hip_paged_fork", FORK), ("cacti_hip_paged_fit", FIT),
                                                                                                   ("cacti_hip_paged_compact", COMPACT))]


@pytest.mark.parametrize("entry,args,change", REFUSED)
def test_refuses(entry, args, change):
    change, why = change
    L = ffi.lib()
    assert getattr(L, entry)(*dict(args, **{k: v for k, v in change.items() if k in args}).values()) < 0
    assert why in L.cacti_hip_last_error().decode()


@pytest.mark.parametrize("change,why", [(dict(P=0), "empty"), (dict(Hkv=0), "empty"), (dict(bits=4), "bits"), (dict(src=None), "null"), (dict(dst=None), "null"),
                                        (dict(slots=66), "misaligned"), (dict(Dh=5000), "too large"), (dict(Hkv=4096, page=4096, Dh=128), "too large"),
                                        (dict(k=[8]), "aligned"), (dict(k=[0]), "null"), (dict(ks=[0]), "scales")])
def test_copy_refuses(change, why):
    import ctypes
    L = ffi.lib()
    a = dict(layers=1, k=[0x1000], v=[0x2000], ks=[0x3000], vs=[0x4000], bits=8, P=4, Hkv=2, page=16, Dh=36, n=2, src=64, dst=64, slots=None, stream=None)
    a.update(change)
    for x in ("k", "v", "ks", "vs"):
        a[x] = ctypes.cast((ctypes.c_void_p * 1)(*a[x]), ctypes.c_void_p)
    assert L.cacti_hip_paged_copy(*a.values()) < 0
    assert why in L.cacti_hip_last_error().decode()


# ---------------------------------------------------------------- the walk
def fork(refs, table, lens, parent, page, W):
    """(refs, table, lens, sequences that do not fit)"""
    P, refs, new, out, bad = len(refs), list(refs), [], [], []
    for b, p in enumerate(parent):
        if p < -1 or p >= len(parent) or (p >= 0 and not 0 <= lens[p] <= W * page):
            bad.append(b)
            new.append(list(table[b])), out.append(lens[b])
            continue
        need = -(-lens[p] // page) if p >= 0 else 0
        new.append([table[p][j] if j < need else -1 for j in range(W)])
        out.append(lens[p] if p >= 0 else 0)
    for rows, d in ((table, -1), (new, 1)):
        for row in rows:
            for x in row:
                if 0 <= x < P:
                    refs[x] += d
    return refs, new, out, bad


def fit(refs, table, first, lens, page, W):
    P, B, refs, table = len(refs), len(table), list(refs), [list(r) for r in table]
    src, dst, slots, bad = [-1] * B, [-1] * B, [0] * B, []
    spans = []
    for b in range(B):
        if not (0 <= first[b] <= lens[b] <= W * page):
            bad.append(b)
            spans.append((W, 0, 0))
            continue
        need = -(-lens[b] // page)
        writes = lens[b] > first[b]
        spans.append((first[b] // page if writes else need, need, first[b] % page if writes else 0))
    loose = [(b, j) for b, (lo, _, _) in enumerate(spans) for j in range(lo, W) if 0 <= table[b][j] < P]
    for b, j in loose:
        refs[table[b][j]] -= 1
    kept, asked = {}, []
    for b, (lo, need, part) in enumerate(spans):
        for j in range(lo, need):
            x = table[b][j]
            if 0 <= x < P and refs[x] == 0 and x not in kept:
                kept[x] = (b, j)
            else:
                asked.append((b, j, x if part and j == lo and 0 <= x < P else -1, part))
    for x in kept:
        refs[x] = 1
    free = iter([x for x in range(P) if refs[x] == 0])
    for b, (lo, need, _) in enumerate(spans):
        for j in range(lo, W):
            if j >= need or (b, j) not in kept.values():
                table[b][j] = -1
    for b, j, x, part in asked:
        y = next(free, None)
        if y is None:
            bad.append(b)
            continue
        refs[y], table[b][j] = 1, y
        if x >= 0:
            src[b], dst[b], slots[b] = x, y, part
    return refs, table, src, dst, slots, bad


def compact(refs, table):
    P, refs = len(refs), list(refs)
    used = sum(r > 0 for r in refs)
    src, dst = [x for x in range(used, P) if refs[x] > 0], [x for x in range(used) if refs[x] == 0]
    to = dict(zip(src, dst))
    for s, d in to.items():
        refs[d], refs[s] = refs[s], 0
    pad = lambda v: v + [-1] * (P // 2 - len(v))
    return refs, [[to.get(x, x) for x in row] for row in table], pad(src), pad(dst), [used]


class Book:
    """Sequences over a pool, with lists beside the tensors."""

    def __init__(self, seed, B, W, page, P, pitch=None):
        import torch
        self.r, self.B, self.W, self.page, self.P = random.Random(seed), B, W, page, P
        self.refs, self.table, self.lens = [0] * P, [[-1] * W for _ in range(B)], [0] * B
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.pitch = pitch or W
        self.wide = torch.full((B, self.pitch), -7, dtype=torch.int32, device="cuda")
        self.d_table = self.wide[:, :W]
        self.d_table.fill_(-1)
        self.d_refs = ints(self.refs)

    def same(self, *pairs):
        for got, want in ((self.d_refs, self.refs), (self.d_table, self.table)) + pairs:
            assert got.cpu().tolist() == want
        assert bool((self.wide[:, self.W:] == -7).all())

    def named(self, bad):
        assert int(self.status) == (1 + max(bad) if bad else 0)
        self.status.zero_()

    def fork(self, parent):
        from cacti_amd import ops
        t, l = ops.paged_fork(self.d_refs, self.d_table, ints(self.lens), ints(parent), self.page, status=self.status)
        self.refs, self.table, self.lens, bad = fork(self.refs, self.table, self.lens, parent, self.page, self.W)
        self.d_table.copy_(t)
        self.same((l, self.lens))
        self.named(bad)

    def fit(self, first, lens):
        from cacti_amd import ops
        out = ops.paged_fit(self.d_refs, self.d_table, ints(first), ints(lens), self.page, status=self.status)
        self.refs, self.table, *want, bad = fit(self.refs, self.table, first, lens, self.page, self.W)
        self.same(*zip(out, want))
        self.named(bad)
        self.lens = list(lens)
        return out

    def compact(self):
        from cacti_amd import ops
        out = ops.paged_compact(self.d_refs, self.d_table)
        self.refs, self.table, *want = compact(self.refs, self.table)
        self.same(*zip(out, want))
        return out


def ints(x):
    import torch
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@GPU
@pytest.mark.parametrize("B,W,page,P,pitch", [(1, 1, 16, 1, None), (3, 4, 16, 7, 9), (8, 5, 16, 30, None), (40, 9, 32, 300, 16), (130, 70, 16, 5000, None),
                                              (1100, 3, 16, 4100, None), (5, 200, 16, 9000, 203)])
def test_a_batch_that_grows_forks_and_shrinks(B, W, page, P, pitch):
    """Steps as a search makes them, and some that it should not: too few pages, lengths and parents that cannot be."""
    print("pages", B, W, page, P, flush=True)
    k = Book(B + P, B, W, page, P, pitch)
    r = k.r
    most = W * page
    for step in range(14):
        first = [min(l, most) if 0 <= l else 0 for l in k.lens]
        kind = r.choice(["grow", "prompt", "back", "fork", "free", "compact", "odd"])
        if step == 0:
            kind = "prompt"
        if kind == "grow":
            k.fit(first, [min(most, l + r.randint(0, 5)) for l in first])
        elif kind == "prompt":
            k.fit(first, [min(most, l + r.choice([0, 0, r.randint(1, most)])) if P > 100 else min(most, r.randint(l, most)) for l in first])
        elif kind == "back":                   # drafted tokens that are not kept, then others
            back = [r.randint(max(0, l - 2 * page), l) for l in first]
            k.fit(back, [min(most, l + r.randint(0, 3)) for l in back])
        elif kind == "fork":
            k.fork([r.choice([b, b, r.randrange(B), r.randrange(B), -1]) for b in range(B)])
        elif kind == "free":
            gone = [l if r.random() < 0.6 else 0 for l in first]
            k.fit(gone, gone)
        elif kind == "compact":
            k.compact()
        else:
            bad = list(first)
            for b in range(0, B, 3):
                bad[b] = r.choice([-1, most + 1, 2 ** 31 - 1, -2 ** 31])
            k.fit(first, bad)
            k.lens = [x if 0 <= x <= most else y for x, y in zip(bad, first)]
            k.fork([r.choice([b, -2, B, 2 ** 31 - 1, r.randrange(B)]) for b in range(B)])
    held = [0] * P
    for row in k.table:
        for x in row:
            if x >= 0:
                held[x] += 1
    assert held == k.refs


@GPU
def test_pages_that_others_hold():
    """Whoever else holds a page (a prompt that is kept for later) is counted in refs, and nobody writes on it."""
    k = Book(1, 3, 4, 16, 12)
    k.fit([0, 0, 0], [40, 0, 0])
    for x in k.table[0]:
        if x >= 0:
            k.refs[x] += 1
    k.d_refs.copy_(ints(k.refs))
    src, dst, slots = k.fit([40, 0, 0], [41, 0, 0])
    assert src.tolist() == [2, -1, -1] and dst.tolist() == [3, -1, -1] and slots.tolist() == [8, 0, 0]
    k.fork([0, 0, 0])
    src, dst, slots = k.fit([41, 41, 41], [42, 41, 45])                       # the second does not write: nobody has the page alone
    assert src.tolist() == [3, -1, 3] and slots.tolist() == [9, 0, 9]
    k.fork([0, -1, 0])
    src, dst, slots = k.fit([42, 0, 42], [43, 0, 43])                         # all who hold it write: the first keeps it
    assert src.tolist()[0] == -1 and src.tolist()[2] >= 0
    k.fit([0, 0, 0], [0, 0, 0])
    assert sum(k.refs) == 3


@GPU
def test_more_sequences_than_a_workgroup_remembers():
    k = Book(5, 2300, 3, 16, 6000)
    r = k.r
    k.fit([0] * 2300, [r.randrange(49) for _ in range(2300)])
    k.fork([r.choice([b, r.randrange(2300)]) for b in range(2300)])
    k.fit(k.lens, [min(48, l + r.randrange(3)) for l in k.lens])
    back = [r.randrange(l + 1) for l in k.lens]
    k.fit(back, [r.choice([l, min(48, l + 7), 49]) for l in back])
    k.lens = [min(l, 48) for l in k.lens]
    k.compact()


@GPU
@pytest.mark.parametrize("P,share", [(1, 0.0), (2, 1.0), (1023, 0.5), (1025, 0.97), (16384, 0.999), (16385, 0.5), (40001, 0.9995), (70000, 0.02), (33000, 1.0)])
def test_pools_of_many_pages_with_gaps(P, share):
    """Pages that others hold, at random: the free ones among them are few, or far up, or more than one look finds."""
    k = Book(P, 40, 9, 16, P)
    k.refs = [int(k.r.random() < share) * k.r.choice([1, 3]) for _ in range(P)]
    if share > 0.9:
        k.refs[P // 2:] = [1] * (P - P // 2 - 1) + [0]
    k.d_refs.copy_(ints(k.refs))
    for lens in ([k.r.choice([0, 1, 16, 17, 144]) for _ in range(40)], [k.r.randrange(145) for _ in range(40)]):
        k.fit([min(a, b) for a, b in zip(k.lens, lens)], lens)
    k.compact()
    k.fit([0] * 40, [0] * 40)
    k.compact()


@GPU
def test_numbers_of_a_table_that_are_no_pages():
    k = Book(2, 2, 4, 16, 10)
    k.fit([0, 0], [40, 20])
    k.table[0] = [0, 10, 2, 2 ** 31 - 1]
    k.refs[1] = 0
    k.d_table.copy_(ints(k.table)), k.d_refs.copy_(ints(k.refs))
    k.fork([0, 0])
    k.fit([33, 33], [34, 64])


@GPU
@pytest.mark.parametrize("bits,Dh", [(8, 36), (16, 100), (8, 128)])
@pytest.mark.parametrize("layers,with_slots", [(1, True), (3, False), (37, True)])
def test_copy(bits, Dh, layers, with_slots):
    import torch
    from cacti_amd import ops
    P, H, page = 9, 3, 16
    Dp = (Dh + 15) // 16 * 16
    g = torch.Generator().manual_seed(bits + Dh)
    caches, want = [], []
    src, dst = [4, -1, 7, 2, 3, 0, 9, 1], [0, 5, 8, 2, -1, 6, 1, 2 ** 31 - 1]
    slots = [16, 3, 1, 5, 4, 0, 8, 8] if with_slots else None
    for _ in range(layers):
        kv = [torch.randint(0, 256 if bits == 8 else 65536, (P, H, page, Dp), generator=g).to(torch.uint8 if bits == 8 else torch.int32).to(
            torch.uint8 if bits == 8 else torch.int16) for _ in range(2)]
        sc = [torch.rand((P, H), generator=g) for _ in range(2)]
        new_kv, new_sc = [x.clone() for x in kv], [x.clone() for x in sc]
        for s, d, m in zip(src, dst, slots or [page] * 8):
            if 0 <= s < P and 0 <= d < P:
                for a, b in zip(new_kv, kv):
                    a[d, :, :m] = b[s, :, :m]
                for a, b in zip(new_sc, sc):
                    if m:
                        a[d] = b[s]
        t = torch.float8_e4m3fn if bits == 8 else torch.float16
        caches.append(tuple(x.cuda().view(t) for x in kv) + (tuple(x.cuda() for x in sc) if bits == 8 else (None, None)))
        want.append(new_kv + (new_sc if bits == 8 else []))
    ops.paged_copy(caches, ints(src), ints(dst), None if slots is None else ints(slots))
    for c, w in zip(caches, want):
        for got, x in zip([y for y in c if y is not None], w):
            got = got.view(torch.uint8 if bits == 8 else torch.int16) if got.dtype is not torch.float32 else got
            # (page 0 is copied to and from: what page 6 gets of it is either, all else is as it should be)
            rest = torch.arange(P) != 6
            assert torch.equal(got.cpu()[rest], x[rest])


@GPU
def test_arguments_that_do_not_go_together():
    import torch
    from cacti_amd import ops
    refs, table, lens = ints([1, 0, 1, 0]), ints([[0, 2], [-1, -1]]), ints([20, 0])
    caches = [ops.paged_cache(4, 2, 16, 36)]
    for bad in ((refs.long(), table, lens, lens, 16), (refs, table.long(), lens, lens, 16), (refs, table, lens[:1], lens, 16), (refs, table, lens, lens[:1], 16),
                (refs, table.t(), lens, lens, 16), (refs, table, None, lens, 16), (refs, table.cpu(), lens, lens, 16)):
        for call in (ops.paged_fork, ops.paged_fit):
            with pytest.raises(AssertionError):
                call(*bad)
    for call in (ops.paged_fork, ops.paged_fit):
        with pytest.raises(ffi.CactiError):
            call(refs, table, lens, lens, 0)
    with pytest.raises(ffi.CactiError):
        ops.paged_fork(refs, table, lens, ints([0, 1]), 16, out=(table, ints([0, 0])))
    with pytest.raises(AssertionError):
        ops.paged_fork(refs, table, lens, ints([0, 1]), 16, out=(table[:1], ints([0, 0])))
    for bad in ((caches[0], refs, refs), (caches, refs.long(), refs), (caches, refs, refs[:2]), (caches, refs, refs, refs[:2]), (caches, refs, None),
                (caches + [ops.paged_cache(5, 2, 16, 36)], refs, refs), (caches + [ops.paged_cache(4, 2, 16, 36, dtype=torch.float16)], refs, refs),
                ([caches[0][:2] + (None, None)], refs, refs)):
        with pytest.raises((AssertionError, TypeError)):
            ops.paged_copy(*bad)
    ops.paged_copy([], refs, refs)
    ops.paged_copy(caches, refs[:0], refs[:0])
    none = [x.shape for x in ops.paged_fit(refs, table[:0], lens[:0], lens[:0], 16)]
    assert none == [(0,), (0,), (0,)]


@GPU
def test_captured_and_replayed():
    """A search step that is captured once: the tables that it writes to are those that the next replay begins from."""
    import torch
    from cacti_amd import ops
    B, W, page, P, L = 6, 4, 16, 40, 2
    k = Book(3, B, W, page, P)
    k.fit([0] * B, [20, 33, 7, 16, 50, 1])
    caches = [ops.paged_cache(P, 2, page, 36, dtype=torch.float16) for _ in range(L)]
    for c in caches:
        for x in c[:2]:
            x.normal_()
    lens, parent = ints(k.lens), ints([1, 1, 0, 4, 4, 4])
    mirror = [[x.clone() for x in c[:2]] for c in caches]

    def step():
        t, l = ops.paged_fork(k.d_refs, k.d_table, lens, parent, page)
        k.d_table.copy_(t)
        src, dst, slots = ops.paged_fit(k.d_refs, k.d_table, l, l + 2, page)
        ops.paged_copy(caches, src, dst, slots)
        torch.add(l, 2, out=lens)
        return src, dst, slots

    state = [k.d_refs, k.d_table, lens] + [x for c in caches for x in c[:2]]
    saved = [x.clone() for x in state]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(state, saved):
        a.copy_(b)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for parents in ([1, 1, 0, 4, 4, 4], [0, 0, 0, 3, 3, -1], [5, 4, 3, 2, 1, 0], [2, 2, 2, 2, 2, 2]):
        parent.copy_(ints(parents))
        g.replay()
        torch.cuda.synchronize()
        refs, table, ln, bad = fork(k.refs, k.table, k.lens, parents, page, W)
        k.refs, k.table, *want, bad2 = fit(refs, table, ln, [x + 2 for x in ln], page, W)
        k.lens = [x + 2 for x in ln]
        assert not bad and not bad2
        k.same((lens, k.lens), *zip(out, want))
        for c, m in zip(caches, mirror):
            for got, x in zip(c[:2], m):
                for s, d, n in zip(*want):
                    if s >= 0:
                        x[d, :, :n] = x[s, :, :n]
                assert torch.equal(got, x)


# ---------------------------------------------------------------- pages that run out
def page_of(x, P):
    """The page that an entry holds, or what is none as it is: -2 - page is one that the sequence may not write on before there is a copy."""
    return -2 - x if x < -1 and -2 - x < P else x


def fit_that_keeps(refs, table, first, lens, page, W):
    """The walk above.  A sequence that there is no page for keeps the one that it was to copy, and nobody writes on that."""
    P = len(refs)
    own = [[page_of(x, P) for x in row] for row in table]
    refs, rows, src, dst, slots, bad = fit(refs, own, first, lens, page, W)
    short, spans, bad = set(), [], set(bad)
    for b in range(len(table)):
        ok = 0 <= first[b] <= lens[b] <= W * page
        need = -(-lens[b] // page)
        spans.append((first[b] // page if first[b] < lens[b] else need, need) if ok else (W, 0))
        rows[b][:spans[b][0]] = table[b][:spans[b][0]]
    for b, (lo, need) in enumerate(spans):
        if lo < need and first[b] % page and 0 <= own[b][lo] < P and rows[b][lo] == -1:
            short.add(own[b][lo])
            refs[own[b][lo]] += 1
            rows[b][lo] = -2 - own[b][lo]
    for b, (lo, need) in enumerate(spans):
        for j in range(lo, need):
            if rows[b][j] == own[b][j] and rows[b][j] in short:
                bad.add(b)
                if j == lo and first[b] % page:
                    rows[b][j] = -2 - own[b][j]
                else:
                    rows[b][j] = -1
                    refs[own[b][j]] -= 1
    return refs, rows, src, dst, slots, bad


class Short(Book):
    """.. with what each position holds: a number of its own, written by the sequence that it is appended to."""

    def __init__(self, *args):
        super().__init__(*args)
        self.slots = [[None] * self.page for _ in range(self.P)]
        self.texts, self.next = [[] for _ in range(self.B)], 0

    def at(self, b, p):
        return page_of(self.table[b][p // self.page], self.P), p % self.page

    def grow(self, lens, back=None):
        """To these lengths, from those now or from `back` on; the sequences that were left out."""
        from cacti_amd import ops
        first = [min(a, b) for a, b in zip(back or self.lens, lens)]
        out = [x.cpu().tolist() for x in ops.paged_fit(self.d_refs, self.d_table, ints(first), ints(lens), self.page, status=self.status)]
        self.refs, self.table, *want, bad = fit_that_keeps(self.refs, self.table, first, lens, self.page, self.W)
        self.same()
        assert out == want
        self.named(bad)
        was = [list(x) for x in self.slots]
        for s, d, n in zip(*out):
            if s >= 0:
                self.slots[d][:n] = was[s][:n]
        for b in range(self.B):
            self.lens[b] = first[b] if b in bad else lens[b]
            del self.texts[b][first[b]:]
            for p in range(first[b], self.lens[b]):
                self.texts[b].append(self.next)
                x, slot = self.at(b, p)
                assert x == self.table[b][p // self.page]
                self.slots[x][slot] = self.next
                self.next += 1
        self.right()
        return sorted(bad)

    def right(self):
        for b in range(self.B):
            assert [self.slots[x][i] for x, i in (self.at(b, p) for p in range(self.lens[b]))] == self.texts[b]
        held = [0] * self.P
        for row in self.table:
            for x in row:
                if page_of(x, self.P) >= 0:
                    held[page_of(x, self.P)] += 1
        assert held == self.refs

    def go_on(self, parent):
        self.table = [[page_of(x, self.P) for x in row] for row in self.table]
        self.fork(parent)
        self.texts = [list(self.texts[p]) if p >= 0 else [] for p in parent]
        self.right()

    def pack(self):
        from cacti_amd import ops
        src, dst, used = [x.cpu().tolist() for x in ops.paged_compact(self.d_refs, self.d_table)]
        marked = [[x < -1 for x in row] for row in self.table]
        self.refs, table, *want = compact(self.refs, [[page_of(x, self.P) for x in row] for row in self.table])
        self.table = [[-2 - x if m else x for x, m in zip(*rows)] for rows in zip(table, marked)]
        self.same()
        assert [src, dst, used] == want
        for s, d in zip(src, dst):
            if s >= 0:
                self.slots[d] = list(self.slots[s])
        self.right()


@GPU
def test_a_page_that_there_was_no_copy_for_stays_the_sequences():
    k = Short(1, 3, 3, 16, 3)
    assert k.grow([20, 0, 0]) == []
    k.go_on([0, 0, 0])
    # all three write on page 1: the second gets the last page there is, the third none, and so the first, who would keep it, does not write on it
    assert k.grow([21, 21, 21]) == [0, 2]
    assert k.table == [[0, -3, -1], [0, 2, -1], [0, -3, -1]] and k.refs == [3, 2, 1]
    assert k.grow([21, 21, 21]) == [0, 2] and k.table[2] == [0, -3, -1]
    assert k.grow([20, 0, 21]) == [] and k.table == [[0, -3, -1], [-1] * 3, [0, 2, -1]]
    assert k.grow([21, 0, 22]) == [] and k.table == [[0, 1, -1], [-1] * 3, [0, 2, -1]]
    # .. of others who hold it and do not write
    k = Short(2, 2, 2, 16, 2)
    k.grow([24, 0])
    k.go_on([0, 0])
    assert k.grow([24, 25]) == [1] and k.table == [[0, 1], [0, -3]] and k.refs == [2, 2]
    # .. of one who goes back and would write over all of it
    k = Short(3, 2, 3, 16, 2)
    k.grow([24, 0])
    k.go_on([0, 0])
    assert k.grow([17, 25], back=[16, 24]) == [0, 1] and k.table == [[0, -1, -1], [0, -3, -1]] and k.refs == [2, 1]
    assert k.grow([0, 25]) == [] and k.table[1] == [0, 1, -1]
    # a sequence that ends, forks and packs with such an entry
    k = Short(4, 3, 2, 16, 3)
    k.grow([24, 0, 0])
    k.go_on([0, 0, -1])
    assert k.grow([24, 24, 16]) == [] and k.grow([25, 25, 17]) == [0, 1, 2]
    k.grow([24, 24, 0])
    k.go_on([1, 1, 1])
    assert k.grow([25, 24, 24]) == [] and k.grow([25, 25, 25]) == [1, 2]
    assert k.grow([0, 24, 24]) == []
    k.pack()
    assert min(k.table[1]) < -1
    assert k.grow([0, 0, 25]) == [] and k.refs == [1, 1, 0]


@GPU
@pytest.mark.parametrize("seed,B,W,page,P", [(1, 5, 4, 16, 6), (2, 12, 5, 16, 14), (3, 40, 6, 32, 45), (4, 3, 2, 16, 3), (5, 200, 3, 16, 180)])
def test_answers_from_a_pool_that_is_too_small(seed, B, W, page, P):
    """Sequences that grow, fork and end while pages run out again and again: what each has written is there, and who was left out goes on
    when there are pages."""
    print("pages", seed, B, W, page, P, flush=True)
    k, out, copied = Short(seed, B, W, page, P), 0, 0
    r, most = k.r, W * page
    for step in range(25):
        alive = [b for b in range(B) if k.lens[b]]
        kind = r.choice(["grow", "fork", "fork", "free", "back", "pack"]) if alive else "prompts"
        if kind == "prompts":
            k.grow([r.randint(1, 2 * page) if b % 3 == 0 else 0 for b in range(B)])
        elif kind == "fork":
            k.go_on([b if r.random() < 0.4 else r.choice(alive) for b in range(B)])
        elif kind == "free":
            k.grow([l if r.random() < 0.7 else 0 for l in k.lens])
        elif kind == "back":
            back = [r.randint(max(0, l - 5), l) for l in k.lens]
            k.grow([min(most, l + r.randint(0, 4)) for l in back], back)
        elif kind == "pack":
            k.pack()
        parts = [page_of(k.table[b][l // page], P) for b, l in enumerate(k.lens) if l % page]
        bad = k.grow([min(most, l + r.choice([0, 1, 1, 3])) if l else 0 for l in k.lens])
        out += len(bad)
        copied += len(parts) - len(set(parts))
    assert out > 0 and copied > 0
    while True:                                # the others end, one by one, until everybody goes on
        bad = k.grow([min(most, l + 1) if l else 0 for l in k.lens])
        if not bad:
            break
        alive = [b for b in range(B) if k.lens[b] and b not in bad] or bad[1:]
        k.grow([0 if b == alive[0] else l for b, l in enumerate(k.lens)])


@pytest.mark.parametrize("change", [dict(parent=0x3000), dict(parent=0x2004), dict(lens=0x201c), dict(refs=0x2000 - 32), dict(refs=0x3004), dict(new_lens=0x1000),
                                    dict(new_lens=0x2000 - 4), dict(new_lens=0x1018)])
def test_fork_refuses_results_over_operands(change):
    test_refuses("cacti_hip_paged_fork", FORK, (change, "another operand"))


@GPU
def test_more_sequences_than_a_workgroup_remembers_and_too_few_pages():
    k = Short(9, 2100, 2, 16, 1000)
    k.grow([20 if b % 100 == 0 else 0 for b in range(2100)])
    k.go_on([b // 100 * 100 for b in range(2100)])
    bad = k.grow([21] * 2100)
    assert len(bad) > 1000 and bad[-1] == 2099
    k.grow([0 if b in bad[::3] else l for b, l in enumerate(k.lens)])
    assert k.grow([l and 21 for l in k.lens])
    k.grow([l if b % 2 else 0 for b, l in enumerate(k.lens)])
    assert k.grow([l and 21 for l in k.lens]) == []
