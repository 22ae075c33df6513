"""What the paged calls promise of batches whose numbers do not fit together, of operands that share memory and of sizes at the ends
of their ranges.  The plain forms and bounds are those of test_paged.py."""
import os
import subprocess

import numpy as np
import pytest

from cacti_amd import ffi
from test_paged import APPEND, ATTEND, ATTENDS, Batch, E4M3, check_append, check_attention, numpy_of, same_bits

GPU = pytest.mark.gpu
CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cacti_amd", "csrc")


# ---------------------------------------------------------------- numbers that do not fit together
MISFITS = ["len too long", "more rows than positions", "rows beyond T", "all rows beyond T", "rows before 0", "falling starts",
           "more than max_new"]
# n, H, Hkv, max_new: few rows; a prompt by itself; prompts and a token beside them; query heads that fill more than a tile
BATCHES = [([2, 3, 2], 4, 2, None), ([300], 4, 2, None), ([140, 1, 90], 4, 2, None), ([3, 2], 72, 1, None)]


def misfit(B, what, max_new):
    """(starts, lens, max_new, the bad sequence) of batch B where one sequence's numbers do not fit."""
    starts, lens, bad = B.starts.astype(np.int64), np.asarray(B.lens, np.int64), B.B - 1
    if what == "len too long":
        lens[bad] = B.W * B.page + 1
    elif what == "more rows than positions":
        lens[bad] = B.n[bad] - 1
    elif what == "rows beyond T":
        starts[-1] = B.T + 5
    elif what == "all rows beyond T":
        starts[-2:] = B.T + 5, B.T + 9
        if B.B > 1:
            starts[-2] = B.T                                  # (the sequence before it has all rows from its first on)
            lens[-2] = max(lens[-2], starts[-2] - starts[-3])
    elif what == "rows before 0":
        starts[0], bad = -2, 0
    elif what == "falling starts":
        starts[-1] = starts[-2] - 1
    else:
        bad = int(np.argmax(B.n))
        max_new = max(1, B.n[bad] - 1) if B.n[bad] < 100 else 70
        lens[bad] = max(lens[bad], B.n[bad])
    return starts, lens, max_new, bad


@GPU
@pytest.mark.parametrize("what", MISFITS)
@pytest.mark.parametrize("n,H,Hkv,max_new", BATCHES)
def test_attention_names_and_clears_what_does_not_fit(n, H, Hkv, max_new, what):
    """status is 1 + b, every row of sequence b that there is is zeros, rows of no sequence stay, the others are as ever."""
    import torch
    from cacti_amd import ops
    if what == "more than max_new" and max(n) > 100 and len(n) > 1:
        n = [300, 1, 60]
    for bits in (8, 16):
        print("paged_attention", n, H, Hkv, what, bits, flush=True)
        B = Batch(len(n) + sum(n) + bits, n, [x + 20 for x in n], H, Hkv, 64, 16, bits, spare_rows=2)
        starts, lens, mn, bad = misfit(B, what, max_new)
        B.n = [int(starts[b + 1] - starts[b]) if b != bad else 0 for b in range(B.B)]
        B.starts, B.lens = starts.astype(np.int32), [int(x) for x in lens]
        want, tol = np.full((B.T, H, 64), 7.0), np.zeros((B.T, H, 64))
        good = [b for b in range(B.B) if b != bad]
        o, t = B.attend(B.split()[0], (B.kp, B.vp, B.ks, B.vs))
        for b in good:
            rows = slice(starts[b], starts[b + 1])
            want[rows], tol[rows] = o[rows], t[rows]
        want[max(starts[bad], 0):max(min(starts[bad + 1], B.T), 0)] = 0
        cache = B.put()
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = torch.full((B.T, H, 64), 7.0, dtype=torch.float16, device="cuda")
        ops.paged_attention(B.d["q"], cache, *B.at(), B.alpha, max_new=mn, out=out, status=status)
        assert int(status) == bad + 1
        off = np.abs(out.cpu().numpy().astype(np.float64) - want) > tol
        assert not off.any(), "rows %s" % np.unique(np.argwhere(off)[:, 0])


@GPU
@pytest.mark.parametrize("n,H,Hkv,max_new", BATCHES)
@pytest.mark.parametrize("length", [-2 ** 31, -2 ** 31 + 1, -1, 2 ** 31 - 1])
def test_lengths_at_the_ends_of_32_bits(n, H, Hkv, max_new, length):
    """A length from which the rows cannot be taken off within 32 bits is one that does not fit like any other."""
    import torch
    from cacti_amd import ops
    for bits in (8, 16):
        print("paged", n, H, Hkv, length, bits, flush=True)
        B = Batch(7 + bits, n, [x + 20 for x in n], H, Hkv, 64, 16, bits)
        was, bad = B.put(), B.B - 1
        cache = B.put()
        lens = torch.tensor(B.lens[:-1] + [length], dtype=torch.int32, device="cuda")
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        ops.paged_append(B.d["k"], B.d["v"], cache, B.d["table"], B.d["starts"], lens, B.d["cos"], B.d["sin"], status=status, max_new=max_new)
        assert int(status) == bad + 1
        for g, w in zip(cache, was):
            if w is not None:
                same_bits(numpy_of(g)[B.table[bad]], numpy_of(w)[B.table[bad]], "pages")
        status.zero_()
        out = ops.paged_attention(B.d["q"], cache, B.d["table"], B.d["starts"], lens, B.alpha, status=status, max_new=max_new)
        assert int(status) == bad + 1 and not out[B.starts[bad]:].any()

@GPU
@pytest.mark.parametrize("starts", [[0, 100, 68, 120], [0, 100, 70, 90], [0, 16, 0, 90]])
def test_append_names_falling_starts(starts):
    """Wherever the numbers of the pages' units put the sequence that they fall behind."""
    import torch
    from cacti_amd import ops
    for bits in (8, 16):
        B = Batch(17, [100, 0, 20], [110, 5, 100], 4, 2, 64, 16, bits)
        cache, was = B.put(), B.put()
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        d = torch.tensor(starts, dtype=torch.int32, device="cuda")
        ops.paged_append(B.d["k"], B.d["v"], cache, B.d["table"], d, B.d["lens"], B.d["cos"], B.d["sin"], status=status)
        assert int(status) == 2
        for g, w in zip(cache, was):
            if w is not None:
                same_bits(numpy_of(g)[B.table[1]], numpy_of(w)[B.table[1]], "pages")


# ---------------------------------------------------------------- sizes at the ends of their ranges
@pytest.mark.parametrize("page", [16, 48, 256])
def test_no_more_positions_than_are_counted_in_32_bits(page):
    """Positions and steps of up to 64 of them, with what a tile of rows has too many, are formed in 32 bits: 2^30 at most."""
    L = ffi.lib()
    W = (1 << 31) // page - 1
    for W, refused in ((W, True), ((1 << 30) // page + 1, True), ((1 << 30) // page, False)):
        for f, args in ((L.cacti_hip_paged_append, APPEND), (L.cacti_hip_paged_attention_f16, ATTEND)):
            # (a wrong pitch of the rotation's and of the output's rows ends the calls that are not refused for their table)
            assert f(*dict(args, page=page, W=W, ldt=W, **({"ldk": 12} if args is APPEND else {"ldo": 30})).values()) < 0
            assert ("too many rows, sequences or pages" in L.cacti_hip_last_error().decode()) == refused


@pytest.mark.parametrize("T,B,H,Hkv,max_new,W,refused", [(8192, 2048, 64, 8, 8192, 512, False), (8192, 2048, 64, 8, 8, 512, False),
                                                         (65536, 1024, 64, 64, 65536, 4096, False), (65536, 1024, 64, 64, 65536, 32768, True),
                                                         (1, 1, 8, 8, 1, 1 << 22, False), (1 << 18, 64, 64, 8, 4096, 64, True)])
def test_work_that_is_counted_in_32_bits(T, B, H, Hkv, max_new, W, refused):
    """Tiles of a batch are no more than its rows make, however many one sequence may have.  (The output in the queries' place ends the
    calls that are not refused for their work.)"""
    L = ffi.lib()
    args = dict(ATTEND, T=T, B=B, H=H, Hkv=Hkv, max_new=max_new, W=W, ldt=W, ldq=H * 8, ldo=H * 8, ws_bytes=1 << 40)
    assert L.cacti_hip_paged_attention_f16(*args.values()) < 0
    assert ("too many rows and positions" if refused else "output") in L.cacti_hip_last_error().decode()


@GPU
@pytest.mark.parametrize("T,W", [(65536, 256), (128, 4060)])
def test_rows_of_many_sequences_are_no_endless_work(T, W):
    """Starts that fall again and again give every second sequence all rows, which is more work than 32 bits count: nothing is done."""
    import torch
    from cacti_amd import ops
    B, H, page = 1024, 64, 256
    print("paged_attention", T, W, flush=True)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    cache = ops.paged_cache(1, H, page, 4, dtype=torch.float16)
    q = torch.zeros((T, H, 4), dtype=torch.float16, device="cuda")
    status = i32([0])
    ops.paged_attention(q, cache, torch.zeros((B, W), dtype=torch.int32, device="cuda"), i32([0, T] * (B // 2) + [0]), i32([W * page] * B), 0.5,
                        status=status)
    assert int(status) == B


@GPU
@pytest.mark.parametrize("H", [64, 160])
def test_many_sequences_of_many_heads_to_a_key_head(H):
    """A token's query heads fill more than a tile of the few rows, or than a prompt's: what puts the parts together is launched for the
    tiles that all rows make, not for those that each sequence might have."""
    B = Batch(H, [1 if b % 50 == 3 else 0 for b in range(2048)], [40 + b % 50 for b in range(2048)], H, 1, 8, 16, 16, spare_rows=8151)
    assert B.T == 8192
    check_attention(B)
    B = Batch(H + 1, [2, 0, 3, 1, 0], [70, 1, 300, 20, 5], H, 1, 8, 16, 8, spare_rows=3)
    check_attention(B)


@GPU
def test_a_bound_of_no_rows_is_refused():
    """max_new = 0 with rows and sequences there, as the C calls refuse it; nothing is returned that nobody wrote."""
    from cacti_amd import ops
    B = Batch(91, [2, 1], [20, 40], 4, 2, 64, 16, 8)
    cache = B.put()
    append = lambda rows, max_new: ops.paged_append(B.d["k"][:rows], B.d["v"][:rows], cache, *B.at(), B.d["cos"], B.d["sin"], q=B.d["q"][:rows],
                                                    max_new=max_new)
    attend = lambda rows, max_new: ops.paged_attention(B.d["q"][:rows], cache, *B.at(), 1.0, max_new=max_new)
    for f in (append, attend):
        for max_new in (0, -1):
            with pytest.raises(AssertionError, match="max_new"):
                f(3, max_new)
        assert f(0, 0).shape == (0, 4, 64)


# ---------------------------------------------------------------- operands that share memory
SHARE = r"""
#include <stdio.h>

#include <set>

#include "operands.h"

int main()
{
    for (int64_t rows : {1, 2, 3})
        for (int64_t lda = 1; lda <= 7; lda++)
            for (int64_t ldb = 1; ldb <= 7; ldb++)
                for (int64_t wa = 1; wa <= lda; wa++)
                    for (int64_t wb = 1; wb <= ldb; wb++)
                        for (int64_t d = -25; d <= 25; d++) {
                            std::set<int64_t> of_a;
                            bool share = false;
                            for (int64_t i = 0; i < rows; i++)
                                for (int64_t k = 0; k < wa; k++) of_a.insert(i * lda + k);
                            for (int64_t i = 0; i < rows; i++)
                                for (int64_t k = 0; k < wb; k++) share = share || of_a.count(d + i * ldb + k);
                            const bool got = cacti::rows_share(rows, (void *)1000, lda, wa, (void *)(1000 + 2 * d), ldb, wb);
                            if (got != share && (share || lda == ldb || rows == 1)) {
                                printf("rows %ld, pitches %ld %ld, widths %ld %ld, %ld apart: %d\n", (long)rows, (long)lda, (long)ldb, (long)wa, (long)wb,
                                       (long)d, (int)got);
                                return 1;
                            }
                        }
    return 0;
}
"""


def test_rows_that_share_memory_are_found(tmp_path):
    """Against sets of addresses; of different pitches rows may be taken to share that lie between each other."""
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(SHARE)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=undefined", "-fno-sanitize-recover", "-Wall", "-Werror", "-I" + CSRC, str(src),
                           "-o", str(exe)])
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr


# rows of 64 heads of queries, 32 of keys, 32 of values, as the product before leaves them; so many sequences that a call that passes is
# too large to be launched
Q, K, V, FAR = 0x100000, 0x100000 + 1024, 0x100000 + 1536, 0x900000
QKV = dict(APPEND, T=5, B=(1 << 20) - 1, H=64, Hkv=32, max_new=5, q=Q, k=K, v=V, qr=Q, ldq=1024, ldk=1024, ldv=1024, ldqr=1024)


@pytest.mark.parametrize("change,why", [
    (dict(), "in one call"), (dict(qr=FAR), "in one call"), (dict(qr=FAR, ldqr=512), "in one call"), (dict(q=FAR, ldq=512, qr=Q), "in one call"),
    (dict(qr=Q - 5 * 2048), "in one call"), (dict(ldqr=2048), "place"), (dict(ldqr=512), "place"),
    (dict(qr=Q + 2048), "place"), (dict(qr=Q - 4 * 2048), "place"), (dict(qr=Q + 8), "place"), (dict(q=FAR, qr=K), "keys or values"),
    (dict(q=FAR, qr=V - 8), "keys or values"), (dict(q=FAR, qr=V, k=FAR), "keys or values"), (dict(q=FAR, qr=Q + 8), "keys or values"),
    (dict(q=FAR, ldqr=512), "keys or values")])
def test_append_refuses_rotated_queries_in_another_place(change, why):
    """The queries' own place, with their pitch, or memory of their own; the columns of q, k and v may lie in the same rows."""
    L = ffi.lib()
    assert L.cacti_hip_paged_append(*dict(QKV, **change).values()) < 0
    assert why in L.cacti_hip_last_error().decode()


@pytest.mark.parametrize("change", [dict(), dict(out=64 + 8), dict(out=64 + 3 * 64), dict(ldo=64), dict(out=128, ldo=32), dict(ldq=64, ldo=64, out=64 + 56)])
def test_attention_refuses_an_output_that_shares_memory_with_the_queries(change):
    L = ffi.lib()
    assert L.cacti_hip_paged_attention_f16(*dict(ATTEND, **change).values()) < 0
    assert "shares memory" in L.cacti_hip_last_error().decode()


@GPU
def test_queries_and_output_in_the_columns_of_one_buffer():
    import torch
    from cacti_amd import ops
    for n, lens in (([2, 1], [30, 70]), ([150, 3], [160, 20])):
        B = Batch(92, n, lens, 4, 2, 100, 16, 16)
        cache = B.put()
        want = ops.paged_attention(B.d["q"], cache, *B.at(), B.alpha)
        both = torch.full((B.T, 1000), 7.0, dtype=torch.float16, device="cuda")
        q, out = both[:, 40:440].view(-1, 4, 100), both[:, 440:840].view(-1, 4, 100)
        q.copy_(B.d["q"])
        assert ops.paged_attention(q, cache, *B.at(), B.alpha, out=out) is out
        assert torch.equal(out, want) and torch.equal(q, B.d["q"]) and bool((both[:, :40] == 7).all()) and bool((both[:, 840:] == 7).all())
        with pytest.raises(ffi.CactiError, match="shares memory"):
            ops.paged_attention(q, cache, *B.at(), B.alpha, out=both[:, 436:836].view(-1, 4, 100))


# ---------------------------------------------------------------- scales
@GPU
@pytest.mark.parametrize("apart", [12, 18, 24])
@pytest.mark.parametrize("n,lens", [([1], [300]), ([2, 1], [200, 90]), ([150, 1], [260, 70])])
def test_attention_of_a_page_with_one_large_value(n, lens, apart):
    """A page whose scale one value made: the weights of the other pages' codes are 2^-apart of its own, and have their bits all the same."""
    B = Batch(93 + apart, n, lens, 4, 2, 64, 16, 8)
    B.vs[:] = 2.0 ** -14
    for b in range(B.B):
        p = B.table[b, 1]
        B.vs[p] = 2.0 ** (apart - 14)
        B.vp[p] = 0
        B.vp[p, :, 5, 3] = 0x70                               # 128
    check_attention(B)


@GPU
@pytest.mark.parametrize("n,lens", [([2], [200]), ([90], [200])])
def test_attention_of_scales_at_the_ends(n, lens):
    """The least and the largest of the value scales, and key scales that are subnormal or near the largest."""
    for what in ("least", "largest beside small ones", "keys of nothing", "keys far up"):
        print("paged_attention", n, what, flush=True)
        B = Batch(94, n, lens, 4, 2, 64, 16, 8)
        odd, even = B.table[0, 1::2], B.table[0, ::2]
        if what == "least":
            B.vs[:] = 2.0 ** -40
        elif what == "largest beside small ones":                 # scores of about 80 against 0
            B.vs[odd], B.vs[even] = 2.0 ** 40, 2.0 ** -10
            B.vp[odd], B.kp[odd], B.kp[even] = 0, 0, 0x38             # 1
            B.qkv[:, :256] = np.abs(B.qkv[:, :256])
            B.ks[:] = 16.0
        elif what == "keys of nothing":
            B.ks[:] = 2.0 ** -140
        else:
            B.ks[:], B.kp[:] = 2.0 ** 100, 0
        check_attention(B)


# ---------------------------------------------------------------- tables without a page to spare
def tight(B, r):
    """B's table as wide as its longest sequence, no page's number where a sequence has no position."""
    B.W = max(1, max(-(-l // B.page) for l in B.lens))
    B.table = np.ascontiguousarray(B.table[:, :B.W])
    for b, l in enumerate(B.lens):
        B.table[b, -(-l // B.page):] = r.choice([-1, B.P, 2 ** 31 - 1, -2 ** 31])
    return B


@GPU
@pytest.mark.parametrize("bits", [8, 16])
@pytest.mark.parametrize("n,lens,H,Hkv,Dh,page", ATTENDS)
def test_pages_that_are_not_a_sequences_are_not_looked_up(n, lens, H, Hkv, Dh, page, bits):
    """(A number of the table that is no page's is named in status, and check_attention wants none.)"""
    print("paged_attention", n, lens, H, Hkv, Dh, page, bits, flush=True)
    r = np.random.default_rng(bits)
    for more in (dict(), dict(max_new=max(n))):
        check_attention(tight(Batch(sum(lens) + Dh + bits + 5, n, lens, H, Hkv, Dh, page, bits), r), **more)


@GPU
@pytest.mark.parametrize("seed", range(6))
def test_pages_of_drawn_batches(seed):
    r = np.random.default_rng(seed)
    G = int(r.choice([1, 2, 3, 8]))
    B = int(r.integers(1, 9))
    n = [int(x) for x in r.integers(0, 180 if seed % 2 else 9, B)]
    lens = [x + int(r.integers(0, 700)) for x in n]
    Hkv, Dh, page, bits = int(r.choice([1, 2])), int(r.choice([20, 64, 100])), 16 * int(r.integers(1, 9)), 8 if seed % 3 else 16
    print("paged_attention", n, lens, G * Hkv, Hkv, Dh, page, bits, flush=True)
    check_attention(tight(Batch(seed, n, lens, G * Hkv, Hkv, Dh, page, bits, spare_rows=1), r))


# ---------------------------------------------------------------- the bound where the sum is that of the weights as they were
class Exact(Batch):
    """But for prompts in 16 bits the weights' rounding is in the numerator alone: sum p |v| 2^-11 and half a step of the output, 2^-11 |o|
    less than what test_paged.py allows for all forms."""

    def attend(self, q, cache):
        o, tol = super().attend(q, cache)
        return o, tol - 2.0 ** -11 * np.abs(o)


EXACT = [c + (bits,) for c in ATTENDS + [([1], [4000], 2, 2, 64, 32), ([6, 1], [1500, 900], 8, 2, 128, 32)] for bits in (8, 16)
         if bits == 8 or max(c[0]) * c[2] // c[3] <= 128]


@GPU
@pytest.mark.parametrize("n,lens,H,Hkv,Dh,page,bits", EXACT)
def test_attention_divides_by_the_weights_as_they_were(n, lens, H, Hkv, Dh, page, bits):
    print("paged_attention", n, lens, H, Hkv, Dh, page, bits, flush=True)
    check_attention(Exact(sum(lens) + Dh + bits + 9, n, lens, H, Hkv, Dh, page, bits), max_new=max(n))


# ---------------------------------------------------------------- drafted tokens that are taken back
@GPU
@pytest.mark.parametrize("slot", [5, 0])
def test_a_large_draft_that_is_taken_back_leaves_its_page_the_scale(slot):
    """In 8 bits a sequence's length takes back the positions of drafted tokens, not what they did to a page that has older ones: its
    scale stays, and the older codes are those of the larger scale.  A page that begins with the drafted tokens is as if new."""
    import torch
    from cacti_amd import ops
    first = 16 + slot
    was = Batch(95, [3], [first + 3], 2, 2, 64, 16, 8)
    was.qkv[2, 128:] = 3000                                   # the second drafted token
    cache, drafted = check_append(was)
    now = Batch(96, [2], [first + 2], 2, 2, 64, 16, 8)
    now.table, now.W, now.P = was.table, was.W, was.P
    now.kp, now.vp, now.ks, now.vs = drafted
    _, want = now.append()
    now.put()
    ops.paged_append(now.d["k"], now.d["v"], cache, *now.at(), now.d["cos"], now.d["sin"])
    for name, g, w in zip(("k pages", "v pages", "k scale", "v scale"), cache, want):
        same_bits(numpy_of(g), w, name)
    page = was.table[0, 1]
    for before, after_draft, after in ((was.ks, drafted[2], want[2]), (was.vs, drafted[3], want[3])):
        assert (after_draft[page] >= 4).all() and (before[page] < 0.1).all()
        assert (after[page] == after_draft[page]).all() if slot else (after[page] < 0.1).all()
    if slot:                                                  # older values, whose codes were up to 448 at a scale below 2^-4
        old, new = E4M3[was.vp[page, :, :slot]] * was.vs[page][:, None, None], E4M3[want[1][page, :, :slot]] * want[3][page][:, None, None]
        assert (np.abs(old - new) <= 2.0 ** -10 * want[3][page].max() + 2.0 ** -4 * np.abs(old)).all() and (old != new).any()
