"""What the paged calls promise of batches whose numbers do not fit together, of operands that share memory and of sizes at the ends
of their ranges.  The plain forms and bounds are those of test_paged.py."""
import numpy as np
import pytest

from cacti_amd import ffi
from test_paged import APPEND, ATTEND, Batch, numpy_of, same_bits

GPU = pytest.mark.gpu


# ---------------------------------------------------------------- numbers that do not fit together
# n, H, Hkv, max_new: few rows; a prompt by itself; prompts and a token beside them; query heads that fill more than a tile
BATCHES = [([2, 3, 2], 4, 2, None), ([300], 4, 2, None), ([140, 1, 90], 4, 2, None), ([3, 2], 72, 1, None)]


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
