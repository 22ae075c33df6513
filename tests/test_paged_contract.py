"""What the paged calls promise of batches whose numbers do not fit together, of operands that share memory and of sizes at the ends
of their ranges.  The plain forms and bounds are those of test_paged.py."""
import numpy as np
import pytest

from test_paged import Batch, numpy_of, same_bits

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
