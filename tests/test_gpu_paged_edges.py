"""The paged cache, attention over it and rotary positions at their edges: failures among many
entries, values that are not finite, lengths and indices out of range.  Helpers and tolerances
are those of test_gpu_paged."""
import numpy as np
import pytest
import torch

import paged_ref as R
from blt_burn_amd import BltError, cache as C, fused_ops as F
from test_gpu_paged import DEV, TYPES, Made, att_tol, check_attention, f64, i32

pytestmark = pytest.mark.gpu


# ---- failures among many entries ------------------------------------------------------

@pytest.mark.parametrize("n", [65, 200, 1024, 3000])
def test_a_bad_entry_among_many_is_always_reported(n):
    """The block's waves find errors while others still look at the pending status: every one
    of them is reported, and nothing is changed."""
    c = C.PagedCache(1, 1, 64, num_pages=n + 8, max_seqs=2 * n, max_len=32, page_size=8)
    c.reserve(i32([5] * n))
    c.check()
    lens, refs, table = c.lens.clone(), c.refcount.clone(), c.page_table.clone()
    ids = np.arange(n)
    ones = i32([1] * n)
    for at in sorted({0, 1, 63, 64, n // 2, n - 1}):
        for bad, word in ((-1, "range"), (2 * n, "range"), (int(ids[at - 1]), "twice")):
            who = ids.copy()
            who[at] = bad
            for _ in range(8):
                c.reserve(ones, i32(who))
                with pytest.raises(BltError, match=word):
                    c.check()
            dst = n + ids
            dst[at] = bad if word == "range" else n + ids[at - 1]
            for _ in range(8):
                c.fork(i32(ids), i32(dst))
                with pytest.raises(BltError, match=word):
                    c.check()
    assert torch.equal(c.lens, lens) and torch.equal(c.refcount, refs)
    assert torch.equal(c.page_table, table) and int(c._sync.abs().max()) == 0
