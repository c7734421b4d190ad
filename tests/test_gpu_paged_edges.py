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


# ---- values that are not finite -------------------------------------------------------

ODD = [float("inf"), -float("inf"), float("nan")]


def same_value(got, value):
    """Every one of `got` is +inf, -inf or NaN, as `value` is."""
    return bool(np.isnan(got).all() if np.isnan(value) else (got == value).all())


@pytest.mark.parametrize("value", ODD)
@pytest.mark.parametrize("d,H,Hkv", [(64, 2, 2), (128, 4, 1)])
@pytest.mark.parametrize("L", [64 * k for k in (3, 5, 9, 17, 33, 67, 140)])
def test_attention_f32_infinite_values_in_the_last_part(L, d, H, Hkv, value):
    """One token over L keys in parts, with a value that is not finite in the last one's
    last tile, which the token sees whole: it comes through the join as it is, whatever
    the number of parts."""
    m = Made([L], Hkv=Hkv, d=d, dtype=torch.float32)
    torch.manual_seed(L)
    q = torch.randn(1, H, d, device=DEV)
    want = f64(m.cache.attention(0, q, i32([0, 1])))
    pos = L - 7
    m.kv[1][0, m.table[0, pos // 16], :, pos % 16, 5] = value
    got = f64(m.cache.attention(0, q, i32([0, 1])))
    assert same_value(got[:, :, 5], value)
    rest = np.arange(d) != 5
    assert np.array_equal(got[..., rest], want[..., rest])


def check_odd_values(m, q, bad, value, window=0, n=None, rows=None):
    """A copy of `value` at (position, column) pairs `bad` of sequence 0's values: the rows that
    see one have it in that column, as it is, and everything else is the rest's attention."""
    L, d = int(m.lens[0]), q.shape[-1]
    n = len(q) if n is None else n
    k, v = m.rows(0, 0), m.rows(1, 0)
    for pos, col in bad:
        m.kv[1][0, m.table[0, pos // m.page], :, pos % m.page, col] = value
        v[pos, :, col] = 0.0
    o = f64(m.cache.attention(0, q, i32([0, n]), seqs=i32([0]), window=window))
    at = L - n + np.arange(n)
    hit = np.zeros((n, 1, d), bool)
    for pos, col in bad:
        hit[(pos <= at) & ((pos > at - window) if window else True), 0, col] = True
    hit = np.broadcast_to(hit, o.shape)
    assert hit.any() and same_value(o[hit], value)
    want, A = R.attention(f64(q), k, v, L, True, window)
    tol = att_tol(A, f64(q), k, m.cache.dtype, d, d ** -0.5)
    # (a column with the value taken out has no weight of its own there: not compared)
    assert (np.abs(o - want)[~hit] <= tol[~hit] + 1e-30).all()
    return o


@pytest.mark.parametrize("value", ODD)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("L,n,window", [(1, 1, 0), (5, 5, 0), (31, 31, 0), (31, 1, 0), (200, 150, 0),
                                        (200, 9, 0), (200, 150, 40), (200, 20, 70)])
def test_attention_f32_infinite_values_are_seen_as_they_are(L, n, window, d, value):
    """Also in the first tile that a row sees, where it sees only a part of it."""
    m = Made([L], Hkv=1, d=d, dtype=torch.float32, seed=L)
    torch.manual_seed(n)
    q = torch.randn(n, 2, d, device=DEV)
    check_odd_values(m, q, {(L - 1, 3), (max(L - n, 0), 20), (L // 2, d - 1)}, value, window)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("value", ODD)
@pytest.mark.parametrize("d,n,H", [(64, 150, 1), (128, 150, 1)])
def test_attention_infinite_value_of_a_key_far_above_the_others(d, n, H, value, dtype):
    """The key's score is 200 above those of the tiles before, whose outputs are rescaled to
    nothing: its value is not."""
    L, pos = 200, 195
    m = Made([L], Hkv=1, d=d, dtype=TYPES[dtype])
    m.kv[0][0, :, :, :, 0] = 0.0
    m.kv[0][0, m.table[0, pos // 16], 0, pos % 16, 0] = 25.0 * d ** 0.5
    torch.manual_seed(n)
    q = torch.randn(n, H, d, device=DEV).to(TYPES[dtype])
    q[:, :, 0] = 8.0
    o = check_odd_values(m, q, {(pos, 3)}, value)
    assert np.isfinite(o[:n - 5]).all()


@pytest.mark.parametrize("value", ODD)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("L,n,window", [(40, 40, 0), (200, 150, 0), (200, 150, 40), (700, 100, 0)])
def test_attention_bf16_tiles_infinite_values_are_seen_as_they_are(L, n, window, d, value):
    """(more than 32 rows: the form for tiles of 128 rows)"""
    m = Made([L], Hkv=1, d=d, seed=L)
    torch.manual_seed(n)
    q = torch.randn(n, 2, d, device=DEV).bfloat16()
    check_odd_values(m, q, {(L - 1, 3), (max(L - n, 0), 20), (L // 2, d - 1)}, value, window)


@pytest.mark.parametrize("value", ODD)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("L,n,H,window", [(1, 1, 1, 0), (20, 1, 2, 0), (64, 1, 1, 0), (700, 1, 1, 0), (700, 1, 12, 0),
                                          (3000, 1, 4, 0), (200, 9, 2, 0), (200, 20, 1, 70), (700, 30, 1, 0)])
def test_attention_bf16_few_rows_infinite_values_are_seen_as_they_are(L, n, H, window, d, value):
    """(up to 32 rows: the forms for few rows) in tiles that a row sees whole as well as in others,
    of either sign of what rounding the weight leaves."""
    m = Made([L], Hkv=1, d=d, seed=L)
    torch.manual_seed(n)
    q = torch.randn(n, H, d, device=DEV).bfloat16()
    lo = max(L - n - (window or L) + 1, 0)
    bad = {(L - 1, 3), (max(L - n, 0), 20)} | {(lo + i * 7 % (L - lo), 21 + i) for i in range(16)}
    check_odd_values(m, q, bad, value, window)


@pytest.mark.parametrize("value", ODD)
@pytest.mark.parametrize("d,H", [(64, 1), (128, 3)])
def test_attention_few_rows_infinite_value_of_a_key_far_above_the_others(d, H, value):
    test_attention_infinite_value_of_a_key_far_above_the_others(d, 9, H, value, "bf16")
