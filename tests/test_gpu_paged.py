"""Rotary positions, the paged cache and attention over it on the GPU against
plain 64-bit restatements (paged_ref).

Tolerances, u = half a step of the type (bf16 2^-8, f32 2^-24):
  rotary     |x| + |y| of the pair times mag times (6 u32 + 2e-9): the angle to 2^-32 turn, the
             series' remainders, three roundings of the products; plus u of the output's own
             rounding
  attention  A = sum p |v|.  bf16: p is rounded to bf16 in the numerator and in the sum (2 u A),
             the output once (u A), and f32 work of the scores and sums below u A / 4.
             f32: a score is off by (d + 4) u of sum |q k| scale, times 2 for the sum, the
             exponential and its argument by 8 u (1 + |score|), sums over n keys n u."""
import numpy as np
import pytest
import torch

import paged_ref as R
from blt_burn_amd import BltError, cache as C, fused_ops as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def f64(t):
    return t.detach().double().cpu().numpy()


# ---- rotary ------------------------------------------------------------------------

def check_rotary(got, x, pos, rot, pairs, backward=False, **kw):
    f, mag = R.frequencies(rot, **kw)
    xs = f64(x)
    want = R.rotate(xs, pos, f, mag, pairs, backward)
    half = rot // 2
    i = np.arange(half)
    p, q = (i, i + half) if pairs == "half" else (2 * i, 2 * i + 1)
    size = np.zeros_like(want)
    size[..., p] = size[..., q] = np.abs(xs[..., p]) + np.abs(xs[..., q])
    tol = size * mag * (6 * 2.0 ** -24 + 2e-9) + U[got.dtype] * np.abs(want) * (size > 0)
    assert (np.abs(f64(got) - want) <= tol + 1e-30).all(), np.abs(f64(got) - want).max()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("pairs", ["half", "interleaved"])
@pytest.mark.parametrize("d,rot", [(64, 64), (64, 32), (64, 16), (64, 6), (128, 128), (128, 64), (80, 80),
                                   (10, 4), (2, 2), (512, 512)])
@pytest.mark.parametrize("B,H,K,T", [(1, 1, 0, 1), (2, 3, 1, 7), (1, 12, 12, 130)])
def test_rotary(dtype, pairs, d, rot, B, H, K, T):
    torch.manual_seed(d + rot + T)
    plan = F.RotaryPlan(rot, pairs=pairs)
    x = torch.randn(B, T, H + K, d, device=DEV).to(TYPES[dtype]).transpose(1, 2)  # packed
    pos = torch.randint(0, 9000, (B, T), dtype=torch.int32, device=DEV)
    q, k = x[:, :H], x[:, H:] if K else None
    for back in (False, True):
        qo, ko = F.fused_rotary(q, k, pos, plan, backward=back)
        assert qo.shape == q.shape and (ko is None) == (K == 0)
        check_rotary(qo, q, pos.cpu().numpy()[:, None], rot, pairs, back)
        if K:
            check_rotary(ko, k, pos.cpu().numpy()[:, None], rot, pairs, back)


@pytest.mark.parametrize("scaling,factor", [("linear", 4.0), ("ntk", 8.0), ("yarn", 16.0)])
@pytest.mark.parametrize("back", [False, True])
def test_rotary_scaled_and_far(scaling, factor, back):
    torch.manual_seed(7)
    plan = F.RotaryPlan(64, scaling=scaling, factor=factor, pairs="interleaved")
    T = 300
    x = torch.randn(1, 4, T, 128, device=DEV)
    pos = i32(np.concatenate([np.arange(-50, 50), np.arange(1000000, 1000100),
                              2 ** 31 - 1 - np.arange(100)]))
    qo, _ = F.fused_rotary(x, None, pos, plan, backward=back)
    f, mag = R.frequencies(64, scaling=scaling, factor=factor)
    # the reference's own angle at 2^31 is off by 2^31 * 2^-53 relative steps: 2.4e-7 in all
    want = R.rotate(f64(x), pos.cpu().numpy(), f, mag, "interleaved", back)
    far = np.abs(pos.cpu().numpy().astype(np.float64))[:, None] * 2.0 ** -52
    xs = np.abs(f64(x))
    size = np.zeros_like(xs)
    size[..., 0:64:2] = size[..., 1:64:2] = xs[..., 0:64:2] + xs[..., 1:64:2]
    tol = size * mag * (6 * 2.0 ** -24 + 2e-9 + far) + 2.0 ** -24 * np.abs(want)
    assert (np.abs(f64(qo) - want) <= tol).all()


def test_rotary_gradient_against_differences_and_in_place():
    torch.manual_seed(3)
    plan = F.RotaryPlan(32, scaling="yarn", factor=4.0)
    pos = torch.arange(5000, 5009, dtype=torch.int32, device=DEV)
    x, g = (torch.randn(2, 3, 9, 64, device=DEV) for _ in range(2))
    y, _ = F.fused_rotary(x, None, pos, plan)
    gx, _ = F.fused_rotary(g, None, pos, plan, backward=True)
    e = torch.randn_like(x)
    y2, _ = F.fused_rotary(x + e, None, pos, plan)  # linear: the difference is exact but for rounding
    lhs, rhs = ((y2 - y).double() * g.double()).sum(), (e.double() * gx.double()).sum()
    bound = 16 * 2.0 ** -24 * ((x.abs() + e.abs() + y2.abs()).double() * g.abs().double()).sum() * 2
    assert abs(lhs - rhs) <= bound
    z = x.clone()
    out = F.fused_rotary(z, None, pos, plan, out=(z, None))
    assert out[0] is z and torch.equal(z, y)
    # unaligned rows and odd strides take the element path, with the same bits
    buf = torch.zeros(2, 3, 9, 67, device=DEV)
    buf[..., 1:65] = x
    w, _ = F.fused_rotary(buf[..., 1:65], None, pos, plan)
    assert torch.equal(w, y)
    e0 = torch.empty(0, 3, 9, 64, device=DEV)
    assert F.fused_rotary(e0, None, pos, plan)[0].shape == e0.shape


def test_rotary_refusals():
    plan = F.RotaryPlan(64)
    q = torch.zeros(1, 2, 3, 64, device=DEV)
    pos = i32([0, 1, 2])
    for f in (lambda: F.fused_rotary(q[0], None, pos, plan),
              lambda: F.fused_rotary(q, q[..., :32], pos, plan),
              lambda: F.fused_rotary(q, q.bfloat16(), pos, plan),
              lambda: F.fused_rotary(q, None, pos.long(), plan),
              lambda: F.fused_rotary(q, None, pos[:2], plan),
              lambda: F.fused_rotary(q.half(), None, pos, plan),
              lambda: F.fused_rotary(q[..., :32], None, pos, plan),
              lambda: F.fused_rotary(q, None, pos.cpu(), plan),
              lambda: F.fused_rotary(q, None, pos, plan, out=(q, q)),
              lambda: F.fused_rotary(q, q, pos, plan, out=(q, q[..., :32]))):
        with pytest.raises(BltError):
            f()


# ---- a cache with contents ---------------------------------------------------------

class Made:
    """A cache of random contents: sequence s has lens[s] tokens on shuffled pages; what no
    sequence owns is NaN."""

    def __init__(self, lens, Hkv=2, d=64, page=16, dtype=torch.bfloat16, layers=1, spare=3, slots=None,
                 columns=None, seed=0):
        rng = np.random.default_rng(seed)
        slots = slots or len(lens)
        need = [-(-n // page) for n in lens]
        pool = sum(need) + spare
        order = rng.permutation(pool)
        cols = columns or max(need + [1])
        table = np.full((slots, cols), -1)
        refs = np.zeros(pool, int)
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = order[at:at + n]
            refs[order[at:at + n]] = 1
            at += n
        g = torch.Generator(device=DEV).manual_seed(seed)
        shape = (layers, pool, Hkv, page, d)
        self.kv = []
        for _ in range(2):
            x = torch.randn(shape, generator=g, device=DEV).to(dtype)
            own = torch.zeros((pool, page), dtype=torch.bool)
            for s, n in enumerate(lens):
                for c in range(need[s]):
                    own[table[s, c], :min(page, n - c * page)] = True
            x.masked_fill_(~own.to(DEV)[None, :, None, :, None], float("nan"))
            self.kv.append(x)
        self.table, self.refs = table, refs
        self.lens = np.concatenate([lens, np.zeros(slots - len(lens), int)]).astype(int)
        self.page = page
        self.cache = C.PagedCache.wrap(*self.kv, i32(table), i32(self.lens), i32(refs))

    def rows(self, which, s, layer=0):
        """[len, Hkv, d] of sequence s, in 64 bits."""
        x, n = self.kv[which][layer], self.lens[s]
        pages = torch.tensor(self.table[s, :-(-n // self.page)], device=DEV, dtype=torch.long)
        x = x[pages].transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])
        return f64(x[:n])

    def pool(self):
        c = self.cache
        return R.Pool(f64(c.k), f64(c.v), c.page_table.cpu().numpy().astype(int),
                      c.lens.cpu().numpy().astype(int), c.refcount.cpu().numpy().astype(int))


def att_tol(A, q, keys, dtype, d, scale):
    if dtype == torch.bfloat16:
        return 3.25 * 2.0 ** -8 * A
    u = 2.0 ** -24
    smax = scale * np.abs(q).sum(-1).max() * np.abs(keys).max() if len(keys) and len(q) else 0.0
    return u * (2 * (d + 4) * smax + 16 * (1 + smax) + len(keys) + 16) * A


def check_attention(m, n, H, seqs=None, causal=True, window=0, scale=None, layer=0, seed=1, tail=3,
                    out=None, strided=False):
    c = m.cache
    d = c.head_dim
    seqs = list(range(len(n))) if seqs is None else seqs
    total = sum(n)
    torch.manual_seed(seed)
    if strided:
        q = torch.randn(total + tail, H, 2, d, device=DEV).to(c.dtype)[:, :, 0]
    else:
        q = torch.randn(total + tail, H, d, device=DEV).to(c.dtype)
    starts = i32(np.concatenate([[0], np.cumsum(n)]))
    o = torch.full((total + tail, H, d), 7.0, dtype=c.dtype, device=DEV)
    r = c.attention(layer, q, starts, seqs=i32(seqs), causal=causal, window=window, scale=scale, out=o)
    assert r is o
    assert bool((o[total:] == 7.0).all())  # behind the last sequence
    at = 0
    sc = d ** -0.5 if scale is None else scale
    for s, k in zip(seqs, n):
        keys, vals = m.rows(0, s, layer), m.rows(1, s, layer)
        x = f64(q[at:at + k])
        want, A = R.attention(x, keys, vals, m.lens[s], causal, window, scale)
        err = np.abs(f64(o[at:at + k]) - want)
        tol = att_tol(A, x, keys, c.dtype, d, sc)
        assert (err <= tol + 1e-30).all(), (s, k, err.max(), np.argwhere(~(err <= tol + 1e-30))[:3])
        at += k
    return o


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("H,Hkv", [(2, 2), (8, 2), (6, 1), (7, 7)])
@pytest.mark.parametrize("page", [8, 16, 64, 1024])
def test_attention_ragged(dtype, d, H, Hkv, page):
    # one token, odd lengths around the tiles, whole prompts, a sequence without new tokens
    m = Made([1, 31, 64, 65, 257, 130, 40], Hkv=Hkv, d=d, page=page, dtype=TYPES[dtype], seed=page + d)
    check_attention(m, [1, 1, 64, 3, 257, 0, 40], H)
    check_attention(m, [1, 31, 1, 65, 1, 130, 7], H, strided=True)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 100, 5000])
def test_attention_window(dtype, window):
    m = Made([5, 64, 300, 1001], Hkv=2, d=64, dtype=TYPES[dtype], seed=window)
    check_attention(m, [5, 1, 150, 77], 4, window=window)
    check_attention(m, [2, 64, 300, 1], 4, window=window)


def test_attention_window_past_32_bits_is_none():
    m = Made([90], Hkv=1, d=64)
    q = torch.randn(3, 1, 64, device=DEV).bfloat16()
    want = m.cache.attention(0, q, i32([0, 3]))
    for window in (1 << 30, (1 << 31) - 1, 1 << 31, (1 << 32) + 5):
        assert torch.equal(m.cache.attention(0, q, i32([0, 3]), window=window), want)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d,H,Hkv,page", [(64, 12, 12, 16), (128, 8, 1, 32), (64, 3, 1, 8)])
def test_attention_long_contexts_in_parts(dtype, d, H, Hkv, page):
    # few row tiles and long contexts: the keys are split and the parts joined
    m = Made([9001, 3, 5000], Hkv=Hkv, d=d, page=page, dtype=TYPES[dtype], seed=d)
    check_attention(m, [1, 1, 1], H)
    check_attention(m, [130, 2, 1], H)
    check_attention(m, [1, 1, 5], H, window=4100)


def attention_on_device(q, keys, values, length, window=0):
    """R.attention in 64-bit torch on the GPU, for the large cases."""
    n, H, d = q.shape
    out, mag = (torch.zeros(n, H, d, dtype=torch.float64, device=DEV) for _ in range(2))
    pos = torch.arange(length - n, length, device=DEV)[:, None]
    j = torch.arange(length, device=DEV)
    hide = j > pos
    if window:
        hide |= j <= pos - window
    for h in range(H):
        g = h * keys.shape[1] // H
        p = (q[:, h].double() @ keys[:, g].double().t()) * d ** -0.5
        p = torch.softmax(p.masked_fill_(hide, -float("inf")), -1)
        out[:, h], mag[:, h] = p @ values[:, g].double(), p @ values[:, g].double().abs()
    return out.cpu().numpy(), mag.cpu().numpy()


def device_rows(m, which, s):
    x, n = m.kv[which][0], m.lens[s]
    pages = torch.tensor(m.table[s, :-(-n // m.page)], device=DEV, dtype=torch.long)
    return x[pages].transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])[:n]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_long_items_reload_their_pages(dtype):
    """So many row tiles that none is split, over more pages of 8 than an item's run of
    page indices in LDS."""
    n, L, H = (4100, 8200, 16) if dtype == "bf16" else (1100, 8200, 16)
    m = Made([L], Hkv=H, d=64, page=8, dtype=TYPES[dtype])
    torch.manual_seed(2)
    q = torch.randn(n, H, 64, device=DEV).to(TYPES[dtype])
    o = m.cache.attention(0, q, i32([0, n]))
    k, v = device_rows(m, 0, 0), device_rows(m, 1, 0)
    for a in (0, n // 2, n - 300):  # 300 rows at a time
        rows = slice(a, a + 300)
        keep = L - n + a + 300
        want, A = attention_on_device(q[rows], k[:keep], v[:keep], keep)
        tol = att_tol(A, f64(q[rows]), f64(k[:keep]), TYPES[dtype], 64, 0.125)
        assert (np.abs(f64(o[rows]) - want) <= tol).all()


def test_attention_long_single_tokens_reload_their_pages():
    """The same for single tokens: 130 rows over one sequence of 8300 keys, none split."""
    H = 16
    m = Made([8300], Hkv=H, d=64, page=8)
    torch.manual_seed(3)
    q = torch.randn(130, H, 64, device=DEV).bfloat16()
    o = m.cache.attention(0, q, i32(np.arange(131)), seqs=i32([0] * 130))
    k, v = device_rows(m, 0, 0), device_rows(m, 1, 0)
    for i in (0, 64, 129):
        want, A = attention_on_device(q[i:i + 1], k, v, 8300)
        assert (np.abs(f64(o[i:i + 1]) - want) <= 3.25 * 2.0 ** -8 * A).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_mixed_batch_and_repeats_bit_for_bit(dtype):
    """Single tokens beside one long chunk (in the form for few rows), and the same bits
    every time: the order in which parts end does not matter."""
    rng = np.random.default_rng(8)
    lens = [int(x) for x in rng.integers(1, 3000, 20)] + [2500]
    m = Made(lens, Hkv=2, d=64, dtype=TYPES[dtype])
    first = check_attention(m, [1] * 20 + [70], 4)
    for _ in range(10):
        assert torch.equal(check_again(m, [1] * 20 + [70], 4), first)


def check_again(m, n, H, seed=1, tail=3):
    torch.manual_seed(seed)
    q = torch.randn(sum(n) + tail, H, m.cache.head_dim, device=DEV).to(m.cache.dtype)
    o = torch.full_like(q, 7.0)
    return m.cache.attention(0, q, i32(np.concatenate([[0], np.cumsum(n)])), seqs=i32(range(len(n))), out=o)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_offsets_past_32_bits(dtype):
    """A pool whose byte and element offsets pass 2^32: append, attention, fork, copies and
    compaction on its last pages."""
    page, Hkv, d = 1024, 8, 128
    per = page * Hkv * d
    P = (1 << 32) // per + 40 if dtype == "bf16" else (1 << 31) // per + 40
    k, v = (torch.empty((1, P, Hkv, page, d), dtype=TYPES[dtype], device=DEV) for _ in range(2))
    table = np.full((3, 4), -1)
    table[0, :3] = [P - 1, P - 7, P - 20]
    refs = np.ones(P, int)
    refs[[5, 9, P - 3]] = 0
    n, L = 40, 2 * page + 90
    c = C.PagedCache.wrap(k, v, i32(table), i32([L, 0, 0]), i32(refs))
    torch.manual_seed(6)
    new = torch.randn(L, 2, Hkv, d, device=DEV).to(TYPES[dtype])
    c.append(0, new[:, 0], new[:, 1], i32([0, L]), seqs=i32([0]))
    c.check()
    q = torch.randn(n, Hkv, d, device=DEV).to(TYPES[dtype])

    def right(seq):
        o = c.attention(0, q, i32([0, n]), seqs=i32([seq]))
        want, A = attention_on_device(q, new[:, 0], new[:, 1], L)
        tol = att_tol(A, f64(q), f64(new[:, 0]), TYPES[dtype], d, d ** -0.5)
        assert (np.abs(f64(o) - want) <= tol).all()

    right(0)
    c.fork(i32([0]), i32([1]))           # the partial page into page 5
    c.check()
    assert c.page_table[1, :3].tolist() == [P - 1, P - 7, 5]
    right(1)
    c.free(i32([0]))
    refs = c.refcount.clone()
    refs[:P - 30] = 1                    # everything below is in use but pages 9 and 11
    refs[[9, 11]] = 0
    c.refcount.copy_(refs)
    c.copy_pages(i32([P - 7]), i32([P - 20]))
    assert torch.equal(c.k[0, P - 20], c.k[0, P - 7]) and torch.equal(c.v[0, P - 20], c.v[0, P - 7])
    c.compact()
    c.check()
    live = int((c.refcount > 0).sum())
    assert int(c.page_table[1, :3].max()) < live and bool((c.refcount[:live] > 0).all())
    right(1)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_not_causal_and_scaled(dtype):
    m = Made([200, 64, 1], Hkv=2, d=64, dtype=TYPES[dtype])
    check_attention(m, [9, 64, 1], 4, causal=False)
    check_attention(m, [9, 64, 1], 4, causal=False, scale=0.5, layer=0)
    check_attention(m, [3, 7, 1], 2, scale=1.0)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_rows_that_see_nothing(dtype):
    """More new tokens than keys (the first ones sit before position 0), and a
    sequence without keys: zeros, not NaN."""
    m = Made([4, 0, 33], Hkv=1, d=64, dtype=TYPES[dtype], slots=4)
    o = check_attention(m, [9, 5, 33, 2], 2, seqs=[0, 1, 2, 3])
    assert bool((o[:5] == 0).all()) and bool((o[9:14] == 0).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_order_layers_and_repeated_sequences(dtype):
    m = Made([70, 20, 190], Hkv=2, d=128, dtype=TYPES[dtype], layers=3, slots=5)
    for layer in range(3):
        check_attention(m, [2, 20, 2, 1], 4, seqs=[2, 1, 2, 0], layer=layer)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_more_sequences_than_lanes(dtype):
    rng = np.random.default_rng(5)
    lens = rng.integers(1, 200, 150)
    n = [int(rng.integers(0, 3)) if i % 7 else int(min(lens[i], 40)) for i in range(150)]
    n = [min(a, int(b)) for a, b in zip(n, lens)]
    m = Made(lens.tolist(), Hkv=1, d=64, page=8, dtype=TYPES[dtype])
    check_attention(m, n, 4)


@pytest.mark.parametrize("dtype,d,H,Hkv,B", [("bf16", 64, 12, 12, 96), ("bf16", 128, 8, 8, 70),
                                             ("f32", 64, 12, 12, 44), ("f32", 128, 4, 4, 70)])
def test_attention_row_tiles_just_above_a_round(dtype, d, H, Hkv, B):
    # (more row tiles than blocks the card holds, by less than half: four rounds of parts)
    m = Made([2200 + (7 * i) % 41 for i in range(B)], Hkv=Hkv, d=d, page=64, dtype=TYPES[dtype])
    some = [0, 1, B // 2, B - 1]
    torch.manual_seed(3)
    q = torch.randn(B, H, d, device=DEV).to(m.cache.dtype)
    o = m.cache.attention(0, q, i32(np.arange(B + 1)))
    assert torch.equal(o, m.cache.attention(0, q, i32(np.arange(B + 1))))
    for s in some:
        x = f64(q[s:s + 1])
        want, A = R.attention(x, m.rows(0, s), m.rows(1, s), m.lens[s])
        assert (np.abs(f64(o[s:s + 1]) - want) <= att_tol(A, x, m.rows(0, s), m.cache.dtype, d,
                                                          d ** -0.5) + 1e-30).all(), s
    assert int(m.cache._sync.abs().max()) == 0


@pytest.mark.parametrize("page,window,causal", [(8, 0, True), (32, 130, True), (16, 0, False)])
def test_attention_f32_of_many_long_chunks(page, window, causal):
    # (its own form: tiles of 128 rows, d = 128; a chunk of nothing and one of one token too)
    lens = [1100, 700, 130, 90, 2100, 640, 1, 333]
    m = Made(lens, Hkv=8, d=128, page=page, dtype=torch.float32, seed=page)
    check_attention(m, [300, 700, 130, 0, 257, 129, 1, 64], 32, window=window, causal=causal)
    check_attention(m, [200, 65, 130, 90, 999, 129, 1, 333], 16, window=window, causal=causal,
                    strided=True)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_attention_f32_of_many_long_chunks_masked_values(value):
    m = Made([600, 500, 700, 650], Hkv=8, d=128, dtype=torch.float32)
    m.kv[1][0, m.table[0, 599 // 16], :, 599 % 16, 3] = value  # seen by the last token alone
    torch.manual_seed(1)
    q = torch.randn(1800, 16, 128, device=DEV)
    n = [600, 300, 500, 400]
    starts = i32(np.concatenate([[0], np.cumsum(n)]))
    got = f64(m.cache.attention(0, q, starts))
    m.kv[1][0, m.table[0, 599 // 16], :, 599 % 16, 3] = 0.5
    want = f64(m.cache.attention(0, q, starts))
    ok = np.ones(got.shape, bool)
    ok[599, :, 3] = False
    assert np.array_equal(got[ok], want[ok])
    assert not np.isfinite(got[599, :, 3]).any()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lens", [[1500], [5000], [9000], [20000], [700, 9000, 65]])
def test_attention_of_one_token_joins_many_parts(dtype, lens):
    m = Made(lens, Hkv=2, d=64, page=16, dtype=TYPES[dtype])
    check_attention(m, [1] * len(lens), 2)
    check_attention(m, [1] * len(lens), 6)
    check_attention(m, [2] * len(lens), 4, window=1400)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_peaked_and_large_scores(dtype):
    """Scores far above and below each other (the running max moves by thousands)."""
    m = Made([700, 90], Hkv=1, d=64, dtype=TYPES[dtype])
    m.kv[0].mul_(30.0)
    check_attention(m, [20, 3], 2, scale=1.0 / 64)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_infinite_keys_are_the_rows_own(dtype):
    """-inf and +inf scores: a key whose score is -inf weighs nothing."""
    m = Made([50], Hkv=1, d=64, dtype=TYPES[dtype])
    ref = m.rows(0, 0), m.rows(1, 0)
    page, slot = m.table[0, 10 // 16], 10 % 16
    m.kv[0][0, page, 0, slot] = 0
    m.kv[0][0, page, 0, slot, 5] = -float("inf")
    q = torch.zeros(2, 1, 64, dtype=TYPES[dtype], device=DEV)
    q[:, :, 5] = 1.0
    o = m.cache.attention(0, q, i32([0, 2]))
    keep = np.delete(np.arange(50), 10)
    want, A = R.attention(f64(q)[1:], ref[0][keep], ref[1][keep], 49)
    tol = att_tol(A, f64(q), ref[0], TYPES[dtype], 64, 0.125)
    assert (np.abs(f64(o[1:]) - want) <= tol).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,H,window", [(150, 1, 0), (9, 1, 0), (9, 3, 0), (150, 1, 40), (20, 1, 70)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_attention_masked_values_stay_masked(dtype, d, n, H, window, value):
    """NaN or infinite keys and values at some positions: the queries that see them have them
    in their outputs, in that column only for a value, and no other query has."""
    L = 200
    m = Made([L], Hkv=1, d=d, dtype=TYPES[dtype])
    clean_k, clean_v = m.rows(0, 0), m.rows(1, 0)
    torch.manual_seed(n)
    q = torch.randn(n, H, d, device=DEV).to(TYPES[dtype])
    bad_v = {L - 5: 3, L - n // 2: d - 1, max(L - n, 0): 20, 60: 33}  # position: column
    for pos, colm in bad_v.items():
        m.kv[1][0, m.table[0, pos // 16], 0, pos % 16, colm] = value
    o = f64(m.cache.attention(0, q, i32([0, n]), window=window))
    want, A = R.attention(f64(q), clean_k, np.where(np.isfinite(m.rows(1, 0)), clean_v, 0.0), L, True, window)
    tol = att_tol(A, f64(q), clean_k, TYPES[dtype], d, d ** -0.5)
    at = L - n + np.arange(n)
    hit = np.zeros((n, 1, d), bool)
    for pos, colm in bad_v.items():
        see = (pos <= at) & ((pos > at - window) if window else True)
        hit[see, 0, colm] = True
    hit = np.broadcast_to(hit, o.shape)
    assert not np.isfinite(o[hit]).any()
    assert (np.abs(o - want)[~hit] <= tol[~hit]).all()
    # a NaN key that only the last tokens see
    m2 = Made([L], Hkv=1, d=d, dtype=TYPES[dtype])
    m2.kv[0][0, m2.table[0, (L - 3) // 16], 0, (L - 3) % 16] = float("nan")
    o = f64(m2.cache.attention(0, q, i32([0, n]), window=window))
    want, A = R.attention(f64(q), clean_k, clean_v, L, True, window)
    tol = att_tol(A, f64(q), clean_k, TYPES[dtype], d, d ** -0.5)
    assert (np.abs(o - want)[:-3] <= tol[:-3]).all()
    assert np.isnan(o[-3:]).all()


def test_attention_bad_indices_stay_in_bounds():
    """Page indices outside the pool, lengths beyond the table and unknown sequences: the
    other rows are what they were, nothing is written for an unknown sequence."""
    m = Made([64, 40], Hkv=2, d=64, slots=4)
    c = m.cache
    q = torch.randn(6, 4, 64, device=DEV).bfloat16()
    m.kv[0].nan_to_num_(0.0)
    m.kv[1].nan_to_num_(0.0)
    starts = i32([0, 1, 2, 4, 6])
    good = c.attention(0, q, starts, seqs=i32([0, 1, 0, 1]))
    c.page_table[2] = i32([-5, 1 << 30, 3, -1])
    c.lens[2] = 1 << 29
    c.lens[3] = -7
    o = torch.full_like(q, 3.0)
    c.attention(0, q, starts, seqs=i32([2, 1, 99, -1]), out=o)
    assert torch.equal(o[1:2], good[1:2]) and bool((o[2:] == 3.0).all())
    o = c.attention(0, q, starts, seqs=i32([3, 1, 2, 0]))
    assert bool((o[0] == 0).all()) and torch.equal(o[1:2], good[1:2])
    with pytest.raises(BltError, match="index out of range"):
        c.check()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_starts_out_of_order_change_nothing(dtype):
    """The bounds on the grid and the workspace rest on starts that ascend within q: such a
    call is reported and writes nothing, and the next one finds the counters as they were."""
    m = Made([900, 40, 700], Hkv=2, d=64, slots=80, dtype=TYPES[dtype])
    c = m.cache
    q = torch.randn(40, 8, 64, device=DEV).to(c.dtype)
    order = i32([0, 1, 2])
    starts = i32([0, 10, 20, 40])
    good = c.attention(0, q, starts, seqs=order)
    c.check()
    many = i32([0, 40] * 35 + [0])  # far more tokens than q holds
    for bad in (i32([0, 10, 5, 40]), i32([0, 10, 41, 41]), i32([-1, 10, 20, 40]), many):
        o = torch.full_like(q, 3.0)
        seqs = order if len(bad) == 4 else torch.zeros(len(bad) - 1, device=DEV, dtype=torch.int32)
        c.attention(0, q, bad, seqs=seqs, out=o)
        assert bool((o == 3.0).all())
        with pytest.raises(BltError, match="index out of range"):
            c.check()
        assert torch.equal(c.attention(0, q, starts, seqs=order), good)
        c.check()
    assert int(c._sync.abs().max()) == 0


def test_attention_refusals():
    m = Made([20], Hkv=2, d=64)
    q = torch.zeros(3, 4, 64, device=DEV, dtype=torch.bfloat16)
    s = i32([0, 3])
    a = m.cache.attention
    for f in (lambda: a(0, q.float(), s), lambda: a(0, q[..., :32], s), lambda: a(0, q[:, :3], s),
              lambda: a(1, q, s), lambda: a(0, q, s.long()), lambda: a(0, q, s, seqs=i32([0, 1])),
              lambda: a(0, q, s, window=-1), lambda: a(0, q, s, scale=0.0), lambda: a(0, q, s, scale=1e-31),
              lambda: a(0, q, s, scale=float("inf")),
              lambda: a(0, q, s, out=q[:2]), lambda: a(0, q, s.cpu()), lambda: a(0, q[0], s)):
        with pytest.raises(BltError):
            f()


# ---- append ------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d,rot,pairs", [(64, 64, "half"), (64, 16, "interleaved"), (128, 128, "interleaved"),
                                         (128, 64, "half"), (64, 10, "half"), (64, 0, "")])
@pytest.mark.parametrize("page", [8, 32])
def test_append(dtype, d, rot, pairs, page):
    lens, n, seqs = [1, 33, 300, 8, 90], [1, 2, 300, 0, 17], [0, 1, 2, 3, 4]
    m = Made(lens, Hkv=2, d=d, page=page, dtype=TYPES[dtype], layers=2, slots=6, seed=rot)
    c = m.cache
    total = sum(n)
    torch.manual_seed(1)
    qkv = torch.randn(total + 2, 8, d, device=DEV).to(c.dtype)
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    before = m.pool()
    starts = i32(np.concatenate([[0], np.cumsum(n)]))
    plan = F.RotaryPlan(rot, pairs=pairs) if rot else None
    kw = dict(rotary=plan, q=q, out=torch.full_like(q, 5.0)) if rot else {}
    qo = c.append(1, k, v, starts, seqs=i32(seqs), **kw)
    c.check()
    at = 0
    for s, cnt in zip(seqs, n):
        pos = m.lens[s] - cnt + np.arange(cnt)
        rows = slice(at, at + cnt)
        if cnt and rot:
            check_rotary(qo[rows].transpose(0, 1), q[rows].transpose(0, 1), pos, rot, pairs)
            got = c.k[1][i32(m.table[s, pos // page]).long(), :, i32(pos % page).long()]
            check_rotary(got.transpose(0, 1), k[rows].transpose(0, 1), pos, rot, pairs)
        for p, i in zip(pos, range(at, at + cnt)):
            before.v[1, m.table[s, p // page], :, p % page] = f64(v[i])
            before.k[1, m.table[s, p // page], :, p % page] = \
                f64(c.k[1, m.table[s, p // page], :, p % page]) if rot else f64(k[i])
        at += cnt
    if rot:
        assert bool((qo[total:] == 5.0).all())
    np.testing.assert_array_equal(f64(c.k), before.k)
    np.testing.assert_array_equal(f64(c.v), before.v)


def test_append_without_pages_is_reported_and_writes_nothing():
    m = Made([20], Hkv=1, d=64, slots=3)
    c = m.cache
    before = m.pool()
    k = torch.ones(4, 1, 64, device=DEV, dtype=torch.bfloat16)
    for setup, seq in ((lambda: None, 1),                       # no tokens reserved: before position 0
                       (lambda: c.lens.__setitem__(1, 4), 1),   # a length without a page
                       (lambda: None, 7), (lambda: None, -1)):
        setup()
        c.append(0, k, k, i32([0, 4]), seqs=i32([seq]))
        with pytest.raises(BltError, match="no page"):
            c.check()
    np.testing.assert_array_equal(f64(c.k), before.k)
    c.append(0, k, k, i32([0, 4]), seqs=i32([0]))
    c.check()
    assert bool((c.k[0, m.table[0, 1], 0, :4] == 1).all())
    for f in (lambda: c.append(0, k, k[:3], i32([0, 4])), lambda: c.append(0, k, k, i32([0, 4]), q=k),
              lambda: c.append(2, k, k, i32([0, 4])), lambda: c.append(0, k.float(), k, i32([0, 4])),
              lambda: c.append(0, k, k, i32([0, 4]), out=k)):
        with pytest.raises(BltError):
            f()


# ---- pages -------------------------------------------------------------------------

def same(c, pool, data=True):
    np.testing.assert_array_equal(c.lens.cpu().numpy(), pool.lens)
    np.testing.assert_array_equal(c.refcount.cpu().numpy(), pool.refs)
    t = c.page_table.cpu().numpy()
    for s, n in enumerate(pool.lens):
        cols = -(-n // pool.page)
        np.testing.assert_array_equal(t[s, :cols], pool.table[s, :cols])
    if data:
        np.testing.assert_array_equal(f64(c.k), pool.k)
        np.testing.assert_array_equal(f64(c.v), pool.v)


@pytest.mark.parametrize("dtype,page,d", [("bf16", 8, 64), ("f32", 16, 128), ("bf16", 64, 64)])
@pytest.mark.parametrize("seed", range(4))
def test_pages_random_walk(dtype, page, d, seed):
    """Reserve, fork, trim, free and compact in random order against the host model,
    failures of a full pool among them."""
    rng = np.random.default_rng(seed)
    S, P = 12, 40
    m = Made([0], Hkv=2, d=d, page=page, dtype=TYPES[dtype], layers=2, spare=P, slots=S, columns=24,
             seed=seed)
    c = m.cache
    c.k.copy_(torch.randn(c.k.shape, device=DEV))
    c.v.copy_(torch.randn(c.v.shape, device=DEV))
    pool = m.pool()
    seen_full = False
    for step in range(60):
        op = rng.choice(["reserve", "reserve", "fork", "trim", "free", "compact"])
        if op == "reserve":
            seqs = rng.permutation(S)[:rng.integers(1, 5)]
            cnt = np.minimum(rng.integers(0, 5 * page, len(seqs)), 24 * page - pool.lens[seqs])
            ok = pool.reserve(seqs, cnt)
            c.reserve(i32(cnt), i32(seqs))
        elif op == "fork":
            empty = [s for s in range(S) if pool.lens[s] == 0]
            used = [s for s in range(S) if pool.lens[s] > 0]
            k = min(len(empty), int(rng.integers(1, 4)))
            if not used or not k:
                continue
            src, dst = rng.choice(used, k), empty[:k]
            ok = pool.fork(src, dst)
            c.fork(i32(src), i32(dst))
        elif op == "trim":
            seqs = rng.permutation(S)[:rng.integers(1, 6)]
            lens = rng.integers(0, 6 * page, len(seqs))
            ok = pool.trim(list(seqs), lens)
            c.trim(i32(lens), i32(seqs))
        elif op == "free":
            seqs = rng.choice(S, 3)  # repeats allowed
            ok = pool.trim(list(seqs), [0] * 3)
            c.free(i32(seqs))
        else:
            ok = True
            pool.compact()
            c.compact()
        if ok:
            c.check()
        else:
            seen_full = True
            with pytest.raises(BltError, match="free pages"):
                c.check()
        same(c, pool)
    assert seen_full


@pytest.mark.parametrize("dtype,page,d,Hkv", [("f32", 512, 64, 2), ("bf16", 256, 128, 3), ("f32", 128, 128, 1)])
def test_large_pages_are_copied_in_parts(dtype, page, d, Hkv):
    """Pages of up to 262 KB: a few of them are cut into parts, by a fork (part of a page), a
    trim, a compaction and copy_pages (whole ones)."""
    m = Made([0], Hkv=Hkv, d=d, page=page, dtype=TYPES[dtype], layers=2, spare=16, slots=6, columns=6)
    c = m.cache
    c.k.copy_(torch.randn(c.k.shape, device=DEV))
    c.v.copy_(torch.randn(c.v.shape, device=DEV))
    pool = m.pool()

    def both(what, *lists):
        getattr(c, what)(*(i32(x) for x in lists))
        if what == "reserve":
            pool.reserve(lists[1], np.array(lists[0]))
        elif what == "fork":
            pool.fork(*lists)
        elif what == "trim":
            pool.trim(lists[1], lists[0])
        elif what == "free":
            pool.trim(lists[0], [0] * len(lists[0]))
        else:
            pool.compact()
        c.check()
        same(c, pool)

    both("reserve", [2 * page + page // 3, page + 1, 40], [0, 1, 2])
    both("fork", [0, 0, 2], [3, 4, 5])
    both("trim", [page + page // 2 + 1, 17], [3, 4])
    both("free", [0, 1])
    both("compact")
    k, v = c.k.clone(), c.v.clone()
    c.copy_pages(i32([0, 1]), i32([15, 13]))
    k[:, [15, 13]], v[:, [15, 13]] = k[:, [0, 1]], v[:, [0, 1]]
    assert torch.equal(c.k, k) and torch.equal(c.v, v)


@pytest.mark.parametrize("P", [9001, 20003])  # lists in LDS, and in the workspace
def test_pages_larger_than_one_step_and_many_entries(P):
    """More pages than one block step reads and more entries than threads."""
    S, page = 3000, 8
    m = Made([0], Hkv=1, d=64, page=page, spare=P, slots=S, columns=8, seed=2)
    m.cache.k.nan_to_num_(0.0)
    m.cache.v.nan_to_num_(0.0)
    c, pool = m.cache, m.pool()
    rng = np.random.default_rng(1)
    cnt = rng.integers(0, 20, S)
    assert pool.reserve(range(S), cnt)
    c.reserve(i32(cnt))
    c.check()
    same(c, pool, False)
    gone = rng.permutation(S)[:1700]
    assert pool.trim(list(gone), [0] * len(gone))
    c.free(i32(gone))
    same(c, pool, False)
    keep = np.setdiff1d(np.arange(S), gone)
    src, dst = rng.choice(keep, 1500), gone[:1500]
    assert pool.fork(src, dst)
    c.fork(i32(src), i32(dst))
    c.check()
    same(c, pool, False)
    lens = rng.integers(0, 12, S)
    assert pool.trim(list(range(S)), lens)
    c.trim(i32(lens))
    c.check()
    same(c, pool, False)
    # contents, told apart by their page
    c.k.add_(torch.arange(P, device=DEV).view(1, -1, 1, 1, 1) % 251)
    c.v.add_(torch.arange(P, device=DEV).view(1, -1, 1, 1, 1) % 241)
    pool.k, pool.v = f64(c.k), f64(c.v)
    pool.compact()
    c.compact()
    same(c, pool)


def test_pages_failures_change_nothing():
    m = Made([20, 40], Hkv=1, d=64, page=16, slots=5, columns=4, spare=2)
    c, pool = m.cache, m.pool()
    pool.k, pool.v = pool.k, pool.v
    bad = [(lambda: c.reserve(i32([1, 1]), i32([0, 0])), "twice"),
           (lambda: c.reserve(i32([1]), i32([9])), "range"),
           (lambda: c.reserve(i32([-1]), i32([0])), "range"),
           (lambda: c.reserve(i32([1, 60]), i32([1, 0])), "page table"),
           (lambda: c.reserve(i32([2 ** 31 - 1]), i32([0])), "page table"),
           (lambda: c.reserve(i32([40, 20]), i32([2, 3])), "free pages"),
           (lambda: c.fork(i32([0]), i32([1])), "with tokens"),
           (lambda: c.fork(i32([0, 0]), i32([2, 2])), "twice"),
           (lambda: c.fork(i32([0, 2]), i32([2, 3])), "twice"),
           (lambda: c.fork(i32([0]), i32([0])), "with tokens"),
           (lambda: c.fork(i32([0]), i32([5])), "range"),
           (lambda: c.fork(i32([-1]), i32([2])), "range"),
           (lambda: c.fork(i32([0, 0, 0]), i32([2, 3, 4])), "free pages")]
    for f, word in bad:
        f()
        # while a failure is pending nothing else is taken either
        c.reserve(i32([1]), i32([0]))
        c.fork(i32([0]), i32([4]))
        k = torch.zeros(1, 1, 64, device=DEV, dtype=torch.bfloat16)
        c.append(0, k, k, i32([0, 1]))
        with pytest.raises(BltError, match=word):
            c.check()
        same(c, pool)
    c.check()
    c.trim(i32([3, -1]), i32([7, 0]))
    with pytest.raises(BltError, match="range"):
        c.check()
    c.copy_pages(i32([0, 99, 1]), i32([1, 0, -2]))
    with pytest.raises(BltError, match="range"):
        c.check()
    pool.k[:, 1], pool.v[:, 1] = pool.k[:, 0], pool.v[:, 0]
    same(c, pool)
    with pytest.raises(BltError):
        c.reserve(i32([1, 1]), i32([0]))
    with pytest.raises(BltError):
        c.fork(i32([1]).long(), i32([2]))


# ---- together ----------------------------------------------------------------------

def test_incremental_attention_equals_the_whole_row():
    """A document in chunks and single bytes through reserve, append and attention, then two
    continuations of it: the rows of fused_attention over the whole text."""
    torch.manual_seed(0)
    H, d, T = 12, 64, 400
    plan = F.RotaryPlan(d)
    q, k, v = (torch.randn(2, T, H, d, device=DEV).bfloat16() for _ in range(3))
    pos = torch.arange(T, dtype=torch.int32, device=DEV)
    for x in (q, k, v):
        x[1, :250] = x[0, :250]  # the second text shares a prefix
    qr, kr = F.fused_rotary(q.transpose(1, 2), k.transpose(1, 2), pos, plan)
    want = F.fused_attention(qr.contiguous(), kr.contiguous(), v.transpose(1, 2).contiguous(), True)
    want = want.transpose(1, 2)
    c = C.PagedCache(1, H, d, num_pages=80, max_seqs=4, max_len=T + 16)

    def step(rows, seqs, a, b):
        s, n = i32(seqs), b - a
        c.reserve(i32([n] * len(seqs)), s)
        starts = i32(np.arange(len(seqs) + 1) * n)
        qs, ks, vs = (x[rows, a:b].reshape(-1, H, d) for x in (q, k, v))
        qn = c.append(0, ks, vs, starts, seqs=s, rotary=plan, q=qs)
        return c.attention(0, qn, starts, seqs=s).view(len(seqs), n, H, d)

    got = torch.zeros(2, T, H, d, device=DEV)
    for a, b in ((0, 130), (130, 131), (131, 250)):
        got[:, a:b] = step([0], [3], a, b).float()
    c.fork(i32([3]), i32([1]))
    c.compact()
    for a, b in ((250, 251), (251, 300), (300, 301), (301, T)):
        got[:, a:b] = step([0, 1], [3, 1], a, b).float()
    c.check()
    # both sides are within 3.25 u A of the exact value, and fused_attention scales q before
    # its rounding, which moves a score by u sum |q k| / 8
    qf, kf, vf = f64(qr.transpose(1, 2)), f64(kr.transpose(1, 2)), f64(v)
    for r in range(2):
        _, A = R.attention(qf[r], kf[r], vf[r], T)
        s = np.einsum("ihd,jhd->hij", np.abs(qf[r]), np.abs(kf[r])).max() / 8
        assert (np.abs(f64(got[r]) - f64(want[r])) <= 2.0 ** -8 * (6.5 + 2 * s) * A).all()
    c.free(i32([3, 1]))
    c.check()
    assert int(c.refcount.sum()) == 0


def test_captured_step_follows_growing_lengths():
    """A captured decode step replayed as the sequences grow over page ends, with eager
    work between; and the same step on another stream."""
    torch.manual_seed(4)
    H, d, S = 4, 64, 3
    plan = F.RotaryPlan(d)
    c, e = (C.PagedCache(1, H, d, num_pages=40, max_seqs=S, max_len=160, page_size=8) for _ in range(2))
    first = torch.randn(60, 3, H, d, device=DEV).bfloat16()
    cnt, starts = i32([37, 3, 20]), i32([0, 37, 40, 60])
    one, ones = i32([1] * S), i32([0, 1, 2, 3])

    def fill(x):
        x.reserve(cnt)
        x.append(0, first[:, 1], first[:, 2], starts, rotary=plan)

    def step(x, t):
        x.reserve(one)
        q = x.append(0, t[:, 1], t[:, 2], ones, rotary=plan, q=t[:, 0])
        return x.attention(0, q, ones)

    fill(c)
    fill(e)
    t = torch.randn(S, 3, H, d, device=DEV).bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = step(c, t)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, step(e, t))
    g = torch.cuda.CUDAGraph()
    buf = t.clone()
    lens = c.lens.clone()
    with torch.cuda.graph(g):
        out = step(c, buf)
    assert torch.equal(c.lens, lens)  # captured, not run
    for i in range(12):
        t = torch.randn(S, 3, H, d, device=DEV).bfloat16()
        buf.copy_(t)
        g.replay()
        if i % 3 == 1:
            torch.cuda.synchronize()
        want = step(e, t)
        assert torch.equal(out, want), i
        assert torch.equal(c.lens, e.lens)
    c.check()
    e.check()
    for s in range(S):
        cols = -(-int(c.lens[s]) // 8)
        assert torch.equal(c.page_table[s, :cols], e.page_table[s, :cols])
    assert torch.equal(c.k, e.k) and torch.equal(c.v, e.v)


def test_constructor_refusals():
    for kw in (dict(head_dim=32), dict(page_size=12), dict(page_size=4), dict(dtype=torch.float16),
               dict(num_pages=0)):
        a = dict(n_layers=1, n_kv_heads=1, head_dim=64, num_pages=4, max_seqs=2, max_len=64)
        a.update(kw)
        with pytest.raises(BltError):
            C.PagedCache(**a)
