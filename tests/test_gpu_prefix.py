"""Attention over a prefix that the sequences of a batch share, against the plain 64-bit
restatement that attention without one is held to (the two are joined by f32 work as parts are),
and the operators of prompts, continuations and answers in one run."""
import math

import numpy as np
import pytest
import torch

import packed_ref
import paged_ref as R
from blt_burn_amd import BltError, cache as C, fused_ops as F
from test_gpu_paged import DEV, TYPES, Made, att_tol, f64, i32
from test_gpu_paged_edges import few_tol
from test_gpu_sample import reference as sample_reference

pytestmark = pytest.mark.gpu


def shared(ctx, tails, page=16, seed=0, **kw):
    """Sequences of ctx + tails[s] tokens whose first ctx // page pages are the same."""
    m = Made([ctx + t for t in tails], page=page, seed=seed, **kw)
    m.table[:len(tails), :ctx // page] = m.table[0, :ctx // page]
    m.cache.page_table.copy_(i32(m.table))
    return m


def check(m, n, H, prefix=None, seqs=None, causal=True, scale=None, seed=1, tail=3, layer=0):
    c = m.cache
    d, total = c.head_dim, sum(n)
    ids = list(range(len(n))) if seqs is None else seqs
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randn(total + tail, H, d, generator=g, device=DEV).to(c.dtype)
    starts = i32(np.concatenate([[0], np.cumsum(n)]))
    if prefix is None:
        prefix = c.common_prefix(i32(ids))
    o = torch.full((total + tail, H, d), 7.0, dtype=c.dtype, device=DEV)
    assert c.attention(layer, q, starts, seqs=i32(ids), causal=causal, scale=scale, out=o,
                       prefix=prefix) is o
    assert bool((o[total:] == 7.0).all()) and int(c._sync.abs().max()) == 0
    at = 0
    for s, k in zip(ids, n):
        keys, vals = m.rows(0, s, layer), m.rows(1, s, layer)
        x = f64(q[at:at + k])
        want, A = R.attention(x, keys, vals, m.lens[s], causal, 0, scale)
        err = np.abs(f64(o[at:at + k]) - want)
        tol = att_tol(A, x, keys, c.dtype, d, d ** -0.5 if scale is None else scale)
        assert (err <= tol + 1e-30).all(), (s, k, err.max(), np.argwhere(~(err <= tol + 1e-30))[:3])
        at += k
    return q, o


# ---- how much is shared ---------------------------------------------------------------

def test_common_prefix():
    c = C.PagedCache(1, 1, 64, num_pages=400, max_seqs=90, max_len=1000, page_size=8)
    c.reserve(i32([100, 37, 0, 9]), i32([0, 1, 2, 3]))
    assert c.common_prefix().tolist() == [0]  # nothing shared
    assert c.common_prefix(i32([0])).tolist() == [0] and c.common_prefix(i32([])).tolist() == [0]
    c.fork(i32([0, 0, 0, 1]), i32([10, 11, 12, 13]))
    c.check()
    for ids, want in (([0, 10, 11, 12], 96), ([10, 12], 96), ([1, 13], 32), ([0, 13], 0),
                      ([2, 0, 2, 10], 96), ([2, 2], 0), ([10, 10], 96), ([3, 3], 8)):
        assert c.common_prefix(i32(ids)).tolist() == [want], ids
    c.reserve(i32([60, 60, 60]), i32([10, 11, 12]))
    assert c.common_prefix(i32([10, 11, 12])).tolist() == [96]
    c.fork(i32([10] * 60), i32(list(range(20, 80))))  # deeper ones, more than a wave of them
    c.check()
    assert c.common_prefix(i32([10] + list(range(20, 80)))).tolist() == [160]
    assert c.common_prefix(i32(list(range(20, 80)) + [11])).tolist() == [96]
    c.trim(i32([41]), i32([33]))
    c.check()
    assert c.common_prefix(i32(list(range(20, 80)))).tolist() == [40]
    out = torch.full((1,), -7, dtype=torch.int32, device=DEV)
    assert c.common_prefix(i32([10, 12]), out=out) is out and out.tolist() == [96]
    for bad in (-1, 90, 2 ** 30):
        assert c.common_prefix(i32([10, bad, 11])).tolist() == [0]
        with pytest.raises(BltError, match="range"):
            c.check()


@pytest.mark.parametrize("n,cols", [(3, 2000), (1500, 40), (70, 1100)])
def test_common_prefix_of_many(n, cols):
    rng = np.random.default_rng(n)
    table = np.tile(np.arange(cols), (n, 1))
    k = torch.zeros(1, 4, 1, 8, 64, device=DEV)
    for at in (0, 1, cols // 2, cols - 1, cols):
        t = table.copy()
        if at < cols:
            t[rng.integers(1, n), at] = 7777
        c = C.PagedCache.wrap(k, k.clone(), i32(t), i32([8 * cols] * n), i32([1] * 4))
        assert c.common_prefix().tolist() == [8 * at]


def test_common_prefix_where_every_sequence_parts_elsewhere():
    """Threads that find a difference early must not leave what others have yet to compare."""
    c = C.PagedCache(1, 1, 64, num_pages=16, max_seqs=700, max_len=8 * 640, page_size=8)
    r = np.random.RandomState(4)
    table = np.zeros((700, c.max_pages), np.int32)  # (page numbers that nothing reads)
    c.lens.fill_(8 * 640)
    for _ in range(20):
        table[:] = 1
        first = r.randint(1, 640, 700)
        first[r.randint(0, 700)] = 0
        low = int(r.randint(0, 300))
        for b in range(1, 700):  # one sequence parts at `low`, the others behind it
            table[b, low + first[b] % (640 - low):] = 2
        b = r.randint(1, 700)
        table[b, low] = 3
        c.page_table.copy_(i32(table))
        assert c.common_prefix().tolist() == [8 * low]


# ---- attention with it ------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d,H,Hkv,page", [(64, 12, 12, 16), (64, 6, 2, 8), (128, 8, 1, 32),
                                          (128, 4, 2, 64), (64, 7, 7, 128)])
@pytest.mark.parametrize("ctx", [5, 300, 2500])
def test_prefix(dtype, d, H, Hkv, page, ctx):
    tails = [1, 9, 70, 33, 140]
    m = shared(ctx, tails, Hkv=Hkv, d=d, page=page, dtype=TYPES[dtype], seed=ctx)
    check(m, [1] * 5, H)
    check(m, [1, 0, 3, 1, 2], H)
    check(m, [1, 9, 70, 2, 140], H)  # all of a sequence's own tokens
    check(m, [1, 4, 1], H, seqs=[4, 2, 4], scale=0.2)
    check(m, [1, 1, 5, 1, 2], H, causal=False)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d,H,Hkv", [(64, 4, 4), (128, 8, 2)])
def test_long_prefix_in_parts(dtype, d, H, Hkv):
    m = shared(9000, [3, 500, 40], Hkv=Hkv, d=d, page=16, dtype=TYPES[dtype])
    check(m, [1, 1, 1], H)
    check(m, [3, 200, 40], H)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("B", [40, 65, 130])
def test_many_continuations(dtype, B):
    rng = np.random.default_rng(B)
    tails = rng.integers(1, 60, B).tolist()
    m = shared(700, tails, Hkv=2, d=64, page=16, dtype=TYPES[dtype])
    check(m, [1] * B, 4)
    check(m, [int(rng.integers(0, t + 1)) for t in tails], 4)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_any_number_is_safe(dtype):
    """More than the rows share of the past, no whole pages, nothing, less than nothing: what
    is taken as shared ends before every row's new tokens."""
    m = shared(200, [30, 2, 90], Hkv=2, d=64, page=16, dtype=TYPES[dtype])
    # (up to 192 tokens are shared; of the second sequence 200 are past)
    for n in (0, -5, 1, 16, 17, 150, 192, 199, 200, 207, 2 ** 31 - 1):
        check(m, [1, 2, 3], 4, prefix=i32([n]))
    m = shared(48, [1, 1], Hkv=2, d=64, page=16, dtype=TYPES[dtype])
    check(m, [49, 49], 4, prefix=i32([48]))  # whole rows: nothing is past
    check(m, [1, 40], 4, prefix=i32([48]))


def test_window_does_without():
    m = shared(300, [5, 9], Hkv=2, d=64)
    q = torch.randn(3, 2, 64, device=DEV).bfloat16()
    s = i32([0, 1, 3])
    want = m.cache.attention(0, q, s, window=70)
    assert torch.equal(m.cache.attention(0, q, s, window=70, prefix=m.cache.common_prefix()), want)


def test_layers_and_strides():
    m = shared(100, [4, 7, 1], Hkv=2, d=64, layers=3)
    for layer in range(3):
        check(m, [1, 2, 1], 4, layer=layer)
    q, want = check(m, [1, 2, 1], 4, layer=1)
    wide = torch.zeros(7, 4, 3, 64, dtype=q.dtype, device=DEV)
    wide[:, :, 1] = q
    got = m.cache.attention(1, wide[:, :, 1], i32([0, 1, 3, 4]), prefix=m.cache.common_prefix())
    assert torch.equal(got[:4], want[:4])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_values_that_are_not_finite(dtype, value):
    """In a sequence's own keys they stay with its rows; in the prefix all rows see them."""
    for ctx, n in ((320, [1, 1, 1]), (320, [1, 30, 2])):
        m = shared(ctx, [8, 40, 20], Hkv=1, d=64, page=16, dtype=TYPES[dtype])
        own = m.table[1, (ctx + 40 - 1) // 16]
        m.kv[1][0, own, 0, (ctx + 40 - 1) % 16, 7] = value  # the second sequence's last token
        g = torch.Generator(device=DEV).manual_seed(3)
        q = torch.randn(sum(n), 2, 64, generator=g, device=DEV).to(TYPES[dtype])
        s = i32(np.concatenate([[0], np.cumsum(n)]))
        o = m.cache.attention(0, q, s, prefix=m.cache.common_prefix())
        last = n[0] + n[1] - 1
        assert not bool(torch.isfinite(o[last, :, 7]).any())
        o[last, :, 7] = 0
        assert bool(torch.isfinite(o).all())
        m.kv[1][0, m.table[0, 3], 0, 5, 9] = value  # of the prefix
        o = m.cache.attention(0, q, s, prefix=m.cache.common_prefix())
        got = o[:, :, 9]
        assert bool(torch.isnan(got).all() if math.isnan(value) else (got == value).all())
        assert bool(torch.isfinite(o[0, :, :9]).all())


def test_scores_of_minus_infinity_in_one_of_the_two():
    """A prefix (or an own tail) whose scores are all -inf weighs nothing."""
    for dtype in TYPES.values():
        m = shared(64, [16, 32], Hkv=1, d=64, page=16, dtype=dtype)
        q = torch.randn(2, 1, 64, device=DEV).to(dtype)
        q[..., 0] = 1
        s = i32([0, 1, 2])
        k = m.kv[0]
        for c in range(4):
            k[0, m.table[0, c], :, :, 0] = -math.inf
        got = m.cache.attention(0, q, s, prefix=m.cache.common_prefix())
        for b, L in enumerate((80, 96)):
            want, A = R.attention(f64(q[b:b + 1]), m.rows(0, b)[64:], m.rows(1, b)[64:], L - 64)
            tol = att_tol(A, f64(q[b:b + 1]), m.rows(0, b)[64:], dtype, 64, 0.125)
            assert (np.abs(f64(got[b:b + 1]) - want) <= tol).all()
        for b in range(2):
            for c in range(4, 4 + b + 1):
                k[0, m.table[b, c], :, :, 0] = -math.inf
        assert not m.cache.attention(0, q, s, prefix=m.cache.common_prefix()).any()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_large_scores(dtype):
    m = shared(128, [16, 32], Hkv=1, d=64, page=16, dtype=TYPES[dtype])
    check(m, [1, 2], 2, scale=500.0)
    check(m, [16, 32], 2, scale=500.0)


# ---- lists, failures, graphs ---------------------------------------------------------------

def test_bad_rows_are_reported():
    m = shared(100, [4, 7, 3], Hkv=2, d=64)
    c = m.cache
    q = torch.randn(3, 4, 64, device=DEV).bfloat16()
    prefix = c.common_prefix()
    want = c.attention(0, q, i32([0, 1, 2, 3]), prefix=prefix)
    o = torch.full_like(q, 7.0)
    c.attention(0, q, i32([0, 1, 2, 3]), seqs=i32([0, 99, 2]), prefix=prefix, out=o)
    with pytest.raises(BltError, match="range"):
        c.check()
    assert torch.equal(o[[0, 2]], want[[0, 2]]) and bool((o[1] == 7).all())
    for bad in ([0, 2, 1, 3], [0, 1, 2, 4], [-1, 1, 2, 3]):
        o = torch.full_like(q, 7.0)
        c.attention(0, q, i32(bad), prefix=prefix, out=o)
        with pytest.raises(BltError, match="range"):
            c.check()
        assert bool((o == 7).all())
    for f in (lambda: c.attention(0, q, i32([0, 1, 2, 3]), prefix=prefix.long()),
              lambda: c.attention(0, q, i32([0, 1, 2, 3]), prefix=prefix.cpu()),
              lambda: c.attention(0, q, i32([0, 1, 2, 3]), prefix=i32([0, 1])),
              lambda: c.common_prefix(out=prefix.long()), lambda: c.common_prefix(i32([[0]]))):
        with pytest.raises(BltError):
            f()
    with pytest.raises(TypeError):
        c.attention(0, q, i32([0, 1, 2, 3]), prefix=96)


@pytest.mark.parametrize("d,H,Hkv,chunk", [(64, 4, 4, 1), (64, 8, 2, 6), (128, 4, 1, 2), (128, 8, 2, 7)])
@pytest.mark.parametrize("B", [40, 90])
def test_many_rows_in_one_launch_with_their_prefix(d, H, Hkv, chunk, B):
    """Many short rows: any number as the prefix, rows without tokens, a sequence twice, unknown
    ones, starts that do not ascend, first tokens and last ones that belong to nobody."""
    rng = np.random.default_rng(B + d)
    m = shared(300, rng.integers(8, 40, B).tolist(), Hkv=Hkv, d=d, page=16)
    c = m.cache
    n = rng.integers(0, chunk + 1, B).tolist()
    n[3], n[5] = 0, chunk
    # (18 pages are shared; every row has 19 and more behind it, so a number of 304 would be taken, and wrong)
    for number in (0, -3, 5, 160, 288, 300):
        check(m, n, H, prefix=i32([number]))
    seqs = list(range(B))
    seqs[7] = seqs[20] = 5
    check(m, n, H, seqs=seqs)
    # tokens in front of the first sequence, unknown sequences
    starts = np.concatenate([[0], np.cumsum(n)]) + 9
    q = torch.randn(int(starts[-1]) + 5, H, d, device=DEV).bfloat16()
    want = c.attention(0, q, i32(starts), out=torch.full_like(q, 7.0))
    assert bool((want[:9] == 7).all() and (want[-5:] == 7).all())
    prefix = c.common_prefix()
    got = c.attention(0, q, i32(starts), prefix=prefix, out=torch.full_like(q, 7.0))
    # (both are off by their own rounding and the weights' at most)
    assert bool(((got.float() - want.float()).abs() <= 2 ** -6 * want.float().abs().amax()).all())
    assert bool((got[:9] == 7).all() and (got[-5:] == 7).all())
    bad = list(range(B))
    bad[5], bad[11] = -1, 5000
    o = c.attention(0, q, i32(starts), seqs=i32(bad), prefix=prefix, out=torch.full_like(q, 7.0))
    with pytest.raises(BltError, match="range"):
        c.check()
    lost = torch.zeros(len(q), dtype=torch.bool)
    for b in (5, 11):
        lost[starts[b]:starts[b + 1]] = True
    lost = lost.to(DEV)
    assert bool((o[lost] == 7).all()) and bool((o[~lost] == got[~lost]).all())
    crossed = starts.copy()
    crossed[B // 2] = crossed[-1] + 1
    o = c.attention(0, q, i32(crossed), prefix=prefix, out=torch.full_like(q, 7.0))
    with pytest.raises(BltError, match="range"):
        c.check()
    assert bool((o == 7).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d,H,Hkv", [(64, 4, 4), (64, 8, 2), (128, 8, 1), (128, 4, 2)])
@pytest.mark.parametrize("ctx,tails,n", [(700, [200, 90, 64], [150, 60, 33]), (2000, [900, 40], [100, 40]),
                                         (64, [300, 280, 5, 270], [290, 1, 0, 129])])
def test_chunks_with_their_prefix(dtype, d, H, Hkv, ctx, tails, n):
    """Chunks of more rows than a tile, over own keys in parts and in one."""
    m = shared(ctx, tails, Hkv=Hkv, d=d, page=16, dtype=TYPES[dtype])
    check(m, n, H)
    check(m, n, H, causal=False, prefix=i32([ctx // 2]))


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_not_finite_in_one_launch_with_their_prefix(value):
    m = shared(320, [8] * 50, Hkv=1, d=64, page=16)
    m.kv[1][0, m.table[9, 20], 0, 7, 7] = value  # a sequence's last token
    q = torch.randn(50, 2, 64, device=DEV).bfloat16()
    run = lambda: m.cache.attention(0, q, i32(range(51)), prefix=m.cache.common_prefix())
    o = run()
    assert not bool(torch.isfinite(o[9, :, 7]).any())
    o[9, :, 7] = 0
    assert bool(torch.isfinite(o).all())
    m.kv[1][0, m.table[0, 3], 0, 5, 9] = value  # of the prefix
    got = run()[:, :, 9]
    assert bool(torch.isnan(got).all() if math.isnan(value) else (got == value).all())


def test_one_launch_in_a_graph_and_on_another_stream():
    m = shared(3000, [60] * 50, Hkv=2, d=64, page=16)
    c, s = m.cache, i32(range(51))
    q = torch.randn(50, 8, 64, device=DEV).bfloat16()
    run = lambda: c.attention(0, q, s, prefix=c.common_prefix())
    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for n in range(4):
        q.normal_()
        c.lens[:4].copy_(i32([3000 + 7 * n, 3060, 3001, 2500 - 400 * n]))
        fresh = run()
        torch.cuda.synchronize()
        graph.replay()
        assert torch.equal(held, fresh)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_same_bits_and_in_a_graph(dtype):
    """Captured with its common_prefix; lengths and pages change between the replays."""
    m = shared(3000, [60] * 6, Hkv=2, d=64, page=16, dtype=TYPES[dtype])
    c = m.cache
    q = torch.randn(6, 8, 64, device=DEV).to(TYPES[dtype])
    s = i32(range(7))
    run = lambda: c.attention(0, q, s, prefix=c.common_prefix())
    want = run()
    for _ in range(3):
        assert torch.equal(run(), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for n in range(4):
        q.normal_()
        c.lens.copy_(i32([3000 + 7 * n, 3060, 3001, 2500 - 400 * n, 3033, 3010]))
        fresh = run()
        torch.cuda.synchronize()
        graph.replay()
        assert torch.equal(held, fresh)


# ---- prompts, continuations, answers in one run -----------------------------------------------

def test_prompts_continued_and_answered():
    """Two prompts read whole in one pack, one of them forked into continuations that grow token
    by token: every output against whole-row attention of the tokens so far, every token
    against the definition."""
    torch.manual_seed(0)
    V, H, K, d, dtype = 260, 4, 2, 64, torch.bfloat16
    emb = torch.randn(V, 96, device=DEV)
    wqkv = torch.randn(96, (H + 2 * K) * d, device=DEV) / 10
    head = torch.randn(H * d, V, device=DEV) / 4
    plan = F.RotaryPlan(d)
    prompts = [torch.randint(0, V, (n,), device=DEV) for n in (70, 41)]
    cache = C.PagedCache(1, K, d, num_pages=64, max_seqs=8, max_len=200, page_size=8, dtype=dtype)

    def qkv(tokens):
        x = (emb[tokens] @ wqkv).to(dtype).view(-1, H + 2 * K, d)
        return x[:, :H], x[:, H:H + K], x[:, H + K:]

    def whole(tokens):
        """q, k rotated and v of a row of tokens, and its attention in 64 bits."""
        q, k, v = qkv(tokens)
        pos = torch.arange(len(tokens), dtype=torch.int32, device=DEV)
        q, k = (x[0].transpose(0, 1) for x in
                F.fused_rotary(q.transpose(0, 1)[None], k.transpose(0, 1)[None], pos, plan))
        return q, k, v, packed_ref.attention(q, k, v, [0, len(tokens)], u=2.0 ** -8)

    # the prompts
    starts = i32([0, 70, 111])
    q, k, v = (torch.cat(x) for x in zip(*[whole(t)[:3] for t in prompts]))
    o = F.fused_packed_attention(q, k, v, starts)
    for a, t in ((0, prompts[0]), (70, prompts[1])):
        r = whole(t)[3]
        assert bool(((o[a:a + len(t)].double().cpu() - r["o"]).abs() <= r["tol_o"]).all())
    raw = [torch.cat(x) for x in zip(*[qkv(t) for t in prompts])]
    cache.reserve(i32([70, 41]), i32([0, 1]))
    qr = cache.append(0, raw[1], raw[2], starts, i32([0, 1]), rotary=plan, q=raw[0])
    again = cache.attention(0, qr, starts, i32([0, 1]))
    cache.check()
    # four continuations of the first
    live = [2, 3, 4, 5]
    cache.fork(i32([0] * 4), i32(live))
    prefix = cache.common_prefix(i32(live))
    assert prefix.tolist() == [64]
    rows = [prompts[0].clone() for _ in live]
    out = again[69:70].expand(4, -1, -1)
    one = i32(range(5))
    for step in range(12):
        logits = out.float().reshape(4, -1) @ head
        u = torch.rand(4, device=DEV)
        token = F.fused_sample(logits, u, temperature=0.9, top_k=60, top_p=0.95, min_p=0.001)
        assert torch.equal(token.cpu(), sample_reference(logits, u, 0.9, 60, 0.95, 0.001))
        rows = [torch.cat([r, token[i:i + 1].long()]) for i, r in enumerate(rows)]
        q, k, v = qkv(token.long())
        cache.reserve(i32([1] * 4), i32(live))
        q = cache.append(0, k, v, one, i32(live), rotary=plan, q=q)
        out = cache.attention(0, q, one, i32(live), prefix=prefix)
        for i, t in enumerate(rows):
            r = whole(t)[3]
            assert bool(((out[i].double().cpu() - r["o"][-1]).abs() <= r["tol_o"][-1]).all()), step
    cache.check()
    assert len({tuple(r.tolist()) for r in rows}) > 1


# ---- sequences that do not have the prefix ---------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("B,H,Hkv", [(3, 4, 2), (12, 4, 4), (40, 4, 2), (90, 8, 2)])
@pytest.mark.parametrize("refilled", [False, True])
def test_a_sequence_filled_after_the_prefix_was_taken(dtype, B, H, Hkv, refilled):
    """One that was empty when common_prefix listed it (or dropped since), with tokens of its own now."""
    ctx = 160
    m = Made([ctx + 3 + b % 20 for b in range(B)], Hkv=Hkv, d=64, page=16, dtype=TYPES[dtype], seed=B)
    other = B // 2
    own = m.table[other].copy()
    m.table[:B, :ctx // 16] = m.table[0, :ctx // 16]
    if not refilled:
        m.table[other] = own
    m.cache.page_table.copy_(i32(m.table))
    full = m.cache.lens.clone()
    if not refilled:
        m.cache.lens[other] = 0
    prefix = m.cache.common_prefix()
    assert prefix.tolist() == [ctx]
    m.table[other] = own
    m.cache.page_table.copy_(i32(m.table))
    m.cache.lens.copy_(full)
    check(m, [1] * B, H, prefix=prefix)
    check(m, [1 + b % 3 for b in range(B)], H, prefix=prefix)
    check(m, [1] * B, H, prefix=prefix, causal=False)
    # without that sequence's tokens, or without the sequence, the prefix is taken as before
    check(m, [1 if b != other else 0 for b in range(B)], H, prefix=prefix)
    ids = [b for b in range(B) if b != other]
    check(m, [1] * (B - 1), H, prefix=prefix, seqs=ids)
    # the first row is the one that does not have it
    ids = [other] + ids
    check(m, [1] * B, H, prefix=prefix, seqs=ids)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("B", [4, 40])
def test_a_sequence_loses_and_regains_the_prefix_between_replays(dtype, B):
    ctx = 320
    m = Made([ctx + 5 + b % 30 for b in range(B)], Hkv=2, d=64, page=16, dtype=TYPES[dtype], seed=B)
    own = m.table[1].copy()
    m.table[:B, :ctx // 16] = m.table[0, :ctx // 16]
    tables = [i32(m.table)]
    m.table[1] = own
    tables.append(i32(m.table))
    c, s, prefix = m.cache, i32(range(B + 1)), i32([ctx])
    q = torch.randn(B, 4, 64, device=DEV).to(TYPES[dtype])
    c.page_table.copy_(tables[0])
    run = lambda: c.attention(0, q, s, prefix=prefix)
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for n in range(5):
        q.normal_()
        c.page_table.copy_(tables[n % 2])
        fresh, plain = run(), c.attention(0, q, s)
        torch.cuda.synchronize()
        graph.replay()
        assert torch.equal(held, fresh)
        # (both are off by their outputs' rounding, 2^-8 at most, and less by their weights')
        assert bool(((held.float() - plain.float()).abs() <= 2 ** -6 * plain.float().abs().amax()).all())


# ---- accuracy ------------------------------------------------------------------------------

@pytest.mark.parametrize("d,H,Hkv,n,B", [(64, 4, 4, 1, 40), (64, 6, 2, 5, 30), (64, 8, 1, 4, 9), (128, 4, 4, 1, 48),
                                         (128, 8, 2, 3, 12), (128, 8, 1, 4, 20), (64, 4, 2, 2, 3)])
@pytest.mark.parametrize("causal,scale", [(True, None), (False, None), (True, 0.25)])
def test_short_rows_are_rounded_once_with_their_prefix_too(d, H, Hkv, n, B, causal, scale):
    """As without a prefix: the weights of rows of up to 32 tokens keep 2^-15."""
    tails = [n + 7 * b % 50 for b in range(B)]
    m = shared(720, tails, Hkv=Hkv, d=d, page=16, seed=d + B)
    g = torch.Generator(device=DEV).manual_seed(B)
    q = torch.randn(n * B, H, d, generator=g, device=DEV).bfloat16()
    starts = i32(np.arange(B + 1) * n)
    o = f64(m.cache.attention(0, q, starts, causal=causal, scale=scale, prefix=m.cache.common_prefix()))
    x = f64(q)
    for s in range(B):
        keys, vals, rows = m.rows(0, s), m.rows(1, s), slice(s * n, s * n + n)
        want, A = R.attention(x[rows], keys, vals, m.lens[s], causal, 0, scale)
        err, tol = np.abs(o[rows] - want), few_tol(want, A, x[rows], keys, d, scale or d ** -0.5)
        assert (err <= tol).all(), (s, (err / tol).max())


# ---- f32 rows in tiles of 128 ------------------------------------------------------------------

@pytest.mark.parametrize("ctx,tails,n", [
    (160, [300, 250, 270, 260], [290, 250, 256, 260]),      # both launches in tiles of 128
    (700, [1500, 40, 700], [500, 30, 600]),                 # own keys in several parts
    (300, [16 + b % 40 for b in range(64)], [16] * 64),     # the prefix in tiles of 128, the tails of 32
    (300, [16 + b % 9 for b in range(62)], [16] * 62)])     # and the prefix in two parts
@pytest.mark.parametrize("causal", [True, False])
def test_f32_in_tiles_of_128_rows(ctx, tails, n, causal):
    m = shared(ctx, tails, Hkv=8, d=128, page=16, dtype=torch.float32, seed=len(n))
    check(m, n, 32, causal=causal)
    check(m, n, 32, causal=causal, prefix=i32([ctx // 2]), scale=0.2)
