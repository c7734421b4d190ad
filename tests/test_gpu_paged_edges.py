"""The paged cache, attention over it and rotary positions at their edges: failures among many
entries, values that are not finite, lengths and indices out of range.  Helpers and tolerances
are those of test_gpu_paged."""
import numpy as np
import pytest
import torch

import paged_ref as R
from blt_burn_amd import BltError, cache as C, fused_ops as F, model as M, synth
from test_gpu_paged import DEV, TYPES, Made, att_tol, check_attention, check_rotary, device_rows, f64, i32

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


# ---- gradients ------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("pairs,d,rot", [("half", 64, 64), ("interleaved", 128, 32), ("half", 10, 4)])
@pytest.mark.parametrize("back", [False, True])
def test_rotary_passes_gradients(dtype, pairs, d, rot, back):
    """Autograd's gradients of q and k are the transposed rotation of the outputs' ones."""
    torch.manual_seed(rot)
    kw = dict(scaling="yarn", factor=4.0)
    plan = F.RotaryPlan(rot, pairs=pairs, **kw)
    pos = torch.randint(0, 9000, (2, 7), dtype=torch.int32, device=DEV)
    x = torch.randn(2, 7, 5, d, device=DEV).to(TYPES[dtype]).requires_grad_()
    q, k = x.transpose(1, 2)[:, :3], x.transpose(1, 2)[:, 3:]
    qo, ko = F.fused_rotary(q, k, pos, plan, backward=back)
    with torch.no_grad():
        plain = F.fused_rotary(q, k, pos, plan, backward=back)
    assert torch.equal(qo, plain[0]) and torch.equal(ko, plain[1])
    gq, gk = torch.randn_like(qo), torch.randn_like(ko)
    (gx,) = torch.autograd.grad([qo, ko], x, [gq, gk], retain_graph=True)
    at = pos.cpu().numpy()[:, None]
    check_rotary(gx.transpose(1, 2)[:, :3], gq, at, rot, pairs, not back, **kw)
    check_rotary(gx.transpose(1, 2)[:, 3:], gk, at, rot, pairs, not back, **kw)
    # one output alone: the other input's part is zero
    for out, g, mine in ((qo, gq, slice(0, 3)), (ko, gk, slice(3, 5))):
        (g1,) = torch.autograd.grad(out, x, g, retain_graph=True)
        assert torch.equal(g1.transpose(1, 2)[:, mine], gx.transpose(1, 2)[:, mine])
        assert int((g1 != 0).sum()) <= g1.transpose(1, 2)[:, mine].numel()


def test_rotary_gradients_of_shared_and_broadcast_inputs():
    torch.manual_seed(5)
    plan = F.RotaryPlan(64)
    pos = torch.arange(100, 109, dtype=torch.int32, device=DEV)
    one = torch.randn(1, 1, 9, 64, device=DEV, requires_grad=True)
    q = one.expand(2, 4, 9, 64)
    qo, none = F.fused_rotary(q, None, pos, plan)
    assert none is None
    qo.sum().backward()  # an expanded gradient
    want = R.rotate(np.ones((1, 1, 9, 64)), pos.cpu().numpy(), *R.frequencies(64), "half", True) * 8
    # eight values of at most 2 (6 u + 2e-9) off each, summed in f32
    assert (np.abs(f64(one.grad) - want) <= 8 * 2 * (6 * 2.0 ** -24 + 2e-9 + 8 * 2.0 ** -24)).all()
    # only k needs one; the second derivative is the rotation again
    k = torch.randn(2, 1, 9, 64, device=DEV, requires_grad=True)
    ko = F.fused_rotary(q.detach(), k, pos, plan)[1]
    g = torch.randn_like(ko).requires_grad_()
    (gk,) = torch.autograd.grad(ko, k, g, create_graph=True)
    e = torch.randn_like(gk)
    (gg,) = torch.autograd.grad(gk, g, e)
    assert torch.equal(gg, F.fused_rotary(e, None, pos, plan)[0])
    # against differences: the rotation is linear
    e = torch.randn_like(k)
    y0, y1 = ko.detach(), F.fused_rotary(k.detach() + e, None, pos, plan)[0]
    lhs, rhs = ((y1 - y0).double() * g.double()).sum(), (e.double() * gk.double()).sum()
    bound = 32 * 2.0 ** -24 * ((k.abs() + e.abs() + y1.abs()).double() * g.abs().double()).sum()
    assert abs(lhs - rhs) <= bound
    for f in (lambda: F.fused_rotary(one, None, pos, plan, out=(one, None)),
              lambda: F.fused_rotary(q.detach(), k, pos, plan, out=(q.detach().clone(), k))):
        with pytest.raises(BltError, match="gradient"):
            f()
    with torch.no_grad():
        z = one.detach().clone()
        F.fused_rotary(one, None, pos, plan, out=(z, None))
        assert torch.equal(z, F.fused_rotary(one, None, pos, plan)[0])


def test_rotary_outputs_need_a_gradient_as_their_inputs_do():
    plan, pos = F.RotaryPlan(64), torch.arange(9, dtype=torch.int32, device=DEV)
    for nq, nk in ((False, False), (True, False), (False, True), (True, True)):
        q = torch.randn(1, 2, 9, 64, device=DEV, requires_grad=nq)
        k = torch.randn(1, 1, 9, 64, device=DEV, requires_grad=nk)
        qo, ko = F.fused_rotary(q, k, pos, plan)
        assert (qo.requires_grad, ko.requires_grad) == (nq, nk)
        if nq or nk:
            (qo.sum() + 2 * ko.sum()).backward()
        want = [F.fused_rotary(torch.full_like(x, g).detach(), None, pos, plan, backward=True)[0]
                for x, g in ((q, 1.0), (k, 2.0))]
        for x, need, w in ((q, nq, want[0]), (k, nk, want[1])):
            assert torch.equal(x.grad, w) if need else x.grad is None


def test_rotary_gradient_in_a_captured_graph():
    """Forward and gradient captured and replayed with eager work between, against the eager
    ones; the leaf is used by nothing else while it is captured."""
    torch.manual_seed(6)
    plan = F.RotaryPlan(64, pairs="interleaved")
    pos = torch.arange(9, dtype=torch.int32, device=DEV)
    x = torch.randn(2, 3, 9, 64, device=DEV, requires_grad=True)
    g = torch.randn(2, 3, 9, 64, device=DEV)

    def step(x, g):
        y, _ = F.fused_rotary(x, None, pos, plan)
        return y, torch.autograd.grad(y, x, g)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(x, g)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, gx = step(x, g)
    for i in range(5):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
        g.copy_(torch.randn_like(g))
        graph.replay()
        if i % 2:
            torch.cuda.synchronize()
        e = x.detach().clone().requires_grad_()
        want = step(e, g)
        assert torch.equal(y, want[0]) and torch.equal(gx, want[1]), i


# ---- lengths that no sequence can have ---------------------------------------------------

def test_lengths_out_of_range_stay_in_bounds():
    """A negative length, or one past the table, in the caller's tensors: reserve, fork and trim
    report it and touch nothing outside the sequences' own rows."""
    page, S, cols, P = 8, 4, 6, 20
    kv = [torch.randn(2, P, 1, page, 64, device=DEV).bfloat16() for _ in range(2)]
    around = torch.full((3, S, cols), -77, dtype=torch.int32, device=DEV)
    table, lens, refs = around[1], i32([13, 0, 0, 5]), torch.zeros(P, dtype=torch.int32, device=DEV)
    table[0, :2], table[3, :1] = i32([4, 9]), i32([2])
    refs[[4, 9, 2]] = 1
    c = C.PagedCache.wrap(*kv, table, lens, refs)
    for bad in (-1, -8, -9, -100, -2 ** 31, cols * page + 1, 2 ** 31 - 1):
        lens[0] = bad
        keep = [t.clone() for t in (*kv, around, lens, refs)]
        for call in (lambda: c.reserve(i32([9, 1]), i32([0, 3])), lambda: c.reserve(i32([300]), i32([0])),
                     lambda: c.fork(i32([0, 3]), i32([1, 2])), lambda: c.fork(i32([3, 0]), i32([1, 2]))):
            call()
            with pytest.raises(BltError, match="range|page table"):
                c.check()
            assert all(torch.equal(a, b) for a, b in zip(keep, (*kv, around, lens, refs)))
        if bad < 0:
            for cut in ([0, 0], [3, 0], [0, 3]):
                lens[0] = bad
                c.trim(i32([3, 4]), i32(cut))
                with pytest.raises(BltError, match="range"):
                    c.check()
                assert int(lens[0]) == 0 and lens[1:3].tolist() == [0, 0]
                assert torch.equal(around[0], keep[2][0]) and torch.equal(around[2], keep[2][2])
                lens[3] = 5
            lens[0] = bad
            c.free(i32([0]))
            with pytest.raises(BltError, match="range"):
                c.check()
            assert int(lens[0]) == 0 and torch.equal(refs, keep[4])
    # and a sound one again
    lens[0] = 13
    c.fork(i32([0]), i32([1]))
    c.check()
    assert lens.tolist() == [13, 13, 0, 5] and table[1, :2].tolist() == [4, 0]


def test_arguments_past_32_bits_are_not_cut():
    m = Made([20, 9], Hkv=2, d=64, layers=2)
    c = m.cache
    q = torch.zeros(3, 4, 64, device=DEV, dtype=torch.bfloat16)
    k, v = c.k.clone(), c.v.clone()
    for layer in (-1, 2, 1 << 32, (1 << 32) + 1, -(1 << 32), 1 << 70):
        with pytest.raises(BltError, match="layer"):
            c.attention(layer, q, i32([0, 3]))
        with pytest.raises(BltError, match="layer"):
            c.append(layer, q[:, :2], q[:, :2], i32([0, 3]))
    for window in (-1, -(1 << 32), 5 - (1 << 32), -(1 << 70)):
        with pytest.raises(BltError, match="window"):
            c.attention(0, q, i32([0, 3]), window=window)
    assert torch.equal(c.k.nan_to_num(), k.nan_to_num()) and torch.equal(c.v.nan_to_num(), v.nan_to_num())


# ---- the workspace ---------------------------------------------------------------------

def test_attention_workspace_grows_with_the_calls():
    """A cache takes no more memory than its calls need; larger and smaller ones in any order
    give what a fresh cache gives."""
    base = torch.cuda.memory_allocated()
    m = Made([3000, 900], Hkv=12, d=64)
    size = sum(t.numel() * t.element_size() for t in m.kv)
    assert torch.cuda.memory_allocated() - base < size + (4 << 20)
    torch.manual_seed(1)
    q = torch.randn(1000, 12, 64, device=DEV).bfloat16()

    def call(cache, n):
        return cache.attention(0, q[:sum(n)], i32(np.concatenate([[0], np.cumsum(n)])))

    one = call(m.cache, [1, 1])
    assert torch.cuda.memory_allocated() - base < size + (24 << 20)
    for n in ([500, 500], [1, 1], [900, 100], [3, 2], [0, 1], [1, 1]):
        fresh = C.PagedCache.wrap(*m.kv, m.cache.page_table, m.cache.lens, m.cache.refcount)
        assert torch.equal(call(m.cache, n), call(fresh, n)), n
    assert torch.equal(call(m.cache, [1, 1]), one)
    assert torch.cuda.memory_allocated() - base < size + (160 << 20)


def test_a_captured_call_keeps_its_workspace():
    """A graph captured while the workspace was small is right after it has grown, with eager
    calls of the larger size between its replays."""
    m = Made([5000, 4000], Hkv=4, d=64)
    q = torch.randn(2, 4, 64, device=DEV).bfloat16()
    many = torch.randn(1500, 4, 64, device=DEV).bfloat16()
    one, lots = i32([0, 1, 2]), i32([0, 1000, 1500])
    m.cache.attention(0, q, one)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.cache.attention(0, q, one)
    for i in range(6):
        q.copy_(torch.randn_like(q))
        want_many = m.cache.attention(0, many, lots)
        graph.replay()
        if i % 2:
            torch.cuda.synchronize()
        assert torch.equal(m.cache.attention(0, many, lots), want_many)
        assert torch.equal(out, m.cache.attention(0, q, one)), i
    # and one captured before any call
    m2 = Made([700], Hkv=4, d=64)
    qs, s1 = q[:1], i32([0, 1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m2.cache.attention(0, qs, s1)
    for i in range(4):
        q.copy_(torch.randn_like(q))
        graph.replay()
        assert torch.equal(out, m2.cache.attention(0, qs, s1)), i


def test_a_cache_dropped_while_another_stream_uses_it():
    """record_stream: the memory is not handed out again before that stream is done."""
    m = Made([4000] * 8, Hkv=8, d=64)
    side = torch.cuda.Stream()
    q, starts = torch.randn(8, 8, 64, device=DEV).bfloat16(), i32(np.arange(9))
    want = m.cache.attention(0, q, starts)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            out = m.cache.attention(0, q, starts)
    for t in (q, starts):
        t.record_stream(side)
    m.cache.record_stream(side)
    sizes = [(t.shape, t.dtype) for t in m.kv] + [(t.shape, t.dtype) for t in m.cache._ws]
    del m
    fill = [torch.full(s, 7, dtype=d, device=DEV) for s, d in sizes]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want) and all(bool((f == 7).all()) for f in fill)


# ---- the entropy model, byte by byte -----------------------------------------------------

@pytest.mark.parametrize("dtype,times", [("f32", 1), ("bf16", 2)])
@pytest.mark.parametrize("window,T", [(0, 150), (100, 300)])
def test_the_entropy_model_through_the_cache(window, T, dtype, times):
    """All 14 layers of the entropy model at its sizes over a document that arrives in chunks and
    single bytes, with a continuation forked on the way, against the model's whole-row forward.

    Tolerances: the forward is held to 2e-2 (entropies) and 1e-2 of the largest value
    (embeddings, logits) of an f32 computation, for its bf16 operands.  Through an f32 cache
    everything here is f32: the same bounds.  Through a bf16 one q, k, v and the attention's
    weights and outputs are rounded as the forward rounds them, and nothing else: twice them."""
    cfg = M.entropy_model_config()
    w = M.random_weights(cfg, 4, hidden=2048)
    text = synth.tokens(synth.config_seed(4) + 9, (2, T))
    fork_at = T // 2
    text[1, :fork_at] = text[0, :fork_at]
    tok = torch.from_numpy(text).to(DEV)
    whole = M.LMTransformer(cfg, w, device=0, max_tokens=2 * T, window=window)
    want = whole.forward_with_embeddings(tok)
    f = {n: torch.from_numpy(synth.bf16_to_f32(x)).to(DEV) for n, x in w.items()}
    H, d, t = cfg.resolved_n_heads(), cfg.resolved_head_dim(), TYPES[dtype]
    c = C.PagedCache(cfg.n_layers, H, d, num_pages=64, max_seqs=4, max_len=T, dtype=t)
    plan = F.RotaryPlan(d, theta=cfg.rope_theta)

    def norm(x, weight):
        return F.fused_rms_norm(x[None], weight, cfg.norm_eps)[0]

    def step(rows, seqs, a, b):
        n, s = b - a, i32(seqs)
        starts = i32(np.arange(len(seqs) + 1) * n)
        c.reserve(i32([n] * len(seqs)), s)
        x = f["tok_embeddings"][tok[rows, a:b].reshape(-1).long()]
        for i in range(cfg.n_layers):
            h = norm(x, f["attention_norm"][i])
            q, k, v = ((h @ f[p][i]).view(-1, H, d).to(t) for p in ("wq", "wk", "wv"))
            q = c.append(i, k, v, starts, seqs=s, rotary=plan, q=q)
            o = c.attention(i, q, starts, seqs=s, window=window)
            x = x + o.float().view(-1, H * d) @ f["wo"][i]
            h = norm(x, f["ffn_norm"][i])
            x = x + F.fused_silu_gate((h @ f["w1"][i])[None], (h @ f["w3"][i])[None])[0] @ f["w2"][i]
        logits = norm(x, f["norm"]) @ f["output"]
        entropy = F.fused_entropy(logits[None], cfg.vocab_size)[0]
        return [y.view(len(rows), n, -1) for y in (x, logits, entropy)]

    parts = [[], []]
    for a, b in ((0, 1), (1, fork_at - 1), (fork_at - 1, fork_at)):
        y = step([0], [2], a, b)
        for row in parts:
            row.append([z[0] for z in y])
    c.fork(i32([2]), i32([0]))
    for a, b in ((fork_at, fork_at + 1), (fork_at + 1, T - 2), (T - 2, T - 1), (T - 1, T)):
        y = step([0, 1], [2, 0], a, b)
        for r in range(2):
            parts[r].append([z[r] for z in y])
    c.check()
    x, logits, entropy = (torch.stack([torch.cat([p[j] for p in row]) for row in parts]) for j in range(3))

    def off(got, ref):
        return float((got - ref).abs().max() / ref.abs().max())

    assert off(x, want.pre_norm_embeddings) < times * 1e-2
    assert off(logits, want.logits) < times * 1e-2
    assert float((entropy[..., 0] - want.entropies).abs().max()) < times * 2e-2


# ---- accuracy of the forms for few rows ----------------------------------------------------

def few_tol(want, A, q, keys, d, scale):
    """Up to 32 rows a key head: the weights are two bf16 halves (2^-15 + 2^-22 of each), scores,
    sums and joins f32 as in the f32 forms, and the output is rounded once (2^-8)."""
    return (A * (2.0 ** -15 + 2.0 ** -22) + att_tol(A, q, keys, torch.float32, d, scale)) * 1.01 \
        + 2.0 ** -8 * np.abs(want)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,H,Hkv", [(1, 1, 1), (1, 12, 12), (1, 8, 2), (9, 2, 2), (4, 8, 1), (32, 1, 1)])
@pytest.mark.parametrize("window,causal", [(0, True), (100, True), (0, False)])
def test_attention_few_rows_is_rounded_once(d, n, H, Hkv, window, causal):
    lens = [32, 33, 64, 700, 3000, 6000]
    m = Made(lens, Hkv=Hkv, d=d, seed=n)
    torch.manual_seed(n + H)
    total = n * len(lens)
    q = torch.randn(total, H, d, device=DEV).bfloat16()
    starts = i32(np.arange(len(lens) + 1) * n)
    o = f64(m.cache.attention(0, q, starts, window=window, causal=causal))
    x = f64(q)
    for s, L in enumerate(lens):
        keys, vals, rows = m.rows(0, s), m.rows(1, s), slice(s * n, s * n + n)
        want, A = R.attention(x[rows], keys, vals, L, causal, window)
        err, tol = np.abs(o[rows] - want), few_tol(want, A, x[rows], keys, d, d ** -0.5)
        assert (err <= tol).all(), (L, (err / tol).max())


# ---- many rows ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("B,H,Hkv", [(64, 4, 2), (65, 4, 2), (257, 4, 2), (1000, 2, 1), (4096, 4, 2)])
def test_many_rows(dtype, B, H, Hkv):
    """Rows beyond a wave's lanes, in any order of sequences, some without tokens: what append
    writes, in one call and in calls of 50 rows, and attention of them all."""
    rng = np.random.default_rng(B)
    d, page, t = 64, 8, TYPES[dtype]
    lens = rng.integers(1, 49, B)
    n = np.minimum(rng.integers(0, 4, B), lens)
    order = rng.permutation(B)
    m = Made(lens.tolist(), Hkv=Hkv, d=d, page=page, dtype=t, seed=B)
    c = m.cache
    starts = np.concatenate([[0], np.cumsum(n[order])])
    total = int(starts[-1])
    torch.manual_seed(B)
    x = torch.randn(total + 2, H + 2 * Hkv, d, device=DEV).to(t)
    q, k, v = x[:, :H], x[:, H:H + Hkv], x[:, H + Hkv:]
    plan = F.RotaryPlan(32, pairs="interleaved")
    again = C.PagedCache.wrap(c.k.clone(), c.v.clone(), c.page_table, c.lens, c.refcount)
    qo = c.append(0, k, v, i32(starts), seqs=i32(order), rotary=plan, q=q, out=torch.full_like(q, 5.0))
    assert bool((qo[total:] == 5.0).all())
    for a in range(0, B, 50):
        b, at = min(a + 50, B), slice(int(starts[a]), int(starts[min(a + 50, B)]))
        qs = again.append(0, k[at], v[at], i32(starts[a:b + 1] - starts[a]), seqs=i32(order[a:b]),
                          rotary=plan, q=q[at])
        assert torch.equal(qs, qo[at])
    assert torch.equal(c.k.nan_to_num(), again.k.nan_to_num())
    assert torch.equal(c.v.nan_to_num(), again.v.nan_to_num())
    out = torch.full_like(qo, 7.0)
    c.attention(0, qo, i32(starts), seqs=i32(order), out=out)
    c.check()
    assert bool((out[total:] == 7.0).all()) and int(c._sync.abs().max()) == 0
    # 64-bit reference: every sequence's keys side by side
    row = torch.tensor(np.repeat(order, n[order]), device=DEV)
    length = torch.tensor(lens, device=DEV)
    pos = length[row] - torch.tensor(np.concatenate([np.arange(z, 0, -1) for z in n[order]] or [[]]),
                                     device=DEV)
    pages = c.page_table.clamp(min=0).long()
    keys, vals = (y[0][pages].transpose(2, 3).reshape(B, -1, Hkv, d).nan_to_num().double()
                  for y in (c.k, c.v))
    see = torch.arange(keys.shape[1], device=DEV)[None] <= pos[:, None]
    for h in range(H):
        g = h * Hkv // H
        s = (keys[row, :, g] * qo[:total, None, h].double()).sum(-1) * d ** -0.5
        p = torch.softmax(s.masked_fill(~see, -float("inf")), -1)[..., None]
        want, A = (p * vals[row, :, g]).sum(1), (p * vals[row, :, g].abs()).sum(1)
        smax = float(qo.double().abs().sum(-1).max() * keys.abs().max()) * d ** -0.5
        u = 2.0 ** -24
        tol = u * (2 * (d + 4) * smax + 16 * (1 + smax) + keys.shape[1] + 16) * A
        if dtype == "bf16":  # (1.5 tokens a sequence: a form for few rows)
            tol = (tol + A * (2.0 ** -15 + 2.0 ** -22)) * 1.01 + 2.0 ** -8 * want.abs()
        err = (out[:total, h].double() - want).abs()
        assert bool((err <= tol).all()), float((err / tol).max())


# ---- layouts -----------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_overlapping_rows_are_read_as_they_are(dtype):
    """Rows that overlap (windows of a signal): the new outputs are dense along a head all the
    same, where empty_like lays them out otherwise."""
    torch.manual_seed(2)
    t, T, H, d = TYPES[dtype], 9, 4, 64
    signal = torch.randn(4000, device=DEV).to(t)
    plan, pos = F.RotaryPlan(d), torch.arange(T, dtype=torch.int32, device=DEV)
    m = Made([T], Hkv=H, d=d, dtype=t)
    kv = torch.randn(T, 2, H, d, device=DEV).to(t)
    for st, sh in ((1, 1), (1, d), (8, 1), (64, 32), (0, 0), (0, 64), (1, 0), (24, 8)):
        x = signal.as_strided((T, H, d), (st, sh, 1))
        q = x.transpose(0, 1)[None]
        want, _ = F.fused_rotary(q.contiguous(), None, pos, plan)
        got, k = F.fused_rotary(q, q, pos, plan)
        assert torch.equal(got, want) and torch.equal(k, want), (st, sh)
        got = m.cache.append(0, kv[:, 0], kv[:, 1], i32([0, T]), rotary=plan, q=x)
        assert torch.equal(got, want[0].transpose(0, 1)), (st, sh)
        assert torch.equal(m.cache.attention(0, x, i32([0, T])),
                           m.cache.attention(0, x.contiguous(), i32([0, T]))), (st, sh)


# ---- large scores ------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d,n,H,Hkv", [(64, 1, 2, 2), (128, 1, 4, 1), (64, 20, 1, 1), (64, 150, 2, 1), (128, 90, 2, 2),
                                       (128, 400, 16, 8)])
@pytest.mark.parametrize("scale,size", [(300.0, 1.0), (1e6, 1.0), (1e12, 1.0), (1e25, 1.0), (0.125, 1e6), (1e-4, 1e10)])
def test_attention_of_large_scores_takes_the_largest(scale, size, d, n, H, Hkv, dtype):
    """Where the largest score is far enough above the next for f32 to tell them apart, by more
    than the softmax can see beside it, the output is that key's value, bit for bit."""
    L = max(700, n)
    m = Made([L], Hkv=Hkv, d=d, dtype=TYPES[dtype], seed=n)
    m.kv[0].mul_(size)
    torch.manual_seed(n + d)
    q = (torch.randn(n, H, d, device=DEV) * size).to(TYPES[dtype])
    o = m.cache.attention(0, q, i32([0, n]), scale=scale)
    k, v = device_rows(m, 0, 0).double(), device_rows(m, 1, 0)
    see = torch.arange(L, device=DEV)[None] <= torch.arange(L - n, L, device=DEV)[:, None]
    told = 0
    for h in range(H):
        g = h * Hkv // H
        s = (q[:, h].double() @ k[:, g].t()).masked_fill(~see, -float("inf"))
        # f32 sums of d products: (d + 4) half steps of the sum of their magnitudes
        off = (d + 4) * 2.0 ** -24 * (q[:, h].double().abs() @ k[:, g].abs().t()).amax(-1)
        top = s.topk(2, -1)
        gap = top.values[:, 0] - top.values[:, 1] - 2 * off
        # 700 weights of 2^-140 together are below half a step of any bf16 or f32 value of a
        # normal distribution's size that is not itself below 2^-100
        sure = gap * scale > 100.0
        told += int(sure.sum())
        want = v[top.indices[:, 0], g]
        assert torch.equal(o[:, h][sure], want[sure])
    assert bool(torch.isfinite(o).all()) and float(o.float().abs().max()) <= float(v.float().abs().max()) * 1.01
    assert told * 3 > n * H  # (a third of the rows and more can be told)


# ---- starts ------------------------------------------------------------------------------

@pytest.mark.parametrize("B", [3, 64, 65, 300])
def test_append_reports_starts_out_of_order(B):
    """As attention does: starts that descend, begin below 0 or pass the tokens set the status, and
    nothing outside the rows' own sequences is touched."""
    n, page = 2, 8
    m = Made([20] * B, Hkv=1, d=64, page=page, slots=B + 1)
    c = m.cache
    total = n * B
    x = torch.randn(total, 1, 64, device=DEV).bfloat16()
    free = [p for p in range(c.num_pages) if int(c.refcount[p]) == 0]
    good = np.arange(B + 1) * n
    c.append(0, x, x, i32(good))
    c.check()
    for at, value in ((B, total + 1), (B, total + 1000), (0, -1), (B // 2, total), (B // 2, total + 5), (1, 0),
                      (B, 0)):
        bad = good.copy()
        bad[at] = value
        ascends = (np.diff(bad) >= 0).all() and bad[0] >= 0 and bad[-1] <= total
        for reps in range(3):
            c.append(0, x, x, i32(bad))
            if ascends:
                c.check()
            else:
                with pytest.raises(BltError, match="out of range"):
                    c.check()
    assert bool(torch.isnan(c.k[0, free]).all()) and bool(torch.isnan(c.v[0, free]).all())
    lens = c.lens.tolist()
    assert lens[:B] == [20] * B
    # tokens before the last `total` places of a sequence are what they were
    for s in range(0, B, max(1, B // 7)):
        first = m.rows(1, s)[:max(0, 20 - total)]
        assert np.isfinite(first).all()
