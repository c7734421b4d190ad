"""Attention over packed sequences and its gradient on the GPU against a plain 64-bit
restatement (packed_ref), whose bounds the differences are held to."""
import math

import numpy as np
import pytest
import torch

import blt_burn_amd as pkg
import packed_ref as R
from blt_burn_amd import BltError, fused_ops as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
HEADS = [(64, 12, 12), (64, 6, 2), (128, 2, 2), (128, 8, 1), (128, 6, 2)]
PACKS = [([1], 0), ([5, 0, 7, 1, 64, 63], 3), ([0, 0, 129, 0], 0), ([1] * 150, 9), ([65, 300, 2], 1)]


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def starts_of(lens):
    return [0] + np.cumsum(lens).tolist()


def made(lens, pad, H, K, d, dtype, seed=0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    T = sum(lens) + pad
    x = torch.randn(T, H + 2 * K, d, generator=g, device=DEV).to(dtype)
    do = torch.randn(T, H, d, generator=g, device=DEV).to(dtype)
    return x[:, :H], x[:, H:H + K], x[:, H + K:], do


def near(got, r, name):
    x, want, tol = got.detach().double().cpu(), r[name], r["tol_" + name]
    same = torch.isinf(want) & (x == want)
    bad = ~(((x - want).abs() <= tol + 1e-30) | same)
    assert not bad.any(), (name, (x - want).abs()[bad].max(), int(bad.sum()))


def both(q, k, v, do, st, **kw):
    """o, lse, dq, dk, dv of the package, checked."""
    s = i32(st)
    o, lse = F.fused_packed_attention(q, k, v, s, return_lse=True, **kw)
    grads = F.fused_packed_attention_backward(do, q, k, v, o, lse, s, **kw)
    r = R.attention(q, k, v, st, do=do, u=U[q.dtype], **kw)
    for name, x in zip(("o", "lse", "dq", "dk", "dv"), (o, lse) + grads):
        near(x, r, name)
    near(F.fused_packed_attention(q, k, v, s, **kw), r, "o")
    return (o, lse) + grads


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d,H,K", HEADS)
@pytest.mark.parametrize("pack", range(len(PACKS)))
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 1), (True, 37), (False, 0)])
def test_packed_attention_and_gradient(dtype, d, H, K, pack, causal, window):
    lens, pad = PACKS[pack]
    q, k, v, do = made(lens, pad, H, K, d, TYPES[dtype], seed=pack)
    out = both(q, k, v, do, starts_of(lens), causal=causal, window=window)
    for x in (out[0],) + out[2:]:  # tokens behind the last sequence
        assert not x[sum(lens):].any()
    assert bool((out[1][sum(lens):] == -math.inf).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lens,window", [([1000], 0), ([700, 400], 512), ([1500], 300)])
def test_longer_ones(dtype, lens, window):
    q, k, v, do = made(lens, 0, 4, 2, 64, TYPES[dtype])
    both(q, k, v, do, starts_of(lens), window=window, scale=0.3)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d,H,K", [(64, 12, 4), (64, 8, 1), (128, 8, 1), (128, 12, 4)])
@pytest.mark.parametrize("lens,causal,window", [([700, 0, 500, 45], True, 0), ([900, 300], True, 400),
                                                ([1, 640], False, 0)])
def test_rows_shared_by_several_blocks(dtype, d, H, K, lens, causal, window):
    """Few keys of many rows: their gradients come from several blocks."""
    q, k, v, do = made(lens, 30, H, K, d, TYPES[dtype], seed=d + H)
    out = both(q, k, v, do, starts_of(lens), causal=causal, window=window)
    assert not any(x[sum(lens):].any() for x in (out[0],) + out[2:])


@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("bf16", 128), ("f32", 64)])
def test_many_tiles_in_an_order_of_their_own(dtype, d):
    lens = [900, 1, 640, 0, 159]
    q, k, v, do = made(lens, 11, 40, 40, d, TYPES[dtype], seed=2)
    out = both(q, k, v, do, starts_of(lens))
    assert not any(x[sum(lens):].any() for x in (out[0],) + out[2:])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_layouts(dtype):
    """Rows of any order and alignment give the bits of dense ones."""
    t, d, H, K, lens = TYPES[dtype], 64, 4, 2, [70, 33]
    q, k, v, do = (x.contiguous() for x in made(lens, 2, H, K, d, t))
    want = both(q, k, v, do, starts_of(lens))

    def wide(x):  # rows that are not 16-byte aligned
        y = torch.zeros(x.shape[0], x.shape[1], d + 3, dtype=t, device=DEV)
        y[..., 1:d + 1] = x
        return y[..., 1:d + 1]

    def by_heads(x):
        return x.transpose(0, 1).contiguous().transpose(0, 1)

    def by_dims(x):  # the last dimension is not dense
        return x.transpose(0, 2).contiguous().transpose(0, 2)

    for f in (wide, by_heads, by_dims):
        got = both(f(q), f(k), f(v), f(do), starts_of(lens))
        assert all(torch.equal(a, b) for a, b in zip(got, want)), f
    # one key and value head expanded over all tokens' heads
    ke, ve = k[:, :1].expand(-1, K, -1), v[:, :1].expand(-1, K, -1)
    both(q, ke, ve, do, starts_of(lens))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_out_and_tail(dtype):
    t = TYPES[dtype]
    lens, pad = [40, 3], 200
    q, k, v, do = made(lens, pad, 4, 4, 64, t)
    s = i32(starts_of(lens))
    buf = torch.full((sum(lens) + pad, 6, 64), 7.0, dtype=t, device=DEV)
    o = F.fused_packed_attention(q, k, v, s, out=buf[:, 1:5])
    assert o.data_ptr() == buf[:, 1:5].data_ptr()
    assert torch.equal(o[:43], F.fused_packed_attention(q, k, v, s)[:43])
    assert bool((buf[43:] == 7).all() and (buf[:, 0] == 7).all() and (buf[:, 5] == 7).all())
    # no sequence at all, and no token
    assert not F.fused_packed_attention(q, k, v, i32([0])).any()
    e = [x[:0] for x in (q, k, v, do)]
    o, lse = F.fused_packed_attention(*e[:3], i32([0, 0]), return_lse=True)
    assert o.shape == (0, 4, 64) and lse.shape == (0, 4)
    g = F.fused_packed_attention_backward(e[3], *e[:3], o, lse, i32([0, 0]))
    assert [x.shape[0] for x in g] == [0, 0, 0]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_large_offsets(dtype):
    """Token strides of 2^23 elements: rows lie past 2^32 bytes."""
    t, n = TYPES[dtype], 300
    q, k, v, do = made([n], 0, 2, 1, 64, t)
    far = torch.empty(n << 23, dtype=t, device=DEV)
    x = far.as_strided((n, 7, 64), (1 << 23, 64, 1))
    x[:, :2], x[:, 2:3], x[:, 3:4], x[:, 4:6] = q, k, v, do
    want = both(q.contiguous(), k.contiguous(), v.contiguous(), do.contiguous(), [0, n])
    got = both(x[:, :2], x[:, 2:3], x[:, 3:4], x[:, 4:6], [0, n])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_many_heads_of_few_tokens(dtype):
    """(as many tiles as a pack of many tokens has, and an order of them)"""
    q, k, v, do = made([2, 1], 2, 512, 512, 64, TYPES[dtype])
    both(q, k, v, do, [0, 2, 3])


# ---- values that are not finite ----------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("where", ["q", "k", "v", "do"])
@pytest.mark.parametrize("d,H,K", [(64, 2, 2), (128, 4, 1)])
@pytest.mark.parametrize("window", [0, 20])
def test_not_finite_stays_where_it_is_seen(dtype, value, where, d, H, K, window):
    """One bad value in the middle sequence: other sequences, and of its own the tokens that it
    cannot reach, are what they are without it, within their bounds (not bit for bit: the rows of a
    wave move the offset of their weights together, and weights against another offset round
    otherwise)."""
    lens, at = [50, 90, 40], 50 + 45
    st = starts_of(lens)
    t = TYPES[dtype]
    q, k, v, do = (x.clone() for x in made(lens, 3, H, K, d, t))
    s = i32(st)

    def run():
        o, lse = F.fused_packed_attention(q, k, v, s, window=window, return_lse=True)
        return (o, lse) + F.fused_packed_attention_backward(do, q, k, v, o, lse, s, window=window)

    r = R.attention(q, k, v, st, window=window, do=do, u=U[t])
    dict(q=q, k=k, v=v, do=do)[where][at, 0, 5] = value
    got = run()
    T, end = sum(lens) + 3, st[2]
    i = torch.arange(T)
    last = min(end, at + window) if window else end  # tokens that see the bad key: at .. last - 1
    first = max(st[1], at - window + 1) if window else st[1]  # keys that the bad token sees
    if where in "kv":  # rows at .. last - 1 are reached, and through them keys they see
        rows = (i >= at) & (i < last)
        low = max(st[1], at - window + 1) if window else st[1]
        keys = (i >= low) & (i < last)
    else:
        rows = i == at
        keys = (i >= first) & (i <= at)
    for name, x in zip(("o", "lse", "dq", "dk", "dv"), got):
        keep = ~(keys if name in ("dk", "dv") else rows)
        near(x[keep.to(DEV)], {name: r[name][keep], "tol_" + name: r["tol_" + name][keep]}, name)
    # and it is not lost where it is seen
    if where == "v":
        col = got[0][at:last, :H // K, 5]
        assert bool((~torch.isfinite(col)).all())
    if where == "do":
        assert bool((~torch.isfinite(got[4][first:at + 1, 0, 5])).all())
        assert bool((~torch.isfinite(got[2][at, 0])).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
def test_not_finite_with_rows_shared_by_several_blocks(dtype, d):
    """(as above: one bad dO, one bad q; 8 heads of one key head, sequences of 600 and 500)"""
    st, at, t = [0, 600, 1100], 700, TYPES[dtype]
    q, k, v, do = (x.clone() for x in made([600, 500], 0, 8, 1, d, t))
    r = R.attention(q, k, v, st, do=do, u=U[t])
    q[at, 3, 1], do[at, 5, 2] = math.inf, math.nan
    o, lse = F.fused_packed_attention(q, k, v, i32(st), return_lse=True)
    dq, dk, dv = F.fused_packed_attention_backward(do, q, k, v, o, lse, i32(st))
    i = torch.arange(1100)
    rows, keys = i == at, (i >= 600) & (i <= at)
    for name, x in (("o", o), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        keep = ~(keys if name in ("dk", "dv") else rows)
        near(x[keep.to(DEV)], {name: r[name][keep], "tol_" + name: r["tol_" + name][keep]}, name)
    assert bool(torch.isnan(dv[600:at + 1, 0, 2]).all())
    assert bool((~torch.isfinite(dk[600:at + 1, 0])).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_scores_of_minus_infinity(dtype):
    """Keys whose scores are -inf weigh nothing; a token that has no others gets 0."""
    t = TYPES[dtype]
    q, k, v, do = (x.clone() for x in made([60], 0, 1, 1, 64, t))
    q[..., 0] = 1
    k[:20, :, 0] = -math.inf  # score -inf for everybody
    s = i32([0, 60])
    o, lse = F.fused_packed_attention(q, k, v, s, return_lse=True)
    o2 = F.fused_packed_attention(q, k, v, s)
    assert not o[:20].any() and not o2[:20].any() and bool((lse[:20] == -math.inf).all())
    # the others as if the sequence began behind them
    r = R.attention(q[20:], k[20:], v[20:], [0, 40], u=U[t])
    near(o[20:], r, "o")
    near(o2[20:], r, "o")
    near(lse[20:], r, "lse")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("size", [30.0, 1000.0])
def test_large_scores(dtype, size):
    """Scores in the hundreds and beyond: one key takes nearly everything, nothing overflows."""
    t = TYPES[dtype]
    q, k, v, do = made([200], 0, 2, 2, 64, t)
    q, k = (q.float() * size).to(t), k.clone()
    o, lse = F.fused_packed_attention(q, k, v, i32([0, 200]), return_lse=True)
    r = R.attention(q, k, v, [0, 200], u=U[t])
    near(o, r, "o")
    near(lse, r, "lse")
    g = F.fused_packed_attention_backward(do, q, k, v, o, lse, i32([0, 200]))
    assert all(bool(torch.isfinite(x).all()) for x in g)


# ---- gradients ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_autograd(dtype):
    t = TYPES[dtype]
    lens = [33, 70]
    q, k, v, do = made(lens, 5, 6, 2, 64, t)
    s = i32(starts_of(lens))
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    o, lse = F.fused_packed_attention(*leaves, s, window=40, return_lse=True)
    assert o.requires_grad and not lse.requires_grad
    got = torch.autograd.grad(o, leaves, do)
    want = F.fused_packed_attention_backward(do, q, k, v, o.detach(), lse, s, window=40)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # only what is asked for; a broadcast gradient
    o = F.fused_packed_attention(q, leaves[1], v, s)
    o.sum().backward()
    assert leaves[0].grad is None and leaves[1].grad.shape == k.shape
    one = F.fused_packed_attention_backward(torch.ones_like(q.contiguous()), q, k, v,
                                            *F.fused_packed_attention(q, k, v, s, return_lse=True), s)
    assert torch.equal(leaves[1].grad, one[1])
    # shared leaves: q, k and v views of one tensor
    x = torch.cat([q, k, v], 1).requires_grad_()
    F.fused_packed_attention(x[:, :6], x[:, 6:8], x[:, 8:], s, window=40).backward(do)
    assert all(torch.equal(a, b) for a, b in zip(x.grad.split([6, 2, 2], 1), want))
    with pytest.raises(BltError):
        F.fused_packed_attention(*leaves, s, out=torch.empty_like(q))


def test_gradient_against_differences():
    """<do, o(x + h e) - o(x - h e)> / 2 h against <grad, e>, in f32."""
    lens = [20, 45]
    q, k, v, do = made(lens, 0, 4, 2, 64, torch.float32, seed=5)
    s = i32(starts_of(lens))
    o, lse = F.fused_packed_attention(q, k, v, s, return_lse=True)
    grads = F.fused_packed_attention_backward(do, q, k, v, o, lse, s)
    h = 2.0 ** -6
    for n, x in enumerate((q, k, v)):
        g = torch.Generator(device=DEV)
        g.manual_seed(n)
        e = torch.randn(x.shape, generator=g, device=DEV)

        def at(y):
            args = [q, k, v]
            args[n] = y
            return R.attention(*args, starts_of(lens))["o"]

        # (third differences bound what is left of the central one's error)
        w = do.double().cpu()
        xd, ed = x.double(), e.double()
        f = {j: float((w * at(xd + j * h * ed)).sum()) for j in (-2, -1, 1, 2)}
        diff = (f[1] - f[-1]) / (2 * h)
        third = abs(f[2] - 2 * f[1] + 2 * f[-1] - f[-2]) / (2 * h) / 6
        got = float((grads[n].double() * ed).sum())
        r = R.attention(q, k, v, starts_of(lens), do=do)
        tol = float((r["tol_" + ("dq", "dk", "dv")[n]] * e.double().cpu().abs()).sum())
        assert abs(got - diff) <= 2 * third + tol + 1e-9, (n, got, diff, third)


# ---- runs, streams, graphs ---------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_same_bits_in_every_run_and_in_a_graph(dtype):
    t = TYPES[dtype]
    lens = [300, 77, 1, 150]
    q, k, v, do = (x.clone() for x in made(lens, 20, 4, 2, 128, t))
    s = i32(starts_of(lens))

    def run():
        o, lse = F.fused_packed_attention(q, k, v, s, return_lse=True)
        return (o, lse) + F.fused_packed_attention_backward(do, q, k, v, o, lse, s)

    want = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for n in range(4):  # other inputs and lengths between the replays
        q.normal_()
        do.normal_()
        s.copy_(i32(starts_of([[300, 77, 1, 150], [10, 500, 3, 0], [528, 0, 0, 0], [1, 1, 1, 1]][n])))
        fresh = run()
        torch.cuda.synchronize()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(held, fresh))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_autograd_in_a_graph(dtype):
    """Forward and gradient through autograd, captured together, on leaves without another graph."""
    t = TYPES[dtype]
    q, k, v, do = (x.clone() for x in made([200, 90], 6, 8, 2, 64, t))
    s = i32([0, 200, 290])
    leaves = [x.requires_grad_() for x in (q, k, v)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(F.fused_packed_attention(*leaves, s, window=50), leaves, do)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = F.fused_packed_attention(*leaves, s, window=50)
        grads = torch.autograd.grad(o, leaves, do)
        o = o.detach()
    for n in range(3):
        with torch.no_grad():
            q.normal_()
            do.normal_()
            s.copy_(i32([[0, 200, 290], [0, 10, 280], [0, 0, 296]][n]))
            want, lse = F.fused_packed_attention(q, k, v, s, window=50, return_lse=True)
            fresh = F.fused_packed_attention_backward(do, q, k, v, want, lse, s, window=50)
        torch.cuda.synchronize()
        graph.replay()
        assert torch.equal(o, want) and all(torch.equal(a, b) for a, b in zip(grads, fresh))


def test_starts_that_do_not_ascend_stay_within_the_tensors():
    """Their outputs are not specified, but rows outside the pack are left alone."""
    for t in TYPES.values():
        q, k, v, do = made([100], 0, 2, 2, 64, t)
        for st in ([0, 70, 30, 100], [-5, 1000], [50, 20], [100, 100, 0], [0, 2 ** 31 - 1]):
            s = i32(st)
            o, lse = F.fused_packed_attention(q, k, v, s, return_lse=True)
            g = F.fused_packed_attention_backward(do, q, k, v, o, lse, s)
            assert o.shape == q.shape and len(g) == 3
    torch.cuda.synchronize()


def test_refusals():
    q, k, v, do = made([10], 0, 4, 2, 64, torch.bfloat16)
    s = i32([0, 10])
    o, lse = F.fused_packed_attention(q, k, v, s, return_lse=True)
    for f in (lambda: F.fused_packed_attention(q[..., :32], k[..., :32], v[..., :32], s),
              lambda: F.fused_packed_attention(q, k.float(), v, s),
              lambda: F.fused_packed_attention(q.half(), k.half(), v.half(), s),
              lambda: F.fused_packed_attention(q, k[:9], v, s),
              lambda: F.fused_packed_attention(q, k, v[:, :1], s),
              lambda: F.fused_packed_attention(q[:, :3], k, v, s),
              lambda: F.fused_packed_attention(q, k[:, :0], v[:, :0], s),
              lambda: F.fused_packed_attention(q, k, v, s.long()),
              lambda: F.fused_packed_attention(q, k, v, s.cpu()),
              lambda: F.fused_packed_attention(q, k, v, s[:0]),
              lambda: F.fused_packed_attention(q, k, v, s[None]),
              lambda: F.fused_packed_attention(q, k, v, s, window=-1),
              lambda: F.fused_packed_attention(q, k, v, s, scale=0.0),
              lambda: F.fused_packed_attention(q, k, v, s, scale=math.nan),
              lambda: F.fused_packed_attention(q, k, v, s, out=torch.empty_like(k)),
              lambda: F.fused_packed_attention(q, k, v, s, out=o.float()),
              lambda: F.fused_packed_attention(q, k, v, s, out=o[:, :1].expand(-1, 4, -1)),
              lambda: F.fused_packed_attention(q, k, v, s, out=o[:1].expand(10, -1, -1)),
              lambda: F.fused_packed_attention(q, k, v, s, out=torch.empty(10, 4, 65, device=DEV,
                                                                           dtype=q.dtype)[..., 1:]),
              lambda: F.fused_packed_attention(q.cpu(), k.cpu(), v.cpu(), s.cpu()),
              lambda: F.fused_packed_attention_backward(do, q, k, v, o, lse.half(), s),
              lambda: F.fused_packed_attention_backward(do, q, k, v, o, lse[:5], s),
              lambda: F.fused_packed_attention_backward(do[:5], q, k, v, o, lse, s),
              lambda: F.fused_packed_attention_backward(do, q, k, v, o[:, :2], lse, s)):
        with pytest.raises(BltError):
            f()
    for f in (lambda: F.fused_packed_attention(None, k, v, s),
              lambda: F.fused_packed_attention(q, k, v, [0, 10])):
        with pytest.raises(TypeError):
            f()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d,H,K", [(64, 4, 4), (128, 6, 2)])
@pytest.mark.parametrize("lens", [[40, 3], [130, 0], []])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 9), (False, 0)])
def test_lse_behind_the_last_sequence_with_out(dtype, d, H, K, lens, causal, window):
    """`out` keeps its rows there; lse, a tensor of the call's own, has -inf in all of them."""
    t, n, pad = TYPES[dtype], sum(lens), 200
    q, k, v, _ = made(lens, pad, H, K, d, t)
    st = starts_of(lens)
    used = [torch.full((n + pad, H), 7.0, device=DEV) for _ in range(8)]
    del used  # (memory that the call's tensors are likely to get)
    out = torch.full((n + pad, H, d), 7.0, dtype=t, device=DEV)
    kw = dict(causal=causal, window=window)
    o, lse = F.fused_packed_attention(q, k, v, i32(st), out=out, return_lse=True, **kw)
    assert o is out and bool((o[n:] == 7).all()) and bool((lse[n:] == -math.inf).all())
    r = R.attention(q, k, v, st, u=U[t], **kw)
    near(lse, r, "lse")
    near(o[:n], {x: r[x][:n] for x in ("o", "tol_o")}, "o")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T,H,K,d", [(100, 2, 2, 64), (70, 6, 2, 128), (9, 512, 512, 64)])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 20), (False, 0)])
def test_starts_that_do_not_ascend_write_nothing_beside_the_outputs(dtype, T, H, K, d, causal, window):
    """Through the C entries, whose outputs and workspaces are slices of larger buffers here."""
    L, t, edge = pkg.lib(), TYPES[dtype], 128
    q, k, v, do = (x.contiguous() for x in made([T], 0, H, K, d, t))
    code = 1 if t is torch.bfloat16 else 0

    def inside(shape, kind=t, fill=7):
        n = math.prod(shape)
        whole = torch.full((n + 2 * edge,), fill, dtype=kind, device=DEV)
        return whole, whole[edge:edge + n].view(shape)

    def heads(x):
        return x.data_ptr(), x.shape[1] * d, d

    for st in ([0, 70, 30, T], [-5, 1000], [50, 20], [T, T, 0], [0, 2 ** 31 - 1], [0, -2 ** 31, 5, 2 ** 31 - 1],
               [3] + [T - 1, 0] * 40):
        s, B = i32(st), len(st) - 1
        all_ = [inside((T, h, d)) for h in (H, H, K, K)] + [inside((T, H), torch.float32)]
        o, dq, dk, dv, lse = (x[1] for x in all_)
        stream = torch.cuda.current_stream().cuda_stream
        for bytes_, call in (
                (L.blt_packed_attention_workspace_bytes(B, T, H, K, code),
                 lambda ws, n: L.blt_packed_attention(
                     *heads(q), *heads(k), *heads(v), *heads(o), lse.data_ptr(), code, T, H, K, d, s.data_ptr(),
                     B, causal, window, d ** -0.5, 1, ws, n, stream)),
                (L.blt_packed_attention_backward_workspace_bytes(T, H, K, d, code),
                 lambda ws, n: L.blt_packed_attention_backward(
                     *heads(do), *heads(q), *heads(k), *heads(v), *heads(o), lse.data_ptr(), *heads(dq),
                     *heads(dk), *heads(dv), code, T, H, K, d, s.data_ptr(), B, causal, window, d ** -0.5, ws, n,
                     stream))):
            room = inside((bytes_,), torch.uint8)
            all_.append(room)
            assert call(room[1].data_ptr(), bytes_) == 0
        for whole, _ in all_:
            assert bool((whole[:edge] == 7).all() and (whole[-edge:] == 7).all()), st
        # (the tensors themselves are written whole)
        for x in (dq, dk, dv):
            assert not bool((x == 7).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d,H,K", [(64, 4, 2), (128, 8, 1)])
def test_out_may_be_q(dtype, d, H, K):
    lens = [300, 5, 0, 77]
    q, k, v, _ = made(lens, 9, H, K, d, TYPES[dtype])
    s, kept = i32(starts_of(lens)), q[sum(lens):].clone()
    want = F.fused_packed_attention(q, k, v, s, window=100)
    assert F.fused_packed_attention(q, k, v, s, window=100, out=q) is q
    assert torch.equal(q[:sum(lens)], want[:sum(lens)]) and torch.equal(q[sum(lens):], kept)
