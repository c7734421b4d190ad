"""Tokens drawn from logits on the GPU against the definition in 64 bits, token for token: a
running sum is off by less than vocab 2^-42 of the largest weight, so the chance that a random
number falls between the two is below 2^-20 for all rows here together, and none does."""
import math

import numpy as np
import pytest
import torch

from blt_burn_amd import BltError, fused_ops as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def reference(logits, u, t=1.0, k=0, p=1.0, m=0.0):
    """Tokens of rows [R, V] (settings: numbers or one for each row)."""
    x, u = logits.double().cpu().numpy(), u.double().cpu().numpy()
    R, V = x.shape
    t, k, p, m = (np.broadcast_to(np.asarray(s, np.float64), (R,)) for s in (t, k, p, m))
    out = np.full(R, -1)
    for r in range(R):
        row = x[r]
        if np.isnan(row).any() or row.max() == -np.inf:
            continue
        if not (0 <= t[r] < np.inf and k[r] >= 0 and p[r] > 0 and 0 <= m[r] <= 1):
            continue
        order = np.argsort(-row, kind="stable")
        if t[r] == 0:
            out[r] = order[0]
            continue
        if k[r] > 0:
            order = order[:int(k[r])]
        y = row[order]
        with np.errstate(invalid="ignore"):
            w = np.where(y == y[0], 1.0, np.exp((y - y[0]) / t[r]))
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        keep = w >= m[r]
        if p[r] < 1:
            keep &= (before < p[r] * w.sum()) | (np.arange(len(w)) == 0)
        mass = np.zeros(V)
        mass[order[keep]] = w[keep]
        run = np.cumsum(mass)
        out[r] = np.argmax(run > u[r] * run[-1])
    return torch.from_numpy(out.astype(np.int32))


def logits_of(R, V, dtype, seed=0, spread=3.0):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    x = spread * torch.randn(R, V, generator=g, device=DEV)
    return x.to(dtype), torch.rand(R, generator=g, device=DEV)


SETTINGS = [dict(), dict(t=0.7), dict(t=0.0), dict(k=1), dict(k=7), dict(k=50, t=1.5), dict(p=0.9),
            dict(p=0.5, t=0.6), dict(p=1e-9), dict(m=0.05), dict(m=1.0), dict(k=40, p=0.95, m=0.02),
            dict(k=10 ** 9, p=0.999999), dict(k=200, p=0.3, t=2.0), dict(t=30.0, p=0.8)]


def names(s):
    return {dict(t="temperature", k="top_k", p="top_p", m="min_p")[a]: b for a, b in s.items()}


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V,R", [(1, 5), (2, 9), (63, 20), (64, 20), (65, 20), (260, 300), (321, 9),
                                 (513, 9), (1000, 9), (1024, 9), (1025, 9), (4097, 9), (8200, 5),
                                 (16384, 5), (16385, 5), (50001, 4), (131072, 3), (1 << 20, 1)])
def test_sample(dtype, V, R):
    x, u = logits_of(R, V, TYPES[dtype], seed=V)
    for s in SETTINGS:
        got = F.fused_sample(x, u, **names(s))
        assert got.dtype == torch.int32 and got.shape == (R,)
        assert torch.equal(got.cpu(), reference(x, u, **s)), s


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [260, 3000, 40000])
def test_a_setting_for_each_row(dtype, V):
    R = 24
    x, u = logits_of(R, V, TYPES[dtype], seed=1)
    rng = np.random.default_rng(2)
    t = rng.choice([0.0, 0.5, 1.0, 2.0], R).astype(np.float32)
    k = rng.choice([0, 1, 5, 100, 10 ** 6], R).astype(np.int32)
    p = rng.choice([0.2, 0.9, 1.0, 3.0], R).astype(np.float32)
    m = rng.choice([0.0, 0.1, 1.0], R).astype(np.float32)
    t[3], t[4], k[5], p[6], p[7], m[8], m[9] = -1, math.nan, -2, 0, math.nan, 1.5, math.nan
    dev = [torch.from_numpy(a).to(DEV) for a in (t, k, p, m)]
    got = F.fused_sample(x, u, *dev).cpu()
    assert torch.equal(got, reference(x, u, t, k, p, m))
    assert bool((got[3:10] == -1).all()) and bool((got[10:] >= 0).all())


# ---- ties, masks, values that are not finite ----------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [70, 260, 1024, 5000, 16384, 70000])
def test_equal_logits(dtype, V):
    """Rows of one value, of two, of a few: ranks of equal logits go by index, and sums are exact."""
    R = 12
    g = torch.Generator(device=DEV)
    g.manual_seed(V)
    x = torch.zeros(R, V, device=DEV)
    x[4:8] = torch.randint(0, 2, (4, V), generator=g, device=DEV).float()
    x[8:] = torch.randint(0, 5, (4, V), generator=g, device=DEV).float() / 4
    x = x.to(TYPES[dtype])
    u = torch.rand(R, generator=g, device=DEV)
    u[0], u[1], u[4] = 0, 1 - 2.0 ** -24, 0
    for s in (dict(), dict(k=3), dict(k=V - 1), dict(k=V // 2, p=0.5), dict(p=0.25), dict(p=0.5),
              dict(k=V // 3, p=0.7, t=0.5), dict(m=1.0), dict(m=0.9, p=0.99)):
        assert torch.equal(F.fused_sample(x, u, **names(s)).cpu(), reference(x, u, **s)), s
    # exactly on the border: u n of n equal tokens is the n-th, top_p 1/2 of four the first two
    four = torch.full((4, V), -math.inf, device=DEV).to(TYPES[dtype])
    four[:, [5, 17, 40, 69]] = 2.0
    u = torch.tensor([0.0, 0.25, 0.5, 0.75], device=DEV)
    assert F.fused_sample(four, u).tolist() == [5, 17, 40, 69]
    assert F.fused_sample(four, u, top_p=0.5).tolist() == [5, 5, 17, 17]
    assert F.fused_sample(four, u, top_k=1).tolist() == [5] * 4
    assert F.fused_sample(four, u, temperature=0).tolist() == [5] * 4


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [260, 4000, 33000])
def test_masks_and_values_that_are_not_finite(dtype, V):
    inf, nan = math.inf, math.nan
    x, u = logits_of(16, V, TYPES[dtype], seed=3)
    x[0] = -inf                      # nothing left
    x[1] = -inf
    x[1, V - 1] = -5                 # one left
    x[2, ::2] = -inf
    x[3, 7] = nan
    x[4, 9] = inf                    # takes everything
    x[5, 9] = x[5, V // 2] = inf
    x[6] = -inf
    x[6, 3] = nan
    x[7] = torch.finfo(x.dtype).min  # the type's lowest value is a value
    x[8] = torch.finfo(x.dtype).min
    x[8, 11] = 0
    x[9] = torch.finfo(x.dtype).max
    x[10, :5] = -0.0
    x[10, 5:] = 0.0
    x[11] = inf
    for s in (dict(), dict(t=0.0), dict(k=5), dict(p=0.9), dict(k=V - 2, p=0.5, m=0.01), dict(m=1.0),
              dict(t=1e-30), dict(t=1e30, p=0.9)):
        got = F.fused_sample(x, u, **names(s)).cpu()
        assert torch.equal(got, reference(x, u, **s)), s
        assert got[[0, 3, 6]].tolist() == [-1] * 3 and int(got[1]) == V - 1 and int(got[4]) == 9
        assert int(got[8]) == 11
    un = u.clone()
    un[2] = nan
    got = F.fused_sample(x, un).cpu()
    assert int(got[2]) == -1 and torch.equal(got[3:], F.fused_sample(x, u).cpu()[3:])


@pytest.mark.parametrize("V", [260, 2048, 20000])
def test_many_tokens_between_two_bins(V):
    """Logits within few steps of each other, or on both sides of 0, over many orders."""
    g = torch.Generator(device=DEV)
    g.manual_seed(V)
    R = 6
    near = 1 + 2.0 ** -23 * torch.randint(0, 9000, (R, V), generator=g, device=DEV)
    tiny = torch.randn(R, V, generator=g, device=DEV) * 10.0 ** -(
        40 * torch.rand(R, V, generator=g, device=DEV))
    wide = torch.randn(R, V, generator=g, device=DEV) * 1e4
    u = torch.rand(R, generator=g, device=DEV)
    for x in (near, tiny, wide):
        for s in (dict(k=V // 2), dict(p=0.5), dict(k=V // 3, p=0.9), dict(k=17, t=1e-3),
                  dict(p=0.7, t=3e3)):
            assert torch.equal(F.fused_sample(x, u, **names(s)).cpu(), reference(x, u, **s)), s


@pytest.mark.parametrize("V", [300, 2000, 20000])
@pytest.mark.parametrize("t", [1e-6, 1e-300, 5e-324, 1e30, 1e300])
def test_extreme_temperatures(V, t):
    """Only the largest logits are left, or all are alike."""
    x, u = logits_of(6, V, torch.float32, seed=V)
    x[:3, V // 3] = x[:3, V // 2] = x[:3].amax(1) + 1  # (two largest ones)
    for s in (dict(t=t), dict(t=t, p=0.7), dict(t=t, k=5, m=0.1)):
        assert torch.equal(F.fused_sample(x, u, **names(s)).cpu(), reference(x, u, **s)), s


def test_more_rows_than_one_round_of_launches():
    """Rows of 17000 tokens are in two parts, 4096 rows a round: each row as in a call of its own."""
    n, V = 4100, 17000
    x, u = logits_of(n, V, torch.bfloat16, seed=8)
    t = torch.rand(n, device=DEV) + 0.5
    k = torch.arange(n, dtype=torch.int32, device=DEV) % 60
    p, m = 1 - 0.5 * torch.rand(n, device=DEV), 0.01 * torch.rand(n, device=DEV)
    got = F.fused_sample(x, u, t, k, p, m)
    for rows in (slice(0, 40), slice(4080, 4100)):
        want = reference(x[rows], u[rows], *(y[rows].double().cpu().numpy() for y in (t, k, p, m)))
        assert torch.equal(got[rows].cpu(), want)
        assert torch.equal(got[rows], F.fused_sample(x[rows], u[rows], t[rows], k[rows], p[rows],
                                                     m[rows]))


def test_all_tokens_in_turn():
    """u over a fine grid draws every kept token as often as its weight says."""
    x, _ = logits_of(1, 260, torch.float32, seed=9, spread=1.0)
    n = 1 << 14
    u = (torch.arange(n, device=DEV) + 0.5) / n
    got = F.fused_sample(x.expand(n, -1), u, top_p=0.8).cpu()
    assert torch.equal(got, reference(x.cpu().expand(n, -1), u, p=0.8))
    assert bool((got[1:] >= got[:-1]).all())
    y = x.double().cpu()[0]
    w = torch.softmax(y, 0)
    order = torch.argsort(y, descending=True, stable=True)
    c = w[order].cumsum(0)
    keep = order[(c - w[order]) < 0.8]
    share = torch.zeros(260, dtype=torch.float64)
    share[keep] = w[keep] / w[keep].sum()
    assert (torch.bincount(got.long(), minlength=260) - n * share).abs().max() <= 2


# ---- layouts, graphs, refusals --------------------------------------------------------------

@pytest.mark.parametrize("V", [260, 3000, 20000])
def test_layouts_and_out(V):
    x, u = logits_of(6, V + 9, torch.bfloat16, seed=4)
    want = reference(x[:, 3:V + 3], u, k=20)
    got = F.fused_sample(x[:, 3:V + 3], u, top_k=20)  # rows of a wider tensor, any alignment
    assert torch.equal(got.cpu(), want)
    y = x[:, 3:V + 3].contiguous()
    assert torch.equal(F.fused_sample(y.view(2, 3, V), u.view(2, 3), top_k=20).cpu(),
                       want.view(2, 3))
    assert torch.equal(F.fused_sample(y.t().contiguous().t(), u, top_k=20).cpu(), want)
    assert int(F.fused_sample(y[0], u[0], top_k=20)) == int(want[0])
    assert torch.equal(F.fused_sample(x[::2, 3:V + 3], u[::2], top_k=20).cpu(), want[::2])
    out = torch.full((6,), 7, dtype=torch.int32, device=DEV)
    assert F.fused_sample(y, u, top_k=20, out=out) is out and torch.equal(out.cpu(), want)
    assert F.fused_sample(y[:0], u[:0]).shape == (0,)
    one = F.fused_sample(y[:1].expand(6, -1), u)  # one row for all
    assert torch.equal(one.cpu(), reference(y[:1].expand(6, -1), u))


def test_rows_past_32_bits():
    """A row stride that takes rows past 2^32 bytes."""
    big = torch.empty(3 << 30, dtype=torch.bfloat16, device=DEV)
    x, u = logits_of(3, 300, torch.bfloat16)
    v = big.as_strided((3, 300), ((1 << 30) + 17, 1))
    v.copy_(x)
    assert torch.equal(F.fused_sample(v, u), F.fused_sample(x, u))


@pytest.mark.parametrize("V", [260, 3000, 20000])
def test_in_a_graph_and_on_another_stream(V):
    x, u = logits_of(8, V, torch.float32, seed=5)
    t = torch.full((8,), 0.8, device=DEV)
    s = dict(temperature=t, top_p=0.9, top_k=60)
    want = F.fused_sample(x, u, **s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = F.fused_sample(x, u, **s)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = F.fused_sample(x, u, **s)
    for _ in range(4):
        x.normal_(0, 3)
        u.uniform_()
        want = F.fused_sample(x, u, **s)
        torch.cuda.synchronize()
        graph.replay()
        assert torch.equal(held, want)


def test_refusals():
    x, u = logits_of(4, 260, torch.float32)
    for f in (lambda: F.fused_sample(x.half(), u), lambda: F.fused_sample(x.cpu(), u),
              lambda: F.fused_sample(x, u[:3]), lambda: F.fused_sample(x, u.double()),
              lambda: F.fused_sample(x, u.cpu()), lambda: F.fused_sample(x[:, :0], u),
              lambda: F.fused_sample(x, u, temperature=-1), lambda: F.fused_sample(x, u, temperature=math.inf),
              lambda: F.fused_sample(x, u, temperature=math.nan), lambda: F.fused_sample(x, u, top_k=-1),
              lambda: F.fused_sample(x, u, top_p=0.0), lambda: F.fused_sample(x, u, top_p=math.nan),
              lambda: F.fused_sample(x, u, min_p=1.1), lambda: F.fused_sample(x, u, min_p=-0.1),
              lambda: F.fused_sample(x, u, temperature=u.double()),
              lambda: F.fused_sample(x, u, top_k=u), lambda: F.fused_sample(x, u, top_p=u[:2]),
              lambda: F.fused_sample(x, u, out=torch.empty(4, device=DEV)),
              lambda: F.fused_sample(x, u, out=torch.empty(8, dtype=torch.int32, device=DEV)[::2])):
        with pytest.raises(BltError):
            f()
    for f in (lambda: F.fused_sample(None, u), lambda: F.fused_sample(x, 0.5),
              lambda: F.fused_sample(x, u, out=[0])):
        with pytest.raises(TypeError):
            f()


@pytest.mark.parametrize("V,R", [(2000, (1 << 22) + 5), (40, (1 << 26) + 9)])
def test_more_rows_than_one_launch_holds(V, R):
    """Many tokens from one distribution: a launch has at most 2^32 - 1 work-items."""
    x, _ = logits_of(1, V, torch.float32, seed=7)
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    u = torch.rand(R, generator=g, device=DEV)
    got = F.fused_sample(x.expand(R, -1), u, top_k=30, top_p=0.9)
    s = dict(k=30, p=0.9)
    for rows in (slice(0, 50), slice(R // 2 - 25, R // 2 + 25), slice(R - 50, R)):
        assert torch.equal(got[rows].cpu(), reference(x.expand(50, -1), u[rows], **s))
    assert bool((got >= 0).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", [300, 2000, 20000])
@pytest.mark.parametrize("t", [3e37, 1e38, 3e38, 1e39])
def test_logits_further_apart_than_their_type_reaches(dtype, V, t):
    """max - x passes the largest f32, the weight at that temperature does not vanish."""
    g = torch.Generator(device=DEV)
    g.manual_seed(V)
    x = (6.6e38 * (torch.rand(6, V, generator=g, device=DEV, dtype=torch.float64) - 0.5)).to(TYPES[dtype])
    assert bool((x.amax(1) - x.amin(1) == math.inf).all())
    u = torch.rand(6, generator=g, device=DEV)
    for s in (dict(t=t), dict(t=t, p=0.95), dict(t=t, k=V // 2), dict(t=t, k=V - 3, p=0.9, m=1e-3)):
        assert torch.equal(F.fused_sample(x, u, **names(s)).cpu(), reference(x, u, **s)), s


@pytest.mark.parametrize("dtype,step,temperatures", [("f32", 2.0 ** -149, (1e-44, 1e-43, 3e-42)),
                                                     ("bf16", 2.0 ** -133, (1e-40, 1e-39, 2e-38))])
@pytest.mark.parametrize("V", [300, 2000, 20000])
def test_logits_closer_than_their_type_inverts(dtype, step, temperatures, V):
    """Logits a few of the type's smallest steps apart, temperatures whose inverses pass the largest f32."""
    g = torch.Generator(device=DEV)
    g.manual_seed(V)
    x = (step * torch.randint(-40, 40, (6, V), generator=g, device=DEV).double()).to(TYPES[dtype])
    u = torch.rand(6, generator=g, device=DEV)
    assert len(x.unique()) == 80
    for t in temperatures:
        for s in (dict(t=t), dict(t=t, p=0.95), dict(t=t, k=V // 2), dict(t=t, k=V - 3, p=0.9, m=1e-3)):
            assert torch.equal(F.fused_sample(x, u, **names(s)).cpu(), reference(x, u, **s)), s
