"""Packed attention, token sampling and the shared prefix without a GPU: bad arguments end in a status
before anything is launched, and the workspaces hold what the launches lay out in them."""
import math

import pytest
import torch

import blt_burn_amd as pkg
from blt_burn_amd import fused_ops as F
from test_paged_host import L, P, addr, desc


def packed(backward=False, st=256, sh=64, dtype=1, total=100, H=4, Hkv=2, d=64, starts=P, B=2, causal=1,
           window=0, scale=0.125, x=None, lse=P, ws=P, size=1 << 40):
    """One call, with other pointers for some of its tensors (x)."""
    names = ("go", "q", "k", "v", "o") if backward else ("q", "k", "v", "o")
    x = x or {}
    at = lambda n: (x.get(n, P), st, sh)
    args = [a for n in names for a in at(n)] + [lse]
    if backward:
        args += [a for n in ("dq", "dk", "dv") for a in at(n)]
        return L.blt_packed_attention_backward(*args, dtype, total, H, Hkv, d, starts, B, causal, window,
                                               scale, ws, size, None)
    return L.blt_packed_attention(*args, dtype, total, H, Hkv, d, starts, B, causal, window, scale, 1, ws,
                                  size, None)


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("bad,word", [
    (dict(dtype=7), "dtype"), (dict(d=96), "head_dim"), (dict(Hkv=3), "multiple"), (dict(Hkv=0), "multiple"),
    (dict(H=0), "multiple"), (dict(H=65536), "65535"), (dict(B=-1), "int32"), (dict(total=-1), "int32"),
    (dict(total=2 ** 30), "int32"), (dict(total=2 ** 31), "int32"), (dict(window=-1), "window"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=math.nan), "scale"),
    (dict(scale=math.inf), "scale"), (dict(starts=None), "starts"), (dict(st=260), "aligned"),
    (dict(sh=68), "aligned"), (dict(st=-256), "strides"), (dict(st=(1 << 23) + 8), "strides"),
    (dict(sh=-64), "strides"), (dict(dtype=0, st=258), "aligned"), (dict(x=dict(q=None)), "null"),
    (dict(x=dict(v=P + 8)), "aligned"), (dict(x=dict(o=None)), "null")])
def test_bad_packed_calls_are_refused(backward, bad, word):
    assert packed(backward, **bad) < 0
    assert word in pkg.last_error(), pkg.last_error()


def test_packed_calls_without_tokens_and_their_workspaces():
    assert packed(total=0, starts=None, x=dict(q=None, k=None, v=None, o=None)) == 0
    assert packed(True, total=0, starts=None, lse=None, ws=None) == 0
    f = L.blt_packed_attention_workspace_bytes
    assert f(1, 1 << 20, 12, 12, 1) == 0  # one sequence: in the order of its tokens
    need = f(8, 16384, 12, 12, 1)
    assert need == 4 * 128 and f(8, 16384, 12, 12, 0) == 4 * 512
    assert packed(total=16384, H=12, Hkv=12, B=8, ws=None) < 0 and "workspace" in pkg.last_error()
    assert packed(total=16384, H=12, Hkv=12, B=8, size=need - 1) < 0 and "workspace" in pkg.last_error()
    assert packed(total=16384, H=12, Hkv=12, B=8, ws=P + 8) < 0 and "workspace" in pkg.last_error()
    # 512 key heads of two tokens are as many tiles
    assert f(2, 2, 512, 512, 1) == 4
    for bad in ((-1, 5, 4, 2, 1), (2, -1, 4, 2, 1), (2, 5, 4, 3, 1), (2, 1 << 31, 4, 2, 1), (2, 5, 0, 0, 1)):
        assert f(*bad) == 0


def test_gradient_workspaces():
    f = L.blt_packed_attention_backward_workspace_bytes
    order = 2 * 8192 * 4
    stats = lambda total, H, K: K * ((total * (H // K) + 63) // 64) * 512
    # many tiles: nothing but the rows' statistics and the orders
    assert f(100000, 12, 12, 64, 1) == stats(100000, 12, 12) + order
    # few: the parts of dk and dv of every block beside them
    for total, H, K, d, dtype in ((1000, 8, 1, 128, 1), (1000, 12, 4, 64, 1), (1000, 12, 4, 64, 0), (77, 4, 4, 128, 0)):
        more = f(total, H, K, d, dtype) - stats(total, H, K) - order
        part = total * K * 2 * d * 4
        assert more % part == 0 and 2 <= more // part <= 8
    for bad in ((5, 4, 3, 64, 1), (-1, 4, 2, 64, 1), (5, 4, 2, 96, 1), (5, 4, 2, 64, 9), (1 << 30, 4, 2, 64, 1)):
        assert f(*bad) == 0
    need = f(100, 4, 2, 64, 1)
    for kw in (dict(lse=None), dict(ws=None), dict(size=need - 1), dict(ws=P + 4), dict(sh=1 << 29)):
        assert packed(True, **kw) < 0
        assert "null" in pkg.last_error() or "workspace" in pkg.last_error() or "strides" in pkg.last_error()


def sample(x=P, stride=100, dtype=0, rows=4, vocab=100, u=P, t=1.0, ts=None, k=0, ks=None, p=1.0, ps=None,
           m=0.0, ms=None, out=P, ws=P, size=1 << 40):
    return L.blt_fused_sample(x, stride, dtype, rows, vocab, u, t, ts, k, ks, p, ps, m, ms, out, ws, size, None)


@pytest.mark.parametrize("bad,word", [
    (dict(dtype=5), "dtype"), (dict(rows=-1), "vocab"), (dict(vocab=0), "vocab"), (dict(vocab=(1 << 20) + 1), "vocab"),
    (dict(stride=-1), "stride"), (dict(t=-0.5), "temperature"), (dict(t=math.inf), "temperature"),
    (dict(t=math.nan), "temperature"), (dict(k=-1), "top_k"), (dict(p=0.0), "top_p"), (dict(p=math.nan), "top_p"),
    (dict(m=-0.1), "min_p"), (dict(m=1.1), "min_p"), (dict(m=math.nan), "min_p"), (dict(x=None), "null"),
    (dict(u=None), "null"), (dict(out=None), "null"), (dict(vocab=20000, ws=None), "workspace"),
    (dict(vocab=20000, size=100), "workspace"), (dict(vocab=20000, ws=P + 8), "workspace")])
def test_bad_sample_calls_are_refused(bad, word):
    assert sample(**bad) < 0
    assert word in pkg.last_error(), pkg.last_error()


def test_sample_workspaces():
    f = L.blt_fused_sample_workspace_bytes
    assert sample(rows=0, x=None) == 0
    assert f(100, 1) == f(1 << 20, 16384) == 0 < f(1, 16385)
    assert f(64, 131072) == 64 * f(1, 131072)
    # rows go in rounds, so it does not grow without end
    most = max(f(1 << 24, v) for v in (16385, 50000, 131072, 1 << 20))
    assert most < 350 << 20 and f(1 << 24, 131072) == f(1 << 30, 131072)
    assert f(-1, 20000) == f(4, 0) == f(4, (1 << 20) + 1) == 0


def test_bad_prefix_calls_are_refused():
    d = desc()
    call = lambda prefix, **kw: L.blt_paged_attention_prefix(
        addr(d), 0, P, 256, 64, P, 256, 64, kw.get("H", 4), P, None, kw.get("B", 1), kw.get("total", 1), 1, 0.125,
        prefix, kw.get("ws", P), kw.get("size", 1 << 40), None)
    assert call(None) < 0 and "prefix" in pkg.last_error()
    assert call(P, H=3) < 0 and call(P, B=-1) < 0 and call(P, total=-1) < 0
    for kw in (dict(ws=None), dict(size=16), dict(ws=P + 8)):
        assert call(P, **kw) < 0 and "workspace" in pkg.last_error()
    plain, shared = L.blt_paged_attention_workspace_bytes, L.blt_paged_attention_prefix_workspace_bytes
    for B, total in ((1, 1), (4, 4), (4, 400), (64, 64)):
        assert shared(addr(d), B, total, 4) > plain(addr(d), B, total, 4)
    assert shared(None, 1, 1, 4) == 0 and shared(addr(d), -1, 1, 4) == 0
    for args, word in (((None, -1, P), "entries"), ((None, 5, P), "entries"), ((P, 65537, P), "entries"),
                       ((P, 2, None), "null")):
        assert L.blt_cache_common_prefix(addr(d), *args, None) < 0 and word in pkg.last_error()


def test_host_tensors_are_refused():
    q, s = torch.zeros(3, 2, 64), torch.tensor([0, 3], dtype=torch.int32)
    for f in (lambda: F.fused_packed_attention(q, q, q, s),
              lambda: F.fused_packed_attention(q.requires_grad_(), q, q, s),
              lambda: F.fused_packed_attention_backward(q, q, q, q, q, q[..., 0], s),
              lambda: F.fused_sample(torch.zeros(2, 5), torch.zeros(2))):
        with pytest.raises(pkg.BltError):
            f()
    with pytest.raises(TypeError):
        F.fused_packed_attention([1], q, q, s)
    with pytest.raises(TypeError):
        F.fused_sample(None, torch.zeros(2))


@pytest.mark.parametrize("prefix", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim,rows", [(32, 8, 128, 16), (12, 12, 64, 3), (8, 1, 128, 64)])
def test_what_a_cache_keeps_for_its_calls_is_bounded(prefix, heads, kv_heads, dim, rows):
    """Calls that grow token by token: few workspaces, at most four times the largest call's need in all
    beside what calls without a prefix may take."""
    d = desc(n_kv_heads=kv_heads, head_dim=dim, max_seqs=64, max_pages=4096, num_pages=1 << 16)
    c = pkg.cache.PagedCache.__new__(pkg.cache.PagedCache)
    sizes = []
    c._lib, c._ptr, c.n_kv_heads = L, addr(d), kv_heads
    c._workspace = lambda n: sizes.append(n) or torch.empty(n, dtype=torch.uint8, device="meta")
    c._ws, c._wsp, c._ws_bytes, c._ws_for = [], None, 0, None
    f = L.blt_paged_attention_workspace_bytes
    c._ws_most = max(f(addr(d), 65536, 65536 * r, kv_heads) for r in (1, 32, 128))
    need, most = L.blt_paged_attention_prefix_workspace_bytes if prefix else f, 0
    for total in list(range(rows, 1500)) + list(range(1500, 8001, 7)):
        c._room(rows, total, heads, prefix)
        assert c._ws_bytes >= need(addr(d), rows, total, heads)
        most = max(most, need(addr(d), rows, total, heads))
        assert sum(sizes) <= 4 * most + 1.34 * c._ws_most, total
    assert len(sizes) <= 10 and len(c._ws) == len(sizes)
    # one large call alone takes what it needs
    c._ws, c._ws_bytes, sizes[:] = [], 0, []
    c._room(rows, 8000, heads, prefix)
    assert sizes == [need(addr(d), rows, 8000, heads)]


def test_forward_mode_is_refused():
    """A dual tensor needs no gradient, so its tangent would be dropped without a word."""
    import torch.autograd.forward_ad as fw
    q, s = torch.zeros(3, 2, 64), torch.tensor([0, 3], dtype=torch.int32)
    pos = torch.zeros(3, dtype=torch.int32)
    plan = F.RotaryPlan.__new__(F.RotaryPlan)
    x, w = torch.zeros(1, 2, 3, 64), torch.ones(64)
    with fw.dual_level():
        d, dx = fw.make_dual(q, torch.ones_like(q)), fw.make_dual(x, torch.ones_like(x))
        for f in (lambda: F.fused_packed_attention(d, q, q, s), lambda: F.fused_packed_attention(q, d, q, s),
                  lambda: F.fused_packed_attention(q, q, d, s),
                  lambda: F.fused_packed_attention_backward(d, q, q, q, q, q[..., 0], s),
                  lambda: F.fused_rotary(dx, None, pos, plan), lambda: F.fused_rotary(x, dx, pos, plan)):
            with pytest.raises(pkg.BltError, match="forward-mode"):
                f()
            with torch.no_grad(), pytest.raises(pkg.BltError, match="forward-mode"):
                f()


@pytest.mark.parametrize("dim,total", [(128, 1 << 25), (64, 1 << 26)])
def test_a_prefix_call_that_no_launch_holds_is_refused_whole(dim, total):
    """Its second launch would have 2^32 work-items: nothing of the first may run then."""
    d = desc(n_kv_heads=1, head_dim=dim, max_seqs=65536, max_pages=4096, num_pages=1 << 20)
    call = lambda n: L.blt_paged_attention_prefix(addr(d), 0, P, dim, dim, P, dim, dim, 1, P, None, 4, n, 1, 0.125,
                                                  P, P, 1 << 60, None)
    assert call(total) < 0 and "too many" in pkg.last_error(), pkg.last_error()
    assert call(2 ** 31 - 1) < 0 and "too many" in pkg.last_error()
