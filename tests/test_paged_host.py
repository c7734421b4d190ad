"""The incremental operators' refusals and host parts, without a GPU: every bad
argument is turned into a status before anything is launched."""
import ctypes

import numpy as np
import pytest
import torch

import blt_burn_amd as pkg
from blt_burn_amd import _lib
import paged_ref as R

L = pkg.lib()
P = 0x1000  # a pointer that is never followed: all of these calls end in a check


def desc(**kw):
    d = dict(k=P, v=P, page_table=P, lens=P, refcount=P, status=P, sync=P, dtype=1, n_layers=2, num_pages=8,
             n_kv_heads=4, page_size=16, head_dim=64, max_seqs=4, max_pages=8)
    d.update(kw)
    return _lib.PagedCacheDesc(**d)


def addr(s):
    return ctypes.addressof(s)


@pytest.mark.parametrize("bad,word", [
    (dict(dtype=7), "dtype"), (dict(head_dim=96), "head_dim"), (dict(page_size=24), "page_size"),
    (dict(page_size=4), "page_size"), (dict(page_size=2048), "page_size"),
    (dict(n_layers=0), "sizes"), (dict(num_pages=0), "sizes"), (dict(max_pages=1 << 21), "sizes"), (dict(max_seqs=65537), "sizes"),
    (dict(k=0), "null"), (dict(status=0), "null"), (dict(sync=0), "null"), (dict(v=P + 8), "aligned")])
def test_bad_caches_are_refused(bad, word):
    d = desc(**bad)
    calls = [lambda: L.blt_cache_reserve(addr(d), None, P, 1, None),
             lambda: L.blt_cache_trim(addr(d), None, None, 1, None, 0, None),
             lambda: L.blt_cache_fork(addr(d), P, P, 1, None),
             lambda: L.blt_cache_compact(addr(d), P, 1 << 20, None),
             lambda: L.blt_cache_copy_pages(addr(d), P, P, 1, None),
             lambda: L.blt_cache_append(addr(d), 0, P, 256, 64, P, 256, 64, None, 0, 0, None, 0, 0, 0,
                                        P, None, 1, 1, None, None),
             lambda: L.blt_paged_attention(addr(d), 0, P, 256, 64, P, 256, 64, 4, P, None, 1, 1, 1, 0,
                                           1.0, P, 1 << 40, None)]
    for f in calls:
        assert f() < 0
        assert word in pkg.last_error()


def test_bad_lists_and_workspaces_are_refused():
    d = desc()
    assert L.blt_cache_reserve(addr(d), P, P, 8193, None) == -2
    assert L.blt_cache_reserve(addr(d), P, None, 1, None) == -1
    assert L.blt_cache_reserve(addr(d), None, P, 5, None) == -2   # more than max_seqs
    assert L.blt_cache_trim(addr(d), P, P, 2, None, 0, None) == -1
    need = L.blt_cache_workspace_bytes(addr(d), 2)
    big = desc(num_pages=20000)
    assert need > 0 and L.blt_cache_workspace_bytes(addr(big), 0) > 0
    assert L.blt_cache_trim(addr(d), P, P, 2, P, need - 1, None) == -1
    assert L.blt_cache_trim(addr(d), P, P, 2, P + 4, need, None) == -1
    assert L.blt_cache_fork(addr(d), P, None, 2, None) == -1
    assert L.blt_cache_fork(addr(d), P, P, 8193, None) == -2
    assert L.blt_cache_compact(addr(big), None, 1 << 20, None) == -1
    assert L.blt_cache_copy_pages(addr(d), P, P, -1, None) == -2
    # nothing to do: no launch
    assert L.blt_cache_reserve(addr(d), None, None, 0, None) == 0
    assert L.blt_cache_trim(addr(d), None, None, 0, None, 0, None) == 0
    assert L.blt_cache_fork(addr(d), None, None, 0, None) == 0
    assert L.blt_cache_copy_pages(addr(d), None, None, 0, None) == 0


def attend(d, layer=0, q=P, st=256, sh=64, o=P, H=4, starts=P, B=1, total=1, window=0, scale=0.125,
           ws=P, wsb=1 << 40):
    return L.blt_paged_attention(addr(d), layer, q, st, sh, o, st, sh, H, starts, None, B, total, 1,
                                 window, scale, ws, wsb, None)


def test_bad_attention_calls_are_refused():
    d = desc()
    for kw, rc, word in [(dict(layer=2), -2, "layer"), (dict(layer=-1), -2, "layer"),
                         (dict(H=6), -2, "multiple"), (dict(H=0), -2, "multiple"),
                         (dict(window=-1), -2, "window"), (dict(scale=0.0), -2, "scale"),
                         (dict(scale=float("nan")), -2, "scale"), (dict(scale=1e-31), -2, "scale"),
                         (dict(scale=1e31), -2, "scale"), (dict(B=5), -2, "rows"),
                         (dict(B=70000), -2, "rows"), (dict(total=1 << 30), -2, "int32"),
                         (dict(starts=None), -1, "starts"), (dict(q=None), -1, "null"),
                         (dict(q=P + 2), -2, "aligned"), (dict(st=252), -2, "aligned")]:
        assert attend(d, **kw) == rc, kw
        assert word in pkg.last_error(), kw
    long = desc(max_pages=1 << 16)
    assert L.blt_paged_attention_workspace_bytes(addr(long), 1, 1, 4) > 0
    assert attend(long, ws=None) == -1 and "workspace" in pkg.last_error()
    for cache, B, total, H in ((None, 1, 1, 4), (desc(page_size=0), 1, 1, 4),
                               (desc(n_kv_heads=0), 1, 1, 4), (long, -1, 1, 4), (long, 1, -1, 4),
                               (long, 1, 1 << 40, 4), (long, 1 << 20, 1, 4), (long, 1, 1, 1 << 40)):
        assert L.blt_paged_attention_workspace_bytes(cache and addr(cache), B, total, H) == 0
    assert attend(d, B=0) == 0 and attend(d, total=0) == 0


def test_bad_append_and_rotary_calls_are_refused():
    d = desc()
    r = _lib.Rotary(P, 64, 0, 1.0)

    def append(k=P, layer=0, q=None, qo=None, Hq=0, B=1, total=1, rot=None):
        return L.blt_cache_append(addr(d), layer, k, 256, 64, P, 256, 64, q, 256, 64, qo, 256, 64, Hq,
                                  P, None, B, total, rot, None)
    assert append(k=None) == -1
    assert append(layer=5) == -2
    assert append(q=P, qo=P, Hq=4) == -1 and "rotary" in pkg.last_error()
    assert append(q=P, qo=None, Hq=4, rot=addr(r)) == -1
    assert append(B=5) == -2
    assert append(B=0) == 0 and append(total=0) == 0
    for bad in (_lib.Rotary(0, 64, 0, 1.0), _lib.Rotary(P, 63, 0, 1.0), _lib.Rotary(P, 128, 0, 1.0)):
        assert append(rot=addr(bad)) < 0

    def rotary(q=P, k=P, dt=1, B=1, T=4, H=2, d=64, pos=P, r=r):
        return L.blt_fused_rotary(q, k, P, P, dt, B, H, H, T, d, *([64] * 12), pos, 0, addr(r), 0, None)
    assert rotary(dt=3) == -1
    assert rotary(d=65) == -2 and rotary(d=1024) == -2
    assert rotary(T=1 << 31) == -2 and rotary(H=40000) == -2
    assert rotary(q=None) == -1 and rotary(pos=None) == -1
    assert rotary(d=32) == -2                       # rotary_dim 64 of 32
    assert rotary(B=0) == 0 and rotary(T=0) == 0


def freqs(rot, theta=10000.0, scaling=0, factor=1.0, original=8192.0):
    f, mag = np.zeros(max(rot // 2, 1), np.uint64), ctypes.c_float()
    rc = L.blt_rotary_frequencies(rot, theta, scaling, factor, original, f.ctypes.data,
                                  ctypes.addressof(mag))
    return rc, f, mag.value


@pytest.mark.parametrize("rot", [2, 16, 64, 128])
@pytest.mark.parametrize("name,factor", [("none", 1.0), ("linear", 4.0), ("ntk", 8.0),
                                         ("yarn", 16.0), ("yarn", 1.0)])
def test_frequencies(rot, name, factor):
    if name == "ntk" and rot == 2:
        assert freqs(rot, scaling=2, factor=factor)[0] == -2
        return
    rc, f, mag = freqs(rot, scaling=_lib.ROTARY_SCALING[name], factor=factor)
    want, m = R.frequencies(rot, scaling=name, factor=factor)
    assert rc == 0
    # 2^-64 of a turn, and the reference's own 64-bit arithmetic (a few 2^-53)
    np.testing.assert_allclose(f.astype(np.float64) / 2.0 ** 64 * 2 * np.pi, want, rtol=1e-14,
                               atol=2.0 ** -60)
    assert abs(mag - m) <= 2 ** -23 * m


def test_bad_frequencies_are_refused():
    for kw in (dict(rot=3), dict(rot=0), dict(rot=514), dict(rot=64, theta=1.0),
               dict(rot=64, theta=float("nan")), dict(rot=64, scaling=4), dict(rot=64, scaling=1, factor=0.5),
               dict(rot=64, scaling=3, factor=2.0, original=0.0)):
        assert freqs(**kw)[0] < 0, kw


def test_host_tensors_are_refused():
    from blt_burn_amd import cache, fused_ops as F
    with pytest.raises(pkg.BltError):
        cache.PagedCache.wrap(*(torch.zeros(1) for _ in range(5)))
    with pytest.raises(pkg.BltError):
        F.fused_rotary(torch.zeros(1, 1, 1, 64), None, torch.zeros(1, dtype=torch.int32), None)
    with pytest.raises(pkg.BltError):
        F.RotaryPlan(64, pairs="other")
    with pytest.raises(pkg.BltError):
        F.RotaryPlan(64, scaling="other")


def test_host_pool_model():
    # the host model itself, by hand: page size 8
    k = np.arange(1 * 6 * 1 * 8 * 2, dtype=np.float64).reshape(1, 6, 1, 8, 2)
    p = R.Pool(k, -k, np.full((3, 3), -1), np.zeros(3, int), np.zeros(6, int))
    assert p.reserve([0], [12]) and p.table[0, :2].tolist() == [0, 1] and p.lens[0] == 12
    assert p.fork([0, 0], [1, 2])
    assert p.table[1, :2].tolist() == [0, 2] and p.table[2, :2].tolist() == [0, 3]
    assert p.refs.tolist() == [3, 1, 1, 1, 0, 0]
    assert (p.k[0, 2, 0, :4] == k[0, 1, 0, :4]).all() and (p.k[0, 2, 0, 4:] == k[0, 2, 0, 4:]).all()
    assert p.trim([1], [3]) and p.refs.tolist() == [2, 1, 1, 1, 0, 0] and p.table[1, 0] == 2
    assert p.trim([0], [0]) and p.refs.tolist() == [1, 0, 1, 1, 0, 0]
    p.compact()
    assert p.refs.tolist() == [1, 1, 1, 0, 0, 0] and p.table[2, :2].tolist() == [0, 1]
    assert not p.reserve([0], [8 * 4])


def test_the_largest_calls_need_the_most_workspace():
    """What PagedCache allocates (the largest call of every form) covers every call."""
    rng = np.random.default_rng(0)
    for _ in range(3000):
        K, d, dtype = int(rng.choice([1, 2, 4, 8, 12])), int(rng.choice([64, 128])), int(rng.integers(2))
        c = desc(dtype=dtype, n_kv_heads=K, head_dim=d, page_size=int(rng.choice([8, 64, 1024])),
                 max_pages=int(rng.choice([1, 3, 40, 5000])), max_seqs=65536)
        size = lambda B, total, H: L.blt_paged_attention_workspace_bytes(addr(c), B, total, H)
        most = max(size(65536, 65536 * rows, K) for rows in (1, 32, 128))
        B, G = int(rng.choice([1, 2, 20, 70, 300, 65536])), int(rng.choice([1, 2, 4, 7]))
        assert size(B, B * int(rng.choice([1, 2, 7, 33, 64, 65, 200])), K * G) <= most
