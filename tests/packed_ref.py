"""Attention over packed sequences and its gradient, restated in 64 bits on the CPU, with bounds on
the error of a computation that rounds to a type of half a step u where the kernels do."""
import math

import torch


def attention(q, k, v, starts, causal=True, window=0, scale=None, do=None, u=2.0 ** -24):
    """dict of o, lse (dq, dk, dv) and, under "tol_" + name, the bounds on their errors.

    w is what f32 work costs, relative to a weight: a score is off by (d + 4) u32 of sum |q k| scale,
    twice for the sum, its exponential and the arguments by 8 u32 (1 + |score| + |lse|), sums over n
    keys by n u32.
      o   weights of type u in the numerator and, at most, in the sum (2 u), its own rounding
          (u): (3 u + w) A, A = sum p |v|
      dv  weights (u), its own rounding (u): (2 u + w) sum p |do|
      D   o's error (3 u + w) times |do|, summed: E;  dS = p (dP - D) is off by
          p E + p w (sum |do v| + sum |do o|) and its rounding u |dS| (with w)
      dq  scale sum |k| dS's error, and its own rounding u; dk alike"""
    q, k, v = (x.detach().double().cpu() for x in (q, k, v))
    T, H, d = q.shape
    K = k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    r = dict(o=torch.zeros_like(q), lse=torch.full((T, H), -math.inf, dtype=torch.float64))
    r["tol_o"], r["tol_lse"] = torch.zeros_like(q), torch.zeros_like(r["lse"])
    if do is not None:
        do = do.detach().double().cpu()
        for n, x in (("dq", q), ("dk", k), ("dv", v)):
            r[n], r["tol_" + n] = torch.zeros_like(x), torch.zeros_like(x)
    e = 2.0 ** -24
    for a, b in zip(starts[:-1], starts[1:]):
        n = b - a
        i = torch.arange(n)
        hide = torch.zeros(n, n, dtype=torch.bool)
        if causal:
            hide = i[None] > i[:, None]
            if window:
                hide |= i[None] <= i[:, None] - window
        for h in range(H if n else 0):
            qh, kh, vh = q[a:b, h], k[a:b, h // (H // K)], v[a:b, h // (H // K)]
            s = (qh @ kh.T * scale).masked_fill(hide, -math.inf)
            lse = torch.logsumexp(s, -1, keepdim=True)
            p = torch.exp(s - lse)
            o = p @ vh
            size = (qh.abs() @ kh.abs().T * scale).masked_fill(hide, 0)
            w = e * (2 * (d + 4) * size.amax(-1, keepdim=True)
                     + 8 * (1 + s.masked_fill(hide, 0).abs().amax(-1, keepdim=True) + lse.abs()) + n)
            A = p @ vh.abs()
            tol = (3 * u + w) * A
            r["o"][a:b, h], r["lse"][a:b, h] = o, lse[:, 0]
            r["tol_o"][a:b, h], r["tol_lse"][a:b, h] = tol, w[:, 0]
            if do is None:
                continue
            g, kv = do[a:b, h], h // (H // K)
            dp = g @ vh.T
            D = (g * o).sum(-1, keepdim=True)
            ds = p * (dp - D)
            E = (g.abs() * tol).sum(-1, keepdim=True)
            both = g.abs() @ vh.abs().T + (g * o).abs().sum(-1, keepdim=True)
            err = p * E + p * w * both + (u + w) * ds.abs()
            r["dq"][a:b, h] = scale * ds @ kh
            r["tol_dq"][a:b, h] = scale * err @ kh.abs() + u * r["dq"][a:b, h].abs()
            r["dk"][a:b, kv] += scale * ds.T @ qh
            r["tol_dk"][a:b, kv] += scale * err.T @ qh.abs()
            r["dv"][a:b, kv] += p.T @ g
            r["tol_dv"][a:b, kv] += ((u + w) * p).T @ g.abs()
    if do is not None:
        # sums over a key's rows (up to n H / K of them) and the outputs' own rounding
        n = max([b - a for a, b in zip(starts[:-1], starts[1:])] + [0]) * (H // K) * e
        for x in ("dk", "dv"):
            r["tol_" + x] = r["tol_" + x] * (1 + n) + (u + n) * r[x].abs()
    return r
