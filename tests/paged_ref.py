"""Plain restatements of the incremental operators in 64-bit numpy, a sequence at
a time, and a host model of the paged cache's bookkeeping."""
import math

import numpy as np


def frequencies(rot, theta=10000.0, scaling="none", factor=1.0, original=8192):
    i = np.arange(rot // 2, dtype=np.float64)
    f = theta ** (-2 * i / rot)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "ntk":
        return (theta * factor ** (rot / (rot - 2))) ** (-2 * i / rot), 1.0
    if scaling == "yarn":
        def pair(beta):
            return rot * math.log(original / (beta * 2 * math.pi)) / (2 * math.log(theta))
        lo, hi = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), rot - 1)
        ramp = np.clip((i - lo) / max(hi - lo, 0.001), 0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1
    return f, 1.0


def rotate(x, pos, f, mag, pairs, backward=False):
    """x [..., T, d], pos [T] (or broadcast over the leading axes)."""
    half = len(f)
    a = np.asarray(pos, np.float64)[..., None] * f * (-1 if backward else 1)
    c, s = np.cos(a) * mag, np.sin(a) * mag
    y = x.astype(np.float64).copy()
    i = np.arange(half)
    p, q = (i, i + half) if pairs == "half" else (2 * i, 2 * i + 1)
    y[..., p], y[..., q] = x[..., p] * c - x[..., q] * s, x[..., p] * s + x[..., q] * c
    return y


def attention(q, keys, values, length, causal=True, window=0, scale=None):
    """q [n, H, d], keys / values [length, Hkv, d], the n tokens the last ones:
    (out, sum p |v|), a row that sees nothing 0."""
    n, H, d = q.shape
    G = H // keys.shape[1]
    scale = d ** -0.5 if scale is None else scale
    out, mag = np.zeros((n, H, d)), np.zeros((n, H, d))
    pos = length - n + np.arange(n)
    j = np.arange(length)
    see = np.ones((n, length), bool)
    if causal:
        see = j[None] <= pos[:, None]
        if window:
            see &= j[None] > pos[:, None] - window
    any_ = see.any(1)
    for h in range(H):
        if length == 0:
            break
        s = np.where(see, q[:, h].astype(np.float64) @ keys[:, h // G].T.astype(np.float64) * scale,
                     -np.inf)
        p = np.exp(s - np.where(any_, s.max(1), 0)[:, None])
        p /= np.where(any_, p.sum(1), 1)[:, None]
        v = values[:, h // G].astype(np.float64)
        out[:, h], mag[:, h] = p @ v, p @ np.abs(v)
    return out, mag


class Pool:
    """The cache's bookkeeping and page contents on the host."""

    def __init__(self, k, v, table, lens, refs):
        self.k, self.v = k.copy(), v.copy()
        self.table, self.lens, self.refs = table.copy(), lens.copy(), refs.copy()
        self.page = k.shape[3]

    def _free(self, n):
        got = np.flatnonzero(self.refs == 0)[:n]
        return got if len(got) == n else None

    def reserve(self, seqs, counts):
        want = []
        for s, c in zip(seqs, counts):
            a, b = -(-self.lens[s] // self.page), -(-(self.lens[s] + c) // self.page)
            want += [(s, col) for col in range(a, b)]
        got = self._free(len(want))
        if got is None:
            return False
        for (s, col), p in zip(want, got):
            self.table[s, col] = p
            self.refs[p] = 1
        for s, c in zip(seqs, counts):
            self.lens[s] += c
        return True

    def fork(self, src, dst):
        part = [i for i, a in enumerate(src) if self.lens[a] % self.page]
        got = self._free(len(part))
        if got is None:
            return False
        for i, p in zip(part, got):
            a, col = src[i], self.lens[src[i]] // self.page
            fill = self.lens[a] % self.page
            for x in (self.k, self.v):
                x[:, p, :, :fill] = x[:, self.table[a, col], :, :fill]
            self.table[dst[i], col] = p
            self.refs[p] = 1
        for a, b in zip(src, dst):
            full = self.lens[a] // self.page
            self.table[b, :full] = self.table[a, :full]
            np.add.at(self.refs, self.table[a, :full], 1)
            self.lens[b] = self.lens[a]
        return True

    def trim(self, seqs, lens):
        for s, n in zip(seqs, lens):
            if n < self.lens[s]:
                a, b = -(-n // self.page), -(-self.lens[s] // self.page)
                np.subtract.at(self.refs, self.table[s, a:b], 1)
                self.lens[s] = n
        split = []
        for s in dict.fromkeys(seqs):
            n = self.lens[s]
            if n % self.page and self.refs[self.table[s, n // self.page]] > 1:
                split.append(s)
        got = np.flatnonzero(self.refs == 0)[:len(split)]
        for i, s in enumerate(split):
            n = self.lens[s]
            col, fill = n // self.page, n % self.page
            old = self.table[s, col]
            self.refs[old] -= 1
            if i < len(got):
                self.refs[got[i]] = 1
                self.table[s, col] = got[i]
                for x in (self.k, self.v):
                    x[:, got[i], :, :fill] = x[:, old, :, :fill]
            else:
                self.lens[s] = n - fill
        return len(got) == len(split)

    def compact(self):
        live = int((self.refs > 0).sum())
        at = np.arange(len(self.refs))
        movers = at[(self.refs > 0) & (at >= live)]
        holes = at[(self.refs == 0) & (at < live)]
        to = at.copy()
        to[movers] = holes
        self.k[:, holes], self.v[:, holes] = self.k[:, movers], self.v[:, movers]
        self.refs[holes] = self.refs[movers]
        self.refs[movers] = 0
        for s, n in enumerate(self.lens):
            cols = -(-n // self.page)
            self.table[s, :cols] = to[self.table[s, :cols]]
