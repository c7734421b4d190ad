"""Operators of prompts, their continuations and their answers as timed cases, each
beside its plain form.

  prompt    fused_packed_attention: attention over whole prompts of different
            lengths packed behind each other, grouped heads
  train     the same with its gradient: o, dq, dk, dv
  prefix    PagedCache.common_prefix and attention(prefix=...): a step of a
            batch of continuations of one document, whose pages they share
  sample    fused_sample: one token a row by temperature, top-k, top-p and min-p
            from given random numbers

Where `own` is false run() computes the operator in elementary torch operations
in 32 bits (64 for a sample's weights, whose sums are compared); where it is true
it makes the package's calls.  exact() restates each from its definition in 64
bits, a sequence and head (or row) at a time.
"""
import importlib
import math

import numpy as np
import torch

own = False
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32
TYPES = {"bf16": BF16, "f32": F32}
LAYERS = 14  # of the entropy model


def listed():
    return [
        # three short prompts of the entropy model's heads (12 of 64): latency
        dict(name="prompt_short", kind="prompt", seqs=3, longest=90, mix=1, pad=0, heads=12,
             kv_heads=12, dim=64, window=0, dtype="bf16"),
        # a batch of documents of up to 8192 bytes, a padded tail behind them
        dict(name="prompt_batch", kind="prompt", seqs=12, longest=8192, mix=2, pad=100, heads=12,
             kv_heads=12, dim=64, window=0, dtype="bf16"),
        # two long prompts, grouped heads of 128: the largest
        dict(name="prompt_long_grouped", kind="prompt", seqs=2, longest=16384, mix=3, pad=0,
             heads=32, kv_heads=8, dim=128, window=0, dtype="bf16"),
        # f32 throughout
        dict(name="prompt_f32", kind="prompt", seqs=5, longest=1501, mix=4, pad=3, heads=12,
             kv_heads=12, dim=64, window=0, dtype="f32"),
        # training on documents under the model's sliding window
        dict(name="train_window", kind="train", seqs=11, longest=2047, mix=5, pad=17, heads=12,
             kv_heads=12, dim=64, window=512, dtype="bf16"),
        # training on longer ones, grouped heads of 128
        dict(name="train_grouped", kind="train", seqs=4, longest=4096, mix=6, pad=0, heads=32,
             kv_heads=8, dim=128, window=0, dtype="bf16"),
        # the gradient in f32
        dict(name="train_f32", kind="train", seqs=3, longest=1000, mix=7, pad=0, heads=12,
             kv_heads=4, dim=64, window=0, dtype="f32"),
        # the next byte of 48 continuations of a document of 8192, all layers
        dict(name="prefix_step", kind="prefix", seqs=48, ctx=8192, tail=200, chunk=1, mix=8,
             layers=LAYERS, heads=12, kv_heads=12, dim=64, page=16, dtype="bf16"),
        # short drafts of 16 continuations of a long document, grouped heads of 128
        dict(name="prefix_draft_grouped", kind="prefix", seqs=16, ctx=30001, tail=900, chunk=6,
             mix=9, layers=2, heads=32, kv_heads=8, dim=128, page=32, dtype="bf16"),
        # the next byte of one document: latency
        dict(name="sample_byte", kind="sample", rows=1, vocab=260, mix=10, temperature=0.8,
             top_k=50, top_p=0.9, min_p=0.02, each=False, masked=0.0, dtype="f32"),
        # a byte for every position of half a batch, each row with settings of its own
        dict(name="sample_rows", kind="sample", rows=4096, vocab=260, mix=11, temperature=1.0,
             top_k=40, top_p=0.95, min_p=0.05, each=True, masked=0.2, dtype="f32"),
        # a large vocabulary, top-p over all of it
        dict(name="sample_wide", kind="sample", rows=64, vocab=131072, mix=12, temperature=0.9,
             top_k=0, top_p=0.95, min_p=0.0, each=False, masked=0.0, dtype="f32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "train", "train", "prefix", "prefix", "sample", "sample"])
    mix = rng.randrange(1 << 20)
    dtype = rng.choice(["bf16", "bf16", "f32"])
    heads, kv_heads, dim = rng.choice([(12, 12, 64), (12, 12, 64), (12, 4, 64), (32, 8, 128),
                                       (8, 1, 128), (4, 2, 128)])
    if kind in ("prompt", "train"):
        seqs, longest = _log(rng, 1, 64), _log(rng, 1, 16384)
        window = rng.choice([0, 0, 512, 300])
        # at most 2^17 tokens, and as many products as the listed ones of the type have
        seqs = max(1, min(seqs, (1 << 17) // longest))
        most = {"prompt": 1 << 39, "train": 1 << 37}[kind] // (1 if dtype == "bf16" else 64)
        longest = max(1, min(longest, int(math.sqrt(most / (seqs * heads * dim)))))
        return dict(kind=kind, seqs=seqs, longest=longest, mix=mix, pad=rng.choice([0, 0, 1, 77]),
                    heads=heads, kv_heads=kv_heads, dim=dim, window=window, dtype=dtype)
    if kind == "prefix":
        seqs, ctx = _log(rng, 1, 64), _log(rng, 10, 32768)
        chunk = 1 if rng.random() < 0.5 else _log(rng, 1, 64)
        tail = max(chunk, _log(rng, 1, 1000))
        layers = rng.choice([1, 2, LAYERS])
        # the pool: at most 2 GB in bf16
        tail = max(chunk, min(tail, (1 << 29) // (layers * seqs * kv_heads * dim)))
        ctx = max(10, min(ctx, (1 << 29) // (layers * kv_heads * dim)))
        most = (1 << 39) if dtype == "bf16" else (1 << 33)
        chunk = max(1, min(chunk, most // (layers * seqs * heads * dim * (ctx + tail))))
        return dict(kind=kind, seqs=seqs, ctx=ctx, tail=tail, chunk=chunk, mix=mix, layers=layers,
                    heads=heads, kv_heads=kv_heads, dim=dim, page=rng.choice([8, 16, 16, 32, 64]),
                    dtype=dtype)
    rows, vocab = _log(rng, 1, 4096), rng.choice([260, 260, _log(rng, 2, 131072), 32768, 131072])
    rows = max(1, min(rows, (64 * 131072) // vocab))
    return dict(kind=kind, rows=rows, vocab=vocab, mix=mix,
                temperature=rng.choice([0.0, 0.3, 0.7, 1.0, 1.0, 1.5]),
                top_k=rng.choice([0, 0, 1, 5, 50, _log(rng, 1, vocab)]),
                top_p=rng.choice([1.0, 1.0, 0.5, 0.9, 0.95, 0.99]),
                min_p=rng.choice([0.0, 0.0, 0.01, 0.05, 0.3]), each=rng.random() < 0.4,
                masked=rng.choice([0.0, 0.0, 0.3, 0.99]), dtype=dtype)


# ---- shapes of a case ------------------------------------------------------------

def _lengths(case):
    """Tokens of every sequence: the first has the full length, the others anything up to it."""
    r = np.random.RandomState(case["mix"])
    n = 1 + (r.rand(case["seqs"]) * case["longest"]).astype(np.int64)
    n[0] = case["longest"]
    return np.minimum(n, case["longest"])


def _tails(case):
    """(new tokens, own tokens with them) of every continuation."""
    r = np.random.RandomState(case["mix"])
    n = np.minimum(1 + (r.rand(case["seqs"]) * case["chunk"]).astype(np.int64), case["chunk"])
    n[0] = case["chunk"]
    tail = 1 + (r.rand(case["seqs"]) * case["tail"]).astype(np.int64)
    return n, np.maximum(np.minimum(tail, case["tail"]), n)


def _visible(n, length, window=0):
    """Pairs of (token, key) that the last n of `length` tokens see."""
    total = 0
    for a, b in zip(n.tolist(), length.tolist()):
        hi = np.arange(b - a, b) + 1
        total += int((np.minimum(hi, window) if window else hi).sum())
    return total


# ---- inputs ------------------------------------------------------------------------

def _package(name):
    return importlib.import_module("blt-burn_amd." + name)


def _i32(x):
    return torch.as_tensor(np.asarray(x, dtype=np.int32)).to(DEV)


def _starts(n):
    return np.concatenate([[0], np.cumsum(n)])


def _settings(case):
    """temperature, top_k, top_p, min_p: of the case, or a row's own around them."""
    c = case
    if not c["each"]:
        return c["temperature"], c["top_k"], c["top_p"], c["min_p"]
    r = np.random.RandomState(c["mix"])
    t = c["temperature"] * (0.5 + r.rand(c["rows"]))
    k = (c["top_k"] * 2 * r.rand(c["rows"])).astype(np.int32)
    p = 1 - (1 - c["top_p"]) * 2 * r.rand(c["rows"])
    m = c["min_p"] * 2 * r.rand(c["rows"])
    f = [torch.from_numpy(x.astype(np.float32)).to(DEV) for x in (t, np.maximum(p, 0.01), m)]
    return f[0], _i32(k), f[1], f[2]


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    c, t = case, TYPES[case["dtype"]]
    if c["kind"] in ("prompt", "train"):
        n = _lengths(c)
        total, H, K, d = int(n.sum()) + c["pad"], c["heads"], c["kv_heads"], c["dim"]
        # as a projection leaves them: q, k and v of a token side by side
        x = torch.randn((total, H + 2 * K, d), generator=g, device=DEV).to(t)
        st = dict(case=c, q=x[:, :H], k=x[:, H:H + K], v=x[:, H + K:], n=n.tolist(),
                  starts=_i32(_starts(n)))
        if c["kind"] == "train":
            st["do"] = torch.randn((total, H, d), generator=g, device=DEV).to(t)
        if own:
            F = _package("fused_ops")
            st["attention"] = F.fused_packed_attention
            if c["kind"] == "train":
                st["backward"] = F.fused_packed_attention_backward
        return st
    if c["kind"] == "prefix":
        n, tail = _tails(c)
        page, whole = c["page"], c["ctx"] // c["page"]
        length = c["ctx"] + tail
        need = -(-length // page)
        pool = whole + int((need - whole).sum()) + 3
        order = torch.randperm(pool, generator=g, device=DEV).cpu().numpy()
        table, used = np.full((c["seqs"], int(need.max())), -1, np.int64), np.zeros(pool, np.int64)
        table[:, :whole] = order[:whole]
        used[order[:whole]] = c["seqs"]
        at = whole
        for s, k in enumerate((need - whole).tolist()):
            table[s, whole:whole + k] = order[at:at + k]
            used[order[at:at + k]] = 1
            at += k
        shape = (c["layers"], pool, c["kv_heads"], page, c["dim"])
        k, v = (torch.empty(shape, dtype=t, device=DEV) for _ in range(2))
        for layer in list(k) + list(v):  # one at a time: the 32-bit draw of a layer only
            layer.copy_(torch.randn(layer.shape, generator=g, device=DEV))
        q = torch.randn((c["layers"], int(n.sum()), c["heads"], c["dim"]), generator=g,
                        device=DEV).to(t)
        st = dict(case=c, q=q, k=k, v=v, table=_i32(table), lens=_i32(length), refs=_i32(used),
                  starts=_i32(_starts(n)), n=n, length=length, shared=whole * page)
        if own:
            st["cache"] = _package("cache").PagedCache.wrap(k, v, st["table"], st["lens"],
                                                            st["refs"])
        return st
    x = torch.randn((c["rows"], c["vocab"]), generator=g, device=DEV) * 2.5
    # a few likely tokens above a broad rest, as a model's logits have
    likely = torch.randint(0, c["vocab"], (c["rows"], 8), generator=g, device=DEV)
    x.scatter_add_(1, likely, 4 * torch.rand((c["rows"], 8), generator=g, device=DEV))
    if c["masked"]:
        hide = torch.rand(x.shape, generator=g, device=DEV) < c["masked"]
        hide[:, 0] = False
        x.masked_fill_(hide, -math.inf)
    st = dict(case=c, logits=x.to(t), uniform=torch.rand(c["rows"], generator=g, device=DEV),
              settings=_settings(c))
    if own:
        st["sample"] = _package("fused_ops").fused_sample
    return st


# ---- one pass ------------------------------------------------------------------------

def run(state):
    return {"prompt": _prompt, "train": _train, "prefix": _prefix,
            "sample": _sample}[state["case"]["kind"]](state)


def _blocks(st):
    """(rows, key heads) of every sequence, so many heads that their scores stay below 2^28."""
    c, at = st["case"], 0
    for n in st["n"]:
        step = max(1, (1 << 28) // (n * n * (c["heads"] // c["kv_heads"])))
        for h in range(0, c["kv_heads"], step):
            yield slice(at, at + n), slice(h, min(h + step, c["kv_heads"]))
        at += n


def _weights(st, rows, kh):
    """Softmax weights [key heads, group, n, n] of one block in 32 bits, and its q, k, v."""
    c, G = st["case"], st["case"]["heads"] // st["case"]["kv_heads"]
    q = st["q"][rows, kh.start * G:kh.stop * G].float().transpose(0, 1).unflatten(0, (-1, G))
    k, v = (st[x][rows, kh].float().transpose(0, 1) for x in "kv")
    n = k.shape[1]
    s = torch.matmul(q.flatten(1, 2), k.transpose(1, 2)).view(-1, G, n, n)
    s /= math.sqrt(c["dim"])
    i = torch.arange(n, device=DEV)
    hide = i > i[:, None]
    if c["window"]:
        hide = hide | (i <= i[:, None] - c["window"])
    s.masked_fill_(hide, -math.inf)
    s -= s.amax(-1, keepdim=True)
    p = s.exp_()
    p /= p.sum(-1, keepdim=True)
    return p, q, k, v


def _tokens(x):
    """[key heads, group, n, d] -> [n, heads, d]"""
    return x.flatten(0, 1).transpose(0, 1)


def _prompt(st):
    if own:
        return st["attention"](st["q"], st["k"], st["v"], st["starts"],
                               window=st["case"]["window"])
    q, G = st["q"], st["case"]["heads"] // st["case"]["kv_heads"]
    o = torch.zeros(q.shape, dtype=q.dtype, device=DEV)
    for rows, kh in _blocks(st):
        p, _, _, v = _weights(st, rows, kh)
        x = torch.matmul(p.flatten(1, 2), v).view(*p.shape[:3], -1)
        o[rows, kh.start * G:kh.stop * G] = _tokens(x).to(o.dtype)
    return o


def _train(st):
    c, q, k, v, do = st["case"], st["q"], st["k"], st["v"], st["do"]
    if own:
        o, lse = st["attention"](q, k, v, st["starts"], window=c["window"], return_lse=True)
        return (o,) + st["backward"](do, q, k, v, o, lse, st["starts"], window=c["window"])
    G = c["heads"] // c["kv_heads"]
    o, dq, dk, dv = (torch.zeros(x.shape, dtype=x.dtype, device=DEV) for x in (q, q, k, v))
    for rows, kh in _blocks(st):
        qh = slice(kh.start * G, kh.stop * G)
        p, qf, kf, vf = _weights(st, rows, kh)
        g = do[rows, qh].float().transpose(0, 1).unflatten(0, (-1, G))
        y = torch.matmul(p.flatten(1, 2), vf).view(g.shape)
        dv[rows, kh] = torch.matmul(p.flatten(1, 2).transpose(1, 2),
                                    g.flatten(1, 2)).transpose(0, 1).to(dv.dtype)
        ds = torch.matmul(g.flatten(1, 2), vf.transpose(1, 2)).view(p.shape)
        ds -= (g * y).sum(-1, keepdim=True)
        ds *= p
        ds = ds.flatten(1, 2).mul_(1 / math.sqrt(c["dim"]))
        o[rows, qh] = _tokens(y).to(o.dtype)
        dq[rows, qh] = _tokens(torch.matmul(ds, kf).view(g.shape)).to(dq.dtype)
        dk[rows, kh] = torch.matmul(ds.transpose(1, 2),
                                    qf.flatten(1, 2)).transpose(0, 1).to(dk.dtype)
    return o, dq, dk, dv


def _prefix(st):
    c = st["case"]
    if own:
        cache = st["cache"]
        prefix = cache.common_prefix()
        return [cache.attention(layer, st["q"][layer], st["starts"], prefix=prefix)
                for layer in range(c["layers"])]
    H, K, d, page, B = c["heads"], c["kv_heads"], c["dim"], c["page"], c["seqs"]
    G, P, cols = H // K, st["shared"], st["shared"] // page
    starts, lens, most = st["starts"].long(), st["lens"].long(), int(st["n"].max())
    n, at = starts[1:] - starts[:-1], starts[:-1]
    first, own_pages = st["table"][0, :cols].long(), st["table"][:, cols:].clamp(min=0).long()
    row = torch.arange(most, device=DEV)
    take = (at[:, None] + row).clamp(max=st["q"].shape[1] - 1)
    real = row < n[:, None]
    pos = (lens - n)[:, None] + row
    key = P + torch.arange(own_pages.shape[1] * page, device=DEV)
    hide = ~((key <= pos[..., None]) & real[..., None])[:, None, None]
    out = []
    for layer in range(c["layers"]):
        k0, v0 = (x[layer][first].transpose(0, 1).reshape(K, P, d).float()
                  for x in (st["k"], st["v"]))
        k1, v1 = (x[layer][own_pages].transpose(1, 2).reshape(B, K, -1, d).float()
                  for x in (st["k"], st["v"]))
        q = st["q"][layer][take].float().view(B, most, K, G, d).permute(0, 2, 3, 1, 4)
        q = q / math.sqrt(d)
        s0 = torch.matmul(q.transpose(0, 1).reshape(K, -1, d), k0.transpose(1, 2))
        s0 = s0.view(K, B, G, most, P).transpose(0, 1)
        s1 = torch.matmul(q.reshape(B, K, -1, d), k1.transpose(2, 3)).view(B, K, G, most, -1)
        s1.masked_fill_(hide, -math.inf)
        s = torch.cat([s0, s1], -1)
        s -= s.amax(-1, keepdim=True)
        p = s.exp_()
        p /= p.sum(-1, keepdim=True)
        o = torch.matmul(p[..., :P].transpose(0, 1).reshape(K, -1, P), v0)
        o = o.view(K, B, G, most, d).transpose(0, 1)
        o = o + torch.matmul(p[..., P:].reshape(B, K, G * most, -1), v1).view(o.shape)
        out.append(o.permute(0, 3, 1, 2, 4).reshape(B, most, H, d)[real].to(st["q"].dtype))
    return out


def _sample(st):
    temperature, top_k, top_p, min_p = st["settings"]
    if own:
        return st["sample"](st["logits"], st["uniform"], temperature=temperature, top_k=top_k,
                            top_p=top_p, min_p=min_p)
    rows, V = st["logits"].shape

    def column(x):
        return torch.as_tensor(x, device=DEV).to(torch.float64).expand(rows)[:, None]

    t, k, tp, mp = (column(x) for x in (temperature, top_k, top_p, min_p))
    x, order = torch.sort(st["logits"].double(), dim=-1, descending=True, stable=True)
    d = torch.where(x == x[:, :1], 0.0, x - x[:, :1])
    p = torch.where(d == 0, 1.0, (d / t).exp())  # (temperature 0: the largest alone)
    rank = torch.arange(V, device=DEV)
    keep = (rank < torch.where(k > 0, k, V)) & (p >= mp) & ((t > 0) | (rank == 0))
    best = torch.where(rank < torch.where(k > 0, k, V), p, 0.0)
    before = best.cumsum(-1) - best
    keep &= (before < tp * best.sum(-1, keepdim=True)) | (tp >= 1) | (rank == 0)
    mass = torch.zeros_like(p).scatter_(1, order, torch.where(keep, p, 0.0)).cumsum(-1)
    want = st["uniform"].double()[:, None] * mass[:, -1:]
    return (mass > want).to(torch.int8).argmax(-1).to(torch.int32)


# ---- what a pass cannot do without ---------------------------------------------------

def work(case):
    c = case
    e = 2 if c["dtype"] == "bf16" else 4
    if c["kind"] == "sample":
        return {"bytes": c["rows"] * (c["vocab"] * e + 8), "flops": 0}
    H, K, d = c["heads"], c["kv_heads"], c["dim"]
    if c["kind"] in ("prompt", "train"):
        n = _lengths(c)
        total, pairs = int(n.sum()), _visible(n, n, c["window"])
        moved = total * (2 * H + 2 * K) * d * e
        if c["kind"] == "prompt":
            return {"bytes": moved, "flops": 4 * d * H * pairs}
        # besides: the outputs' gradient read, the inputs' written
        return {"bytes": moved + total * (2 * H + 2 * K) * d * e, "flops": 14 * d * H * pairs}
    n, tail = _tails(c)
    shared = c["ctx"] // c["page"] * c["page"]
    keys = shared + int((c["ctx"] + tail - shared).sum())
    pairs = _visible(n, c["ctx"] + tail)
    return {"bytes": c["layers"] * e * d * (2 * K * keys + 2 * H * int(n.sum())),
            "flops": 4 * d * H * pairs * c["layers"]}


# ---- the definition, in 64 bits ------------------------------------------------------

def _attend64(q, k, v, pos, window, do=None):
    """One head: queries at positions pos over keys 0 .. in 64 bits, with the gradients of
    q, k and v where the output's is given."""
    q, k, v = q.double(), k.double(), v.double()
    scale = q.shape[-1] ** -0.5
    key = torch.arange(k.shape[0], device=DEV)
    seen = key[None] <= pos[:, None]
    if window:
        seen &= pos[:, None] - key[None] < window
    p = torch.softmax((scale * (q @ k.t())).masked_fill(~seen, -math.inf), -1)
    o = p @ v
    if do is None:
        return o
    do = do.double()
    dp = do @ v.t()
    ds = p * (dp - (dp * p).sum(-1, keepdim=True))
    return o, scale * (ds @ k), scale * (ds.t() @ q), p.t() @ do


def exact(case, seed):
    c, st = case, prepare(case, seed)
    if c["kind"] == "sample":
        return _exact_sample(st)
    H, K, d = c["heads"], c["kv_heads"], c["dim"]
    if c["kind"] in ("prompt", "train"):
        out = [torch.zeros(st[x].shape, dtype=torch.float64, device=DEV) for x in "qqkv"]
        at = 0
        for n in st["n"]:
            pos, r = torch.arange(n, device=DEV), slice(at, at + n)
            for h in range(H):
                kh = h // (H // K)
                args = (st["q"][r, h], st["k"][r, kh], st["v"][r, kh], pos, c["window"])
                if c["kind"] == "prompt":
                    out[0][r, h] = _attend64(*args)
                    continue
                o, dq, dk, dv = _attend64(*args, st["do"][r, h])
                out[0][r, h], out[1][r, h] = o, dq
                out[2][r, kh] += dk
                out[3][r, kh] += dv
            at += n
        return out[0] if c["kind"] == "prompt" else tuple(out)
    if c["layers"] * c["seqs"] * H * (c["ctx"] + c["tail"]) > 1 << 28:
        return None
    table, n = st["table"].cpu().tolist(), st["n"].tolist()
    out = []
    for layer in range(c["layers"]):
        o = torch.empty(st["q"][layer].shape, dtype=torch.float64, device=DEV)
        at = 0
        for b in range(c["seqs"]):
            L = int(st["length"][b])
            pages = torch.tensor(table[b][:-(-L // c["page"])], device=DEV)
            pos = torch.arange(L - n[b], L, device=DEV)
            for kh in range(K):
                k, v = (x[layer][pages, kh].reshape(-1, d)[:L] for x in (st["k"], st["v"]))
                for h in range(kh * (H // K), (kh + 1) * (H // K)):
                    o[at:at + n[b], h] = _attend64(st["q"][layer][at:at + n[b], h], k, v, pos, 0)
            at += n[b]
        out.append(o)
    return out


def _exact_sample(st):
    logits, u = st["logits"].double().cpu().numpy(), st["uniform"].double().cpu().numpy()
    rows, V = logits.shape
    settings = [np.broadcast_to(x.double().cpu().numpy() if torch.is_tensor(x) else float(x), rows)
                for x in st["settings"]]
    out = np.zeros(rows, np.int32)
    for r in range(rows):
        t, k, tp, mp = (float(x[r]) for x in settings)
        x = logits[r]
        if t == 0:
            out[r] = int(np.argmax(x))
            continue
        ranked = np.argsort(-x, kind="stable")[:int(k) if k > 0 else V]
        w = np.exp((x[ranked] - x[ranked[0]]) / t)
        total, run, n = math.fsum(w), 0.0, 0
        while n < len(w) and w[n] >= mp and (n == 0 or tp >= 1 or run < tp * total):
            run += w[n]
            n += 1
        kept = np.sort(ranked[:n])
        mass = np.cumsum(np.exp((x[kept] - x[ranked[0]]) / t))
        out[r] = kept[int(np.argmax(mass > u[r] * mass[-1]))]
    return torch.from_numpy(out).to(DEV)
