"""A paged key/value cache and attention over it: the incremental form of the
entropy model's attention (the reference runs whole rows, model.rs:620-672).

A step of a running batch is

    cache.reserve(counts, seqs)                      # room for the new tokens
    for each layer:
        q = cache.append(layer, k, v, starts, seqs, rotary=plan, q=q)
        o = cache.attention(layer, q, starts, seqs)

and fork / trim / free / compact open, cut, drop and pack sequences.  All
bookkeeping is on the device: no call synchronises, and all of them can be
captured into a graph.  A call that the state does not allow (no free page, a
sequence too long) sets a bit in the cache's status instead of raising; check()
waits, raises BltError for it and clears it.  Calls on one cache must be
stream-ordered, attention among them: they share its workspace and counters (two
graphs that use one cache must not be replayed at once).  Autograd does not follow
them: what they return carries no gradient.
"""
import ctypes
import functools

import torch

from . import _lib
from ._lib import BltError
from ._torch import call_on, require_cuda
from .fused_ops import RotaryPlan

__all__ = ["PagedCache"]

_TYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}
_FAILURES = ((_lib.CACHE_FULL, "not enough free pages"),
             (_lib.CACHE_TOO_LONG, "a sequence would pass its page table"),
             (_lib.CACHE_BAD_INDEX, "an index out of range"),
             (_lib.CACHE_BUSY, "a sequence twice in a call, or a fork onto one with tokens"),
             (_lib.CACHE_NO_PAGE, "tokens appended where their sequence has no page"))


class PagedCache:
    """k, v [n_layers, num_pages, n_kv_heads, page_size, head_dim] (f32 or bf16) with
    page_table [max_seqs, max_pages], lens [max_seqs] and refcount [num_pages], all
    int32 tensors of the cache's device that may be read at any time (stream-ordered).
    head_dim 64 or 128, page_size a power of two from 8 to 1024.

    Beside them a cache keeps the workspace of its attention calls, as large as the calls
    so far have needed: at most 35 MB for single tokens, 104 MB (head_dim 64) or 136 MB (128)
    for any call, and up to a third more where it has grown.  The first call of a size may
    allocate."""

    def __init__(self, n_layers, n_kv_heads, head_dim, num_pages, max_seqs, max_len, page_size=16,
                 dtype=torch.bfloat16, device=None):
        if dtype not in _TYPES:
            raise BltError("PagedCache: dtype must be float32 or bfloat16")
        if min(n_layers, n_kv_heads, head_dim, num_pages, max_seqs, max_len, page_size) < 1:
            raise BltError("PagedCache: sizes must be positive")
        dev = torch.device("cuda" if device is None else device)
        shape = (n_layers, num_pages, n_kv_heads, page_size, head_dim)
        self._bind(torch.zeros(shape, dtype=dtype, device=dev),
                   torch.zeros(shape, dtype=dtype, device=dev),
                   torch.full((max_seqs, -(-max_len // page_size)), -1, dtype=torch.int32,
                              device=dev),
                   torch.zeros(max_seqs, dtype=torch.int32, device=dev),
                   torch.zeros(num_pages, dtype=torch.int32, device=dev))

    @classmethod
    def wrap(cls, k, v, page_table, lens, refcount):
        """A cache over tensors that the caller owns (shapes as above, contiguous), in
        the state that they describe."""
        self = cls.__new__(cls)
        self._bind(k, v, page_table, lens, refcount)
        return self

    def _bind(self, k, v, page_table, lens, refcount):
        require_cuda(k, v, page_table, lens, refcount)
        if k.dim() != 5 or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in _TYPES:
            raise BltError("PagedCache: k and v must be f32 or bf16 [layers, pages, kv_heads, "
                           "page_size, head_dim]")
        if page_table.dim() != 2 or lens.dim() != 1 or refcount.dim() != 1 or \
                page_table.shape[0] != lens.shape[0] or refcount.shape[0] != k.shape[1]:
            raise BltError("PagedCache: page_table [seqs, columns], lens [seqs], refcount [pages]")
        if any(t.dtype != torch.int32 for t in (page_table, lens, refcount)):
            raise BltError("PagedCache: page_table, lens and refcount must be int32")
        if any(t.device != k.device or not t.is_contiguous()
               for t in (k, v, page_table, lens, refcount)):
            raise BltError("PagedCache: tensors must be contiguous and on one device")
        self.k, self.v = k, v
        self.page_table, self.lens, self.refcount = page_table, lens, refcount
        self.device, self._index, self.dtype = k.device, k.device.index, k.dtype
        self.n_layers, self.num_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        self.max_seqs, self.max_pages = page_table.shape
        words = torch.zeros(1 + _lib.CACHE_SYNC_WORDS, dtype=torch.int32, device=k.device)
        self._status, self._sync = words[:1], words[1:]
        self._desc = _lib.PagedCacheDesc(
            k.data_ptr(), v.data_ptr(), page_table.data_ptr(), lens.data_ptr(),
            refcount.data_ptr(), self._status.data_ptr(), self._sync.data_ptr(), _TYPES[k.dtype], *k.shape[:3],
            k.shape[3], k.shape[4], *page_table.shape)
        self._ptr = ctypes.addressof(self._desc)
        self._lib = _lib.lib()
        self._call = functools.partial(call_on, self.device, self._index)
        self._piece, self._scale = 16 // k.element_size(), self.head_dim ** -0.5
        # the library's own checks, once: an empty list does nothing else
        self._call(self._lib.blt_cache_reserve, "PagedCache", self._ptr, None, None, 0)
        # attention's workspace (parts of its work, see _room): none yet
        self._ws, self._wsp, self._ws_bytes, self._ws_for = [], None, 0, None
        self._ws_most = max(self._lib.blt_paged_attention_workspace_bytes(
            self._ptr, 65536, 65536 * rows, self.n_kv_heads) for rows in (1, 32, 128))

    def _room(self, rows, total, heads):
        """Workspace for attention calls of this size.  It grows by steps of four or more and
        never past the largest call's; what it was before stays, for the graphs that use it."""
        need = self._lib.blt_paged_attention_workspace_bytes(self._ptr, rows, total, heads)
        if need > self._ws_bytes:
            size = max(need, min(4 * self._ws_bytes, self._ws_most))
            self._ws.append(self._workspace(size))
            self._wsp, self._ws_bytes = self._ws[-1].data_ptr(), size
        self._ws_for = (rows, total, heads)

    def record_stream(self, stream):
        """Tensor.record_stream for everything the cache holds: for a cache that is dropped
        while another stream than the one it was made on still uses it."""
        for t in [self.k, self.v, self.page_table, self.lens, self.refcount, self._status] + self._ws:
            t.record_stream(stream)

    # ---- status ---------------------------------------------------------------
    def check(self):
        """Wait for the calls so far; raise BltError if one of them failed, and clear it."""
        bits = int(self._status.item())
        if bits:
            self._status.zero_()
            raise BltError("paged cache: " + "; ".join(t for b, t in _FAILURES if bits & b))

    # ---- lists of sequences ---------------------------------------------------
    def _list(self, t, what, n=None):
        """(pointer, length) of an int32 list on the cache's device, of length n if given."""
        if not isinstance(t, torch.Tensor):
            raise TypeError("expected a torch.Tensor, got %r" % type(t))
        if t.dtype is not torch.int32 or t.get_device() != self._index or t.dim() != 1 or \
                not t.is_contiguous() or (n is not None and t.shape[0] != n):
            raise BltError("PagedCache: %s must be a contiguous int32 [%s] on %s"
                           % (what, "n" if n is None else n, self.device))
        return t.data_ptr(), t.shape[0]

    def _workspace(self, nbytes):
        return torch.empty(nbytes, dtype=torch.uint8, device=self.device)

    def reserve(self, counts, seqs=None):
        """Grow sequence seqs[i] (None: i) by counts[i] tokens; missing pages are the free
        ones with the lowest index.  All or, with a status bit, none."""
        c, n = self._list(counts, "counts")
        s = None if seqs is None else self._list(seqs, "seqs", n)[0]
        self._call(self._lib.blt_cache_reserve, "cache_reserve", self._ptr, s, c, n)

    def trim(self, lens, seqs=None):
        """Cut sequence seqs[i] (None: i) to lens[i] tokens where it is longer."""
        p, n = self._list(lens, "lens")
        s = None if seqs is None else self._list(seqs, "seqs", n)[0]
        size = self._lib.blt_cache_workspace_bytes(self._ptr, max(n, 1))
        ws = self._workspace(size)
        self._call(self._lib.blt_cache_trim, "cache_trim", self._ptr, s, p, n, ws.data_ptr(), size)

    def free(self, seqs):
        """Drop sequences: their pages are free where no other sequence shares them."""
        s, n = self._list(seqs, "seqs")
        self._call(self._lib.blt_cache_trim, "cache_free", self._ptr, s, None, n, None, 0)

    def fork(self, src, dst):
        """Make every dst[i] (a sequence without tokens) a continuation of src[i]: full
        pages are shared, a partly filled last page is copied."""
        a, n = self._list(src, "src")
        b = self._list(dst, "dst", n)[0]
        self._call(self._lib.blt_cache_fork, "cache_fork", self._ptr, a, b, n)

    def compact(self):
        """Move the used pages with the highest indices into the lowest free ones."""
        size = self._lib.blt_cache_workspace_bytes(self._ptr, 0)
        ws = self._workspace(size) if size else None
        self._call(self._lib.blt_cache_compact, "cache_compact", self._ptr,
                   ws.data_ptr() if size else None, size)

    def copy_pages(self, src, dst):
        """Copy page src[i] to page dst[i] in every layer (no index twice in dst, none in
        both)."""
        a, n = self._list(src, "src")
        b = self._list(dst, "dst", n)[0]
        self._call(self._lib.blt_cache_copy_pages, "cache_copy_pages", self._ptr, a, b, n)

    # ---- tokens ---------------------------------------------------------------
    def _rows(self, starts, seqs):
        """(starts pointer, rows, seqs pointer or None)."""
        p, n = self._list(starts, "starts")
        if n < 1:
            raise BltError("PagedCache: starts has one entry more than there are sequences")
        return p, n - 1, None if seqs is None else self._list(seqs, "seqs", n - 1)[0]

    def _layer(self, layer):
        # (here too: past 32 bits the call would see its low bits)
        if not 0 <= layer < self.n_layers:
            raise BltError("PagedCache: no such layer (%r of %d)" % (layer, self.n_layers))
        return layer

    def _tokens(self, t, what, heads=None):
        """t [tokens, heads, head_dim] with a dense last dimension: itself or a copy, its
        pointer, tokens, heads and strides."""
        if not isinstance(t, torch.Tensor):
            raise TypeError("expected a torch.Tensor, got %r" % type(t))
        shape = t.shape
        if t.dtype is not self.dtype or t.get_device() != self._index or len(shape) != 3 or \
                shape[2] != self.head_dim or (heads is not None and shape[1] != heads):
            raise BltError("PagedCache: %s must be %s [tokens, %s, %d] on %s"
                           % (what, self.dtype, "heads" if heads is None else heads,
                              self.head_dim, self.device))
        st, sh, sd = t.stride()
        if sd != 1:
            t = t.contiguous()
            st, sh, sd = t.stride()
        return t, t.data_ptr(), shape[0], shape[1], st, sh

    def _output(self, out, like, total, heads):
        """(out, or a new tensor like `like`; its pointer and strides)"""
        if out is None:
            out = torch.empty_like(like)
            st, sh, sd = out.stride()
            if sd != 1:  # (of overlapping rows)
                out = torch.empty_like(like, memory_format=torch.contiguous_format)
                st, sh, sd = out.stride()
            return out, out.data_ptr(), st, sh
        t, p, n, _, st, sh = self._tokens(out, "out", heads)
        if t is not out or n != total:
            raise BltError("PagedCache: out must match q, with a dense last dimension")
        return out, p, st, sh

    def append(self, layer, k, v, starts, seqs=None, rotary=None, q=None, out=None):
        """Write the new tokens k, v [total, kv_heads, head_dim] into a layer: row b has
        tokens starts[b] .. starts[b + 1] - 1 (int32 [rows + 1]) and they become the last
        ones of sequence seqs[b] (None: b; none twice), whose length already counts them
        (reserve).  rotary: a RotaryPlan that rotates k at its positions, and q [total, heads,
        head_dim] if given, which is returned (into `out`, which may be q; tokens at
        starts[-1] and behind are not written).  starts ascends from 0 on within the
        tokens (else the status is set)."""
        layer = self._layer(layer)
        k, kp, total, _, ks, kh = self._tokens(k, "k", self.n_kv_heads)
        v, vp, n, _, vs, vh = self._tokens(v, "v", self.n_kv_heads)
        p, B, s = self._rows(starts, seqs)
        if n != total:
            raise BltError("PagedCache: k and v must have one number of tokens")
        r, qp, qs, qh, op, os_, oh, Hq = None, None, 0, 0, None, 0, 0, 0
        if rotary is not None:
            if not isinstance(rotary, RotaryPlan):
                raise TypeError("PagedCache.append expects a RotaryPlan")
            if rotary._index != self._index:
                raise BltError("PagedCache: the rotary plan is on another device")
            r = rotary._ptr
        if q is not None:
            if rotary is None:
                raise BltError("PagedCache.append: q is rotated only with a rotary plan")
            q, qp, n, Hq, qs, qh = self._tokens(q, "q")
            if n != total:
                raise BltError("PagedCache: q and k must have one number of tokens")
            out, op, os_, oh = self._output(out, q, total, Hq)
        elif out is not None:
            raise BltError("PagedCache.append: out without q")
        self._call(self._lib.blt_cache_append, "cache_append", self._ptr, layer, kp, ks, kh, vp, vs,
                   vh, qp, qs, qh, op, os_, oh, Hq, p, s, B, total, r)
        return out

    def attention(self, layer, q, starts, seqs=None, causal=True, window=0, scale=None, out=None):
        """Attention of new tokens q [total, heads, head_dim] over a layer of the cache,
        whose lengths already count them (rows as in append; a sequence may appear twice):
        the last of a row's n tokens sits at its sequence's last position.  Query head h
        reads key head h // (heads / kv_heads).  causal: keys up to the token's own
        position, with window > 0 only the last `window` of them; causal=False: every
        key.  scale defaults to head_dim^-0.5.  Returns [total, heads, head_dim] (`out` if
        given, whose rows are 16-byte aligned): 0 where a token sees no key; tokens at
        starts[-1] and behind are not written, nor are those of a row without a sequence,
        nor any where starts does not ascend within q (both set the status).

        A key whose score is -inf weighs nothing.  Scores, sums and f32 outputs are f32
        throughout; in bf16 the softmax's weights are rounded to bf16 where the rows have more
        than 32 tokens on average (heads per key head counted as tokens), and to 2^-15 of
        them below.  That average also chooses the kernel, so a long chunk is best issued
        apart from many single tokens; and calls of more than some hundred rows are best cut
        into several (a call's cost has a part that grows with the square of its rows)."""
        layer = self._layer(layer)
        q, qp, total, H, qs, qh = self._tokens(q, "q")
        p, B, s = self._rows(starts, seqs)
        if H % self.n_kv_heads or H == 0:
            raise BltError("PagedCache: q's heads must be a multiple of the cache's %d"
                           % self.n_kv_heads)
        if (qs | qh) % self._piece or qp % 16:  # rows that are not 16-byte aligned
            q = q.clone(memory_format=torch.contiguous_format)
            qs, qh, _ = q.stride()
            qp = q.data_ptr()
        out, op, os_, oh = self._output(out, q, total, H)
        if self._ws_for != (B, total, H):
            self._room(B, total, H)
        if window < 0:
            raise BltError("PagedCache.attention: window must be >= 0")
        if window > 0x7fffffff:  # longer than any sequence
            window = 0
        self._call(self._lib.blt_paged_attention, "paged_attention", self._ptr, layer, qp, qs, qh, op,
                   os_, oh, H, p, s, B, total, 1 if causal else 0, window,
                   self._scale if scale is None else scale, self._wsp, self._ws_bytes)
        return out
