"""Fused ops with the reference's public signatures (src/fused_ops/mod.rs:155-236).

Each function takes torch tensors on the GPU, allocates its output like the
reference's CubeBackend impl (a fresh contiguous tensor, backend.rs:42-53),
and runs one gfx950 kernel through libblt_hip.so on the current stream.
Inputs are f32 (Burn's default float) or bf16.  Shape mismatches raise
(where the reference panics).
"""
import ctypes

import torch

from . import _lib
from ._lib import EPS_AFTER_SQRT, EPS_INSIDE_SQRT, BltError, check
from ._torch import call_on, contiguous, require_cuda, stream_ptr

__all__ = ["fused_entropy", "fused_rms_norm", "fused_softmax", "fused_l2_norm",
           "fused_silu_gate", "fused_coherence", "fused_attention", "RotaryPlan", "fused_rotary",
           "EPS_AFTER_SQRT", "EPS_INSIDE_SQRT"]


def _dtype_ok(t):
    if t.dtype not in (torch.float32, torch.bfloat16):
        raise BltError("unsupported dtype %s (f32 or bf16)" % t.dtype)


def fused_entropy(logits, vocab_size):
    """[batch, seq, vocab] -> [batch, seq] f32 softmax entropy, natural log
    (mod.rs:155-159; NdArray form patcher.rs:38-63)."""
    require_cuda(logits)
    _dtype_ok(logits)
    if logits.dim() != 3:
        raise BltError("fused_entropy expects [batch, seq, vocab], got %s" % (tuple(logits.shape),))
    b, s, v = logits.shape
    if v != vocab_size:
        raise BltError("vocab_size %d does not match logits' last dim %d" % (vocab_size, v))
    x = contiguous(logits)
    out = torch.empty((b, s), dtype=torch.float32, device=x.device)
    f = (_lib.lib().blt_fused_entropy_f32 if x.dtype == torch.float32
         else _lib.lib().blt_fused_entropy_bf16)
    check(f(x.data_ptr(), out.data_ptr(), b * s, v, stream_ptr(x.device)), "fused_entropy")
    return out


def fused_rms_norm(input, weight, epsilon, eps_mode=EPS_AFTER_SQRT, l2_out=None):
    """[batch, seq, dim] x weight[dim] -> [batch, seq, dim] (mod.rs:162-176).

    eps_mode EPS_AFTER_SQRT is the model's formula x / (sqrt(mean x^2) + eps) * w
    (model.rs:758-770, and the reference's Fusion fallback backend.rs:502-506);
    EPS_INSIDE_SQRT is x / sqrt(mean x^2 + eps) * w (rms_norm_kernel.rs:40-43).
    l2_out, if given, is an f32 [batch, seq] tensor receiving sqrt(sum x^2)."""
    require_cuda(input, weight)
    _dtype_ok(input)
    if input.dim() != 3 or weight.dim() != 1 or weight.shape[0] != input.shape[-1]:
        raise BltError("fused_rms_norm expects x [batch, seq, dim] and weight [dim]")
    x = contiguous(input)
    w = contiguous(weight.to(x.dtype))
    y = torch.empty_like(x)
    rows, dim = x.numel() // x.shape[-1], x.shape[-1]
    l2p = 0
    if l2_out is not None:
        require_cuda(l2_out)
        if l2_out.dtype != torch.float32 or l2_out.numel() != rows or not l2_out.is_contiguous():
            raise BltError("l2_out must be a contiguous f32 tensor with one value per row")
        l2p = l2_out.data_ptr()
    f = (_lib.lib().blt_fused_rms_norm_f32 if x.dtype == torch.float32
         else _lib.lib().blt_fused_rms_norm_bf16)
    check(f(x.data_ptr(), w.data_ptr(), y.data_ptr(), l2p, rows, dim, float(epsilon), eps_mode,
            stream_ptr(x.device)), "fused_rms_norm")
    return y


def fused_softmax(input, dim_size):
    """Softmax over the last dim of an f32 tensor of any rank (mod.rs:179-185)."""
    require_cuda(input)
    if input.dtype != torch.float32:
        raise BltError("fused_softmax takes f32")
    if input.dim() == 0 or input.shape[-1] != dim_size:
        raise BltError("dim_size %d does not match the last dim" % dim_size)
    x = contiguous(input)
    y = torch.empty_like(x)
    check(_lib.lib().blt_fused_softmax_f32(x.data_ptr(), y.data_ptr(), x.numel() // dim_size,
                                           dim_size, stream_ptr(x.device)), "fused_softmax")
    return y


def fused_l2_norm(input):
    """[batch, seq, dim] -> [batch, seq] f32 sqrt(sum x^2) (mod.rs:188-192)."""
    require_cuda(input)
    _dtype_ok(input)
    if input.dim() != 3:
        raise BltError("fused_l2_norm expects [batch, seq, dim]")
    x = contiguous(input)
    b, s, d = x.shape
    out = torch.empty((b, s), dtype=torch.float32, device=x.device)
    f = (_lib.lib().blt_fused_l2_norm_f32 if x.dtype == torch.float32
         else _lib.lib().blt_fused_l2_norm_bf16)
    check(f(x.data_ptr(), out.data_ptr(), b * s, d, stream_ptr(x.device)), "fused_l2_norm")
    return out


def fused_silu_gate(gate_input, up_input):
    """silu(gate) * up, elementwise (mod.rs:195-205)."""
    require_cuda(gate_input, up_input)
    _dtype_ok(gate_input)
    if gate_input.shape != up_input.shape or gate_input.dtype != up_input.dtype:
        raise BltError("fused_silu_gate: gate and up must have one shape and dtype")
    g, u = contiguous(gate_input), contiguous(up_input)
    out = torch.empty_like(g)
    f = (_lib.lib().blt_fused_silu_gate_f32 if g.dtype == torch.float32
         else _lib.lib().blt_fused_silu_gate_bf16)
    check(f(g.data_ptr(), u.data_ptr(), out.data_ptr(), g.numel(), stream_ptr(g.device)),
          "fused_silu_gate")
    return out


def fused_coherence(norms, entropies, epsilon):
    """norms^2 / (entropies + epsilon), f32 (mod.rs:208-220)."""
    require_cuda(norms, entropies)
    if norms.dtype != torch.float32 or entropies.dtype != torch.float32:
        raise BltError("fused_coherence takes f32")
    if norms.shape != entropies.shape:
        raise BltError("fused_coherence: shapes differ")
    n, e = contiguous(norms), contiguous(entropies)
    out = torch.empty_like(n)
    check(_lib.lib().blt_fused_coherence_f32(n.data_ptr(), e.data_ptr(), out.data_ptr(),
                                             n.numel(), float(epsilon), stream_ptr(n.device)),
          "fused_coherence")
    return out


def fused_attention(q, k, v, use_causal_mask, window=0, rope_theta=0.0):
    """Scaled dot-product attention over [batch, heads, seq, head_dim] (mod.rs:225-236).

    f32 q, k, v without a window or RoPE: the reference kernel's semantics
    (attention_kernel.rs:20-125) in f32 throughout, any head_dim <= 256, k and v
    may have another seq length than q (causal: key j visible to query i iff
    j <= i).  bf16 inputs (or a window > 0 / rope_theta > 0, this build's
    extensions for the entropy model) take the MFMA path: head_dim 64, q, k, v
    of one shape, QK^T and PV on bf16 MFMA with an f32 softmax; f32 inputs are
    rounded to bf16 there and the output is returned in the input dtype."""
    require_cuda(q, k, v)
    _dtype_ok(q)
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise BltError("fused_attention expects q, k, v [batch, heads, seq, head_dim]")
    if (q.dtype == torch.float32 and k.dtype == torch.float32 and v.dtype == torch.float32 and
            window == 0 and rope_theta == 0):
        B, H, Tq, d = q.shape
        if tuple(k.shape[:2]) != (B, H) or k.shape[3] != d or k.shape != v.shape:
            raise BltError("fused_attention: k and v must be [batch, heads, seq_kv, head_dim] "
                           "with q's batch, heads and head_dim")
        qc, kc, vc = (contiguous(t) for t in (q, k, v))
        o = torch.empty_like(qc)
        check(_lib.lib().blt_fused_attention_f32(
            qc.data_ptr(), kc.data_ptr(), vc.data_ptr(), o.data_ptr(), B, H, Tq, kc.shape[2], d,
            1 if use_causal_mask else 0, stream_ptr(qc.device)), "fused_attention")
        return o
    if q.shape != k.shape or q.shape != v.shape:
        raise BltError("fused_attention (MFMA path) expects q, k, v of one shape "
                       "[batch, heads, seq, 64]")
    B, H, T, d = q.shape
    in_dtype = q.dtype
    qb, kb, vb = (contiguous(t.to(torch.bfloat16)) for t in (q, k, v))
    o = torch.empty_like(qb)
    ws = None
    if rope_theta > 0:
        nbytes = _lib.lib().blt_attention_workspace_bytes(B, H, T, d)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=qb.device)
    sb, sh, st = H * T * d, T * d, d
    check(_lib.lib().blt_fused_attention_bf16(
        qb.data_ptr(), kb.data_ptr(), vb.data_ptr(), o.data_ptr(), B, H, T, d,
        sb, sh, st, sb, sh, st, sb, sh, st, 1 if use_causal_mask else 0, int(window),
        float(rope_theta), ws.data_ptr() if ws is not None else 0, stream_ptr(qb.device)),
        "fused_attention")
    return o if in_dtype == torch.bfloat16 else o.to(in_dtype)


class RotaryPlan:
    """The frequencies of rotary positions, computed once and kept on a device.

    The first rotary_dim values of a head are rotated, in pairs (i, i + rotary_dim / 2)
    (pairs "half", the model's, model.rs:107-147) or (2 i, 2 i + 1) ("interleaved"), by
    the angles position * theta^(-2 i / rotary_dim).  Angles hold for any int32
    position; there is no table to outgrow.  scaling stretches them for contexts
    longer than a model was trained on (original_len positions, by `factor`):
      "linear"  every frequency divided by factor
      "ntk"     theta times factor^(rotary_dim / (rotary_dim - 2))
      "yarn"    high frequencies kept, low ones divided, a ramp between, and the
                rotated values times 0.1 ln(factor) + 1"""

    def __init__(self, rotary_dim, theta=10000.0, pairs="half", scaling="none", factor=1.0,
                 original_len=8192, device=None):
        if pairs not in ("half", "interleaved"):
            raise BltError("RotaryPlan: pairs must be 'half' or 'interleaved'")
        if scaling not in _lib.ROTARY_SCALING:
            raise BltError("RotaryPlan: scaling must be one of %s" % sorted(_lib.ROTARY_SCALING))
        dev = torch.device("cuda" if device is None else device)
        if dev.type != "cuda":
            raise BltError("RotaryPlan: the table must live on a GPU (got device %s)" % dev)
        n = int(rotary_dim)
        if not 2 <= n <= 512:  # (here too: past 32 bits the call would see its low bits)
            raise BltError("RotaryPlan: rotary_dim must be even, 2 .. 512")
        freq = torch.zeros(max(n // 2, 1), dtype=torch.int64)
        mag = ctypes.c_float()
        check(_lib.lib().blt_rotary_frequencies(n, float(theta), _lib.ROTARY_SCALING[scaling],
                                                float(factor), float(original_len),
                                                freq.data_ptr(), ctypes.addressof(mag)),
              "rotary_frequencies")
        if dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        self.rotary_dim, self.magnitude, self.device = n, mag.value, dev
        self._index, self._lib = dev.index, _lib.lib()
        self.freq = freq.to(dev)
        self._desc = _lib.Rotary(self.freq.data_ptr(), n, 1 if pairs == "interleaved" else 0,
                                 mag.value)
        self._ptr = ctypes.addressof(self._desc)


def _dense_rows(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _output_like(t):
    """A new tensor of t's order of dimensions whose last one is dense (that of overlapping
    rows need not be, in empty_like)."""
    y = torch.empty_like(t)
    return y if y.stride(-1) == 1 else torch.empty_like(t, memory_format=torch.contiguous_format)


class _RotaryGradient(torch.autograd.Function):
    """fused_rotary for inputs that need a gradient: the transposed rotation of the outputs'."""

    @staticmethod
    def forward(ctx, q, k, positions, plan, backward):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions)
        ctx.plan, ctx.turned = plan, backward
        out = fused_rotary(q, k, positions, plan, backward)
        ctx.mark_non_differentiable(*[y for y, need in zip(out, ctx.needs_input_grad)
                                      if y is not None and not need])
        return out

    @staticmethod
    def backward(ctx, gq, gk):
        (positions,) = ctx.saved_tensors
        if gq is None and gk is not None:
            gk, _ = fused_rotary(gk, None, positions, ctx.plan, not ctx.turned)
        elif gq is not None:
            gq, gk = fused_rotary(gq, gk, positions, ctx.plan, not ctx.turned)
        return gq, gk, None, None, None


def fused_rotary(q, k, positions, plan, backward=False, out=None):
    """Rotary positions of q [batch, heads, seq, head_dim] and k (its own number of
    heads; may be None) in one launch: (q', k').  Any strides with a dense last
    dimension are read as they are, e.g. views into a packed QKV tensor.
    positions: int32 [seq] or [batch, seq].  backward=True applies the transposed
    rotation, which turns gradients of q', k' into those of q, k; autograd does so by
    itself for inputs that need a gradient.  out: (q', k') to write, which may be q and k
    themselves; other overlaps are not allowed, nor are inputs that need a gradient."""
    for t in (q, positions) if k is None else (q, k, positions):
        if not isinstance(t, torch.Tensor):
            raise TypeError("expected a torch.Tensor, got %r" % type(t))
    if not isinstance(plan, RotaryPlan):
        require_cuda(q, positions)
        raise TypeError("fused_rotary expects a RotaryPlan")
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        if out is not None:
            raise BltError("fused_rotary: out takes no inputs that need a gradient (use "
                           "torch.no_grad())")
        return _RotaryGradient.apply(q, k, positions, plan, backward)
    index, dtype = plan._index, q.dtype
    if q.get_device() != index or positions.get_device() != index:
        require_cuda(q, positions)
        raise BltError("fused_rotary: tensors and plan must be on one device")
    _dtype_ok(q)
    if q.dim() != 4:
        raise BltError("fused_rotary expects q [batch, heads, seq, head_dim]")
    B, Hq, T, d = q.shape
    rows = positions.shape
    if positions.dtype is not torch.int32 or len(rows) not in (1, 2) or rows[-1] != T or \
            (len(rows) == 2 and rows[0] != B):
        raise BltError("fused_rotary: positions must be int32 [seq] or [batch, seq]")
    pos = _dense_rows(positions)
    x = _dense_rows(q)
    Hk, y, yp, kop, ys, ks = 0, None, None, None, (0, 0, 0), (0, 0, 0)
    if k is not None:
        if k.get_device() != index:
            require_cuda(k)
            raise BltError("fused_rotary: tensors and plan must be on one device")
        Bk, Hk, Tk, dk = k.shape if k.dim() == 4 else (-1, 0, 0, 0)
        if k.dtype is not dtype or Bk != B or Tk != T or dk != d:
            raise BltError("fused_rotary: k must be [batch, kv_heads, seq, head_dim] of q's dtype")
        y = _dense_rows(k)
        yp, ys = y.data_ptr(), y.stride()
    if out is None:
        qo = _output_like(x)
        ko = _output_like(y) if y is not None else None
    else:
        qo, ko = out
        if (ko is None) != (k is None):
            raise BltError("fused_rotary: out must hold a k exactly when k is given")
        for a, b in ((qo, q), (ko, k)):
            if b is None:
                continue
            require_cuda(a)
            if not (a.shape == b.shape and a.dtype == dtype and a.get_device() == index and
                    (a.stride(-1) == 1 or d == 1)):
                raise BltError("fused_rotary: out tensors must match q and k, with a dense last "
                               "dimension")
    xs, qs = x.stride(), qo.stride()
    if ko is not None:
        kop, ks = ko.data_ptr(), ko.stride()
    call_on(plan.device, index, plan._lib.blt_fused_rotary, "fused_rotary", x.data_ptr(), yp,
            qo.data_ptr(), kop, _lib.DTYPE_BF16 if dtype == torch.bfloat16 else _lib.DTYPE_F32, B,
            Hq, Hk, T, d, xs[0], xs[1], xs[2], ys[0], ys[1], ys[2], qs[0], qs[1], qs[2], ks[0],
            ks[1], ks[2], pos.data_ptr(), pos.stride(0) if len(rows) == 2 else 0, plan._ptr,
            1 if backward else 0)
    return qo, ko
