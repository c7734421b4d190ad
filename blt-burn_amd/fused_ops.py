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
from ._torch import call_on, contiguous, no_tangents, require_cuda, stream_ptr

__all__ = ["fused_entropy", "fused_rms_norm", "fused_softmax", "fused_l2_norm",
           "fused_silu_gate", "fused_coherence", "fused_attention", "fused_sample",
           "fused_packed_attention", "fused_packed_attention_backward", "RotaryPlan", "fused_rotary",
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


def _row_setting(x, what, like, dtype, lo, hi):
    """A number of all rows, or a tensor of one each: (number, pointer or None, what to keep)."""
    if isinstance(x, torch.Tensor):
        if x.dtype is not dtype or x.get_device() != like.get_device() or x.shape != like.shape:
            raise BltError("fused_sample: %s must be a number or %s %s on %s"
                           % (what, dtype, tuple(like.shape), like.device))
        x = contiguous(x)
        return 0, x.data_ptr(), x
    if not lo <= x <= hi:  # (here too: past 32 bits the call would see its low bits)
        raise BltError("fused_sample: %s out of range (%r)" % (what, x))
    return x, None, None


def fused_sample(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None):
    """One token a row of logits [..., vocab] (f32 or bf16, vocab up to 2^20), int32 [...], from
    given random numbers uniform [...] (f32 in [0, 1)), beside fused_softmax and fused_entropy of
    the same rows.

    With tokens ranked by logit (descending, equal ones by index) and weights
    e^((logit - max) / temperature), the tokens kept are those among the first top_k (0: all), whose running
    sum of the ranks before them is below top_p times the sum of those (1: all), with a weight of at least
    min_p; drawn is the lowest index whose running sum of kept weights, in the order of the indices,
    is above uniform times their sum.  temperature 0 takes the first of the largest.  Each setting is a number
    or a tensor like uniform (f32; top_k int32) of one for every row.

    A logit of -inf is never drawn.  A row with a NaN, without a logit above -inf or with a setting
    of its own out of range gives -1.  Weights are exact to 2^-42 of the largest or better, sums
    of them exact: the same tokens in every run."""
    require_cuda(logits, uniform)
    _dtype_ok(logits)
    if logits.dim() == 0 or not 1 <= logits.shape[-1] <= 1 << 20:
        raise BltError("fused_sample expects logits [..., vocab], vocab 1 .. 2^20")
    shape, V = logits.shape[:-1], logits.shape[-1]
    if uniform.dtype is not torch.float32 or uniform.shape != shape or \
            uniform.get_device() != logits.get_device():
        raise BltError("fused_sample: uniform must be f32 %s on %s" % (tuple(shape), logits.device))
    x = logits if logits.dim() == 2 and (logits.stride(1) == 1 or V == 1) and \
        logits.stride(0) >= 0 else contiguous(logits)
    u = contiguous(uniform)
    big = float("inf")
    t, tp, t_ = _row_setting(temperature, "temperature", u, torch.float32, 0, 1.7e308)
    k, kp, k_ = _row_setting(top_k, "top_k", u, torch.int32, 0, big)
    p, pp, p_ = _row_setting(top_p, "top_p", u, torch.float32, 5e-324, big)
    m, mp, m_ = _row_setting(min_p, "min_p", u, torch.float32, 0, 1)
    if out is None:
        out = torch.empty(shape, dtype=torch.int32, device=x.device)
    elif not isinstance(out, torch.Tensor):
        raise TypeError("expected a torch.Tensor, got %r" % type(out))
    elif out.dtype != torch.int32 or out.shape != shape or out.device != x.device or \
            not out.is_contiguous():
        raise BltError("fused_sample: out must be contiguous int32 %s on %s"
                       % (tuple(shape), x.device))
    rows, L, ws, size = u.numel(), _lib.lib(), None, 0
    if V > 1024:
        size = L.blt_fused_sample_workspace_bytes(rows, V)
        if size:
            ws = torch.empty(size, dtype=torch.uint8, device=x.device)
    call_on(x.device, x.get_device(), L.blt_fused_sample, "fused_sample", x.data_ptr(),
            x.stride(0) if x.dim() == 2 else V,
            _lib.DTYPE_BF16 if x.dtype == torch.bfloat16 else _lib.DTYPE_F32, rows, V, u.data_ptr(),
            t, tp, min(k, V), kp, p, pp, m, mp, out.data_ptr(), None if ws is None else ws.data_ptr(),
            size)
    return out


def _packed_heads(t, what, like=None, heads=None):
    """t [total, heads, head_dim] with 16-byte aligned rows: itself or a copy, its pointer and
    strides."""
    if not isinstance(t, torch.Tensor):
        raise TypeError("expected a torch.Tensor, got %r" % type(t))
    shape = t.shape
    if like is None:
        require_cuda(t)
        _dtype_ok(t)
        if len(shape) != 3 or shape[2] not in (64, 128):
            raise BltError("fused_packed_attention: %s must be [tokens, heads, head_dim 64 or 128]"
                           % what)
    else:
        n, _, d = like.shape
        if t.get_device() != like.get_device() or t.dtype is not like.dtype or len(shape) != 3 or \
                shape[0] != n or shape[2] != d or (heads is not None and shape[1] != heads):
            raise BltError("fused_packed_attention: %s must be %s [%d, %s, %d] on %s"
                           % (what, like.dtype, n, "heads" if heads is None else heads, d,
                              like.device))
    st, sh, sd = t.stride()
    p = t.data_ptr()
    if sd != 1 or (st | sh) & (3 if t.dtype is torch.float32 else 7) or p & 15 or st > 1 << 23:
        t = t.clone(memory_format=torch.contiguous_format)
        st, sh, _ = t.stride()
        p = t.data_ptr()
    return t, p, st, sh


def _packed_setting(q, k, starts, window, scale):
    H, Hkv = q.shape[1], k.shape[1]
    if Hkv == 0 or H == 0 or H % Hkv:
        raise BltError("fused_packed_attention: heads must be a multiple of kv_heads")
    if not isinstance(starts, torch.Tensor):
        raise TypeError("expected a torch.Tensor, got %r" % type(starts))
    if starts.dtype is not torch.int32 or starts.get_device() != q.get_device() or \
            starts.dim() != 1 or not starts.is_contiguous() or starts.shape[0] < 1:
        raise BltError("fused_packed_attention: starts must be a contiguous int32 [sequences + 1] "
                       "on %s" % q.device)
    if window < 0:
        raise BltError("fused_packed_attention: window must be >= 0")
    # (here too: past 32 bits the call would see its low bits)
    return (0 if window > 0x7fffffff else window), (q.shape[2] ** -0.5 if scale is None else scale)


class _PackedGradient(torch.autograd.Function):
    """fused_packed_attention for inputs that need a gradient."""

    @staticmethod
    def forward(ctx, q, k, v, starts, causal, window, scale):
        o, lse = fused_packed_attention(q, k, v, starts, causal, window, scale, return_lse=True)
        ctx.save_for_backward(q, k, v, o, lse, starts)
        ctx.setting = causal, window, scale
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return o, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_o, _):
        if grad_o is None:
            return (None,) * 7
        q, k, v, o, lse, starts = ctx.saved_tensors
        out = fused_packed_attention_backward(grad_o, q, k, v, o, lse, starts, *ctx.setting)
        return tuple(g if need else None
                     for g, need in zip(out, ctx.needs_input_grad)) + (None,) * 4


def fused_packed_attention(q, k, v, starts, causal=True, window=0, scale=None, out=None,
                           return_lse=False):
    """Attention of whole sequences of different lengths, packed behind each other: q [tokens,
    heads, head_dim], k and v [tokens, kv_heads, head_dim] (f32 or bf16, head_dim 64 or 128,
    heads a multiple of kv_heads; any strides, e.g. views into a packed QKV tensor, are
    read as they are where rows are dense and 16-byte aligned).  Sequence b has the tokens starts[b] ..
    starts[b + 1] - 1 (int32 [sequences + 1], ascending from 0).  causal: a token sees the keys of its
    sequence up to its own, with window > 0 only the last `window` of them; causal=False: all
    of them.  scale defaults to head_dim^-0.5.

    Returns o [tokens, heads, head_dim]; with return_lse also the logarithms of the softmax's sums,
    f32 [tokens, heads] (-inf for none), which fused_packed_attention_backward takes.  Tokens at
    starts[-1] and behind get 0 in a new tensor and are left alone in `out` (lse -inf in both); `out` may be
    q, but must not overlap k or v.  Scores and sums are f32 throughout; in bf16 the weights are rounded to
    bf16, and the sums take the rounded ones, or with return_lse or a gradient those before it, by which the
    gradient's weights go: o's last bits may differ between the two.  Autograd follows it for o
    (once; `out` takes no inputs that need a gradient), forward-mode does not."""
    no_tangents("fused_packed_attention", q, k, v)
    if torch.is_grad_enabled() and (getattr(q, "requires_grad", False)
                                    or getattr(k, "requires_grad", False)
                                    or getattr(v, "requires_grad", False)):
        if out is not None:
            raise BltError("fused_packed_attention: out takes no inputs that need a gradient (use "
                           "torch.no_grad())")
        both = _PackedGradient.apply(q, k, v, starts, causal, window, scale)
        return both if return_lse else both[0]
    q, qp, qs, qh = _packed_heads(q, "q")
    k, kp, ks, kh = _packed_heads(k, "k", q)
    v, vp, vs, vh = _packed_heads(v, "v", q, k.shape[1])
    window, scale = _packed_setting(q, k, starts, window, scale)
    total, H, d = q.shape
    tail = 1 if out is None else 0
    if out is None:
        out = torch.empty((total, H, d), dtype=q.dtype, device=q.device)
        op, os_, oh = out.data_ptr(), H * d, d
    else:
        t, op, os_, oh = _packed_heads(out, "out", q, H)
        if t is not out or (os_ == 0 and total > 1) or (oh == 0 and H > 1):
            raise BltError("fused_packed_attention: out needs dense, 16-byte aligned rows of their own")
    lse = lp = None
    if return_lse:
        lse = torch.empty((total, H), dtype=torch.float32, device=q.device)
        lp = lse.data_ptr()
    L, Hkv, B = _lib.lib(), k.shape[1], starts.shape[0] - 1
    dtype = _lib.DTYPE_BF16 if q.dtype == torch.bfloat16 else _lib.DTYPE_F32
    size, wp = 0, None
    if B > 1 and (total * H >> 5) + Hkv >= 512:  # (below that it takes none)
        size = L.blt_packed_attention_workspace_bytes(B, total, H, Hkv, dtype)
        if size:
            ws = torch.empty(size, dtype=torch.uint8, device=q.device)
            wp = ws.data_ptr()
    call_on(q.device, q.get_device(), L.blt_packed_attention, "packed_attention", qp, qs, qh, kp, ks,
            kh, vp, vs, vh, op, os_, oh, lp, dtype, total, H, Hkv, d, starts.data_ptr(), B,
            1 if causal else 0, window, scale, tail, wp, size)
    return (out, lse) if return_lse else out


def fused_packed_attention_backward(grad_o, q, k, v, o, lse, starts, causal=True, window=0,
                                    scale=None):
    """(dq, dk, dv) of fused_packed_attention from its output's gradient, its o and lse, and its
    other arguments; tokens at starts[-1] and behind get 0.  Sums are f32, in bf16 the weights and
    (as two halves for dq) their gradients are rounded to bf16; the same bits in every run."""
    no_tangents("fused_packed_attention_backward", grad_o, q, k, v, o, lse)
    q, qp, qs, qh = _packed_heads(q, "q")
    total, H, d = q.shape
    k, kp, ks, kh = _packed_heads(k, "k", q)
    Hkv = k.shape[1]
    v, vp, vs, vh = _packed_heads(v, "v", q, Hkv)
    o, op, os_, oh = _packed_heads(o, "o", q, H)
    grad_o, gp, gs, gh = _packed_heads(grad_o, "grad_o", q, H)
    window, scale = _packed_setting(q, k, starts, window, scale)
    if max(qh, gh) * (H // Hkv) > 1 << 29:
        q, grad_o = (t.clone(memory_format=torch.contiguous_format) for t in (q, grad_o))
        qp, gp, qs, gs, qh, gh = q.data_ptr(), grad_o.data_ptr(), H * d, H * d, d, d
    if not isinstance(lse, torch.Tensor):
        raise TypeError("expected a torch.Tensor, got %r" % type(lse))
    if lse.dtype != torch.float32 or lse.device != q.device or lse.shape != (total, H):
        raise BltError("fused_packed_attention_backward: lse must be f32 [tokens, heads]")
    lse = contiguous(lse)
    L = _lib.lib()
    dq = torch.empty((total, H, d), dtype=q.dtype, device=q.device)
    dk, dv = (torch.empty((total, Hkv, d), dtype=q.dtype, device=q.device) for _ in range(2))
    dtype = _lib.DTYPE_BF16 if q.dtype == torch.bfloat16 else _lib.DTYPE_F32
    size = L.blt_packed_attention_backward_workspace_bytes(total, H, Hkv, d, dtype)
    ws = torch.empty(size, dtype=torch.uint8, device=q.device)
    call_on(q.device, q.get_device(), L.blt_packed_attention_backward, "packed_attention_backward",
            gp, gs, gh, qp, qs, qh, kp, ks, kh, vp, vs, vh, op, os_, oh, lse.data_ptr(),
            dq.data_ptr(), H * d, d, dk.data_ptr(), Hkv * d, d, dv.data_ptr(), Hkv * d, d, dtype,
            total, H, Hkv, d, starts.data_ptr(), starts.shape[0] - 1, 1 if causal else 0, window, scale,
            ws.data_ptr(), size)
    return dq, dk, dv


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
    itself for inputs that need a gradient (forward-mode does not).  out: (q', k') to write, which may be q and k
    themselves; other overlaps are not allowed, nor are inputs that need a gradient."""
    for t in (q, positions) if k is None else (q, k, positions):
        if not isinstance(t, torch.Tensor):
            raise TypeError("expected a torch.Tensor, got %r" % type(t))
    no_tangents("fused_rotary", q, k)
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
