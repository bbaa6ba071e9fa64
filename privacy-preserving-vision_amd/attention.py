"""Multi-head attention on the MI355X, forward and backward (csrc/attention.hip, csrc/attention_bwd.hip): what a transformer captioning head does
with caption tokens and with the encoder's cells or pixels, next to the single-step soft attention of ``ppv_amd.decoder.Attention``
(Image_Caption/models.py:57-90).

    out = multihead_attention(q, k, v, causal=..., q_lens=..., k_lens=...)

Scores and probabilities are never stored: the forward pass keeps one number per row (the log of the softmax's denominator), the backward
pass computes the probabilities again from it.  Products run on the matrix pipe in the operands' type (f32: exact f32 products) and
accumulate in f32; softmax statistics are f32, the probabilities are rounded to the operands' type where they enter the next product.  No atomics: the
same bits every time.  No CPU path."""
import torch

from . import _lib
from ._lib import check, ptr, stream_ptr
from .nn_ops import ELEM_TYPES


def _operand(t, Dp):
    """t [B,T,H,D] as the kernels read it: unit last stride, every other stride and the address multiples of 16 bytes, D padded to Dp.
    A view that is already so is taken as it is, any other is copied (zeros behind D add nothing to a product)."""
    v = 16 // t.element_size()
    if (t.shape[3] == Dp and t.stride(3) == 1 and t.data_ptr() % 16 == 0
            and all(s % v == 0 or n == 1 for s, n in zip(t.stride()[:3], t.shape[:3])) and (t.stride(1) <= 1 << 22 or t.shape[1] == 1)):
        return t
    p = torch.empty(t.shape[:3] + (Dp,), dtype=t.dtype, device=t.device)
    if Dp != t.shape[3]:
        p[..., t.shape[3]:].zero_()
    p[..., :t.shape[3]].copy_(t)
    return p


def _strides(t):
    return tuple(0 if n == 1 else s for s, n in zip(t.stride()[:3], t.shape[:3]))


def _describe(q, k, v, out, lo, lse, q_lens, k_lens, causal, scale):
    a = _lib.Attention()
    a.q, a.k, a.v, a.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    a.out_lo, a.lse, a.q_lens, a.k_lens = (None if t is None else t.data_ptr() for t in (lo, lse, q_lens, k_lens))
    (a.sqb, a.sqt, a.sqh), (a.skb, a.skt, a.skh), (a.svb, a.svt, a.svh) = _strides(q), _strides(k), _strides(v)
    a.B, a.Tq, a.H, a.D = q.shape
    a.Tk, a.Hkv = k.shape[1], k.shape[2]
    a.dtype, a.causal, a.scale = ELEM_TYPES[q.dtype], int(causal), scale
    return a


def _padded(D, dtype):
    v = 4 if dtype == torch.float32 else 8
    return (D + v - 1) // v * v


def _forward(q, k, v, q_lens, k_lens, causal, scale, keep):
    """-> (out [B,Tq,H,D padded], what rounding took from it or None, lse or None, the operands as the kernels read them).
    keep: for a backward pass, whose rowsum(dO O) would carry the rounding of a 16-bit O into every score's gradient."""
    B, Tq, H, D = q.shape
    Dp = _padded(D, q.dtype)
    q, k, v = (_operand(t, Dp) for t in (q, k, v))
    out = torch.empty((B, Tq, H, Dp), dtype=q.dtype, device=q.device)
    lse = torch.empty((B, H, Tq), dtype=torch.float32, device=q.device) if keep else None
    lo = torch.empty_like(out) if keep and q.dtype != torch.float32 else None
    if out.numel() == 0:
        return out, lo, lse, q, k, v
    if k.numel() == 0:                                           # no keys at all: every row is empty
        out.zero_()
        return out, lo, lse, q, k, v
    L = _lib.lib()
    a = _describe(q, k, v, out, lo, lse, q_lens, k_lens, causal, scale)
    n = int(L.ppv_attention_fwd_workspace_bytes(a.B, a.H, a.Hkv, a.Tq, a.Tk, a.D, a.dtype))
    ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
    a.workspace = None if ws is None else ws.data_ptr()
    with _lib.device_of(q):
        check(L.ppv_attention_fwd(a, stream_ptr()), "ppv_attention_fwd")
    return out, lo, lse, q, k, v


class _AttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, q_lens, k_lens, causal, scale):
        out, lo, lse, qp, kp, vp = _forward(q, k, v, q_lens, k_lens, causal, scale, True)
        ctx.save_for_backward(qp, kp, vp, out, lo, lse, q_lens, k_lens)
        ctx.cfg = (causal, scale, q.shape[3])
        return out if out.shape[3] == q.shape[3] else out[..., :q.shape[3]].contiguous()

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        q, k, v, out, lo, lse, q_lens, k_lens = ctx.saved_tensors
        causal, scale, D = ctx.cfg
        Dp = out.shape[3]
        dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        dk, dv = (torch.empty(k.shape, dtype=q.dtype, device=q.device) for _ in range(2))
        if q.numel() == 0 or k.numel() == 0:
            grads = [t.zero_() for t in (dq, dk, dv)]
        else:
            L = _lib.lib()
            g = _operand(g, Dp)
            a = _describe(q, k, v, out, lo, lse, q_lens, k_lens, causal, scale)
            a.dout, a.dq, a.dk, a.dv = g.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
            a.sgb, a.sgt, a.sgh = _strides(g)
            ws = torch.empty(int(L.ppv_attention_bwd_workspace_bytes(a.B, a.H, a.Tq)), dtype=torch.uint8, device=q.device)
            a.workspace = ws.data_ptr()
            with _lib.device_of(q):
                check(L.ppv_attention_bwd(a, stream_ptr()), "ppv_attention_bwd")
            grads = [dq, dk, dv]
        if Dp != D:
            grads = [t[..., :D].contiguous() for t in grads]
        return tuple(t if ctx.needs_input_grad[i] else None for i, t in enumerate(grads)) + (None,) * 4


def _lens(name, t, B, T, device):
    if t is None:
        return None
    if not torch.is_tensor(t) or t.dtype not in (torch.int32, torch.int64) or t.shape != (B,):
        raise ValueError(f"multihead_attention: {name} is an int32 or int64 tensor of shape ({B},)")
    if t.device != device:
        raise ValueError(f"multihead_attention: {name} is on {t.device}, q on {device}")
    return t.clamp(0, T).to(torch.int32) if t.dtype == torch.int64 else t.contiguous()


def multihead_attention(q, k, v, causal=False, q_lens=None, k_lens=None, scale=None):
    """softmax(scale q k^T) v for every head.

    q [B,Tq,H,D]; k, v [B,Tk,Hkv,D] with H a multiple of Hkv (query head h reads key head h // (H // Hkv)), D <= 128, all f32, bf16 or f16.  Any strides
    (pass ``x.transpose(1, 2)`` for [B,H,T,D]); views whose last axis is contiguous and whose other strides and address are multiples of
    16 bytes are read in place, others copied.  -> [B,Tq,H,D] of the same type, contiguous.

    q_lens, k_lens  int32 / int64 [B] on the same device (clamped to 0..Tq, 0..Tk): a sequence's queries and keys at or behind its length take
                    no part, whatever they hold; such queries give zeros, such queries and keys zero gradients.
    causal          row i of a sequence with n queries and m keys sees key j if j <= i + m - n: the last query sees every key, so a single new token
                    sees its whole history.  Rows that see nothing give zeros and zero gradients.  (A key's infinite or NaN value that only some of
                    a sequence's rows may see can reach the others of them.)
    scale           > 0, D ** -0.5 by default.

    Gradients to q, k and v (once differentiable); those of shared key heads are the sums over their query heads."""
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 4:
            raise ValueError(f"multihead_attention: {name} is [B, T, H, D]")
        if t.dtype not in ELEM_TYPES or t.dtype != q.dtype:
            raise TypeError("multihead_attention: q, k, v are f32, bf16 or f16, all of one type")
        if t.device != q.device:
            raise ValueError(f"multihead_attention: {name} is on {t.device}, q on {q.device}")
    B, Tq, H, D = q.shape
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != D:
        raise ValueError(f"multihead_attention: shapes q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} do not belong together")
    if H < 1 or k.shape[2] < 1 or H % k.shape[2]:
        raise ValueError(f"multihead_attention: {H} query heads over {k.shape[2]} key heads")
    if not 1 <= D <= 128:
        raise ValueError(f"multihead_attention: head dimension {D} is not in 1..128")
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < 1e30:
        raise ValueError("multihead_attention: scale > 0")
    q_lens, k_lens = _lens("q_lens", q_lens, B, Tq, q.device), _lens("k_lens", k_lens, B, k.shape[1], q.device)
    _lib.require_cuda(q)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _AttentionFn.apply(q, k, v, q_lens, k_lens, bool(causal), scale)
    out = _forward(q.detach(), k.detach(), v.detach(), q_lens, k_lens, bool(causal), scale, False)[0]
    return out if out.shape[3] == D else out[..., :D].contiguous()
