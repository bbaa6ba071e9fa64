"""Multi-head attention on the MI355X, forward and backward (csrc/attention.hip, csrc/attention_bwd.hip): what a transformer captioning head does
with caption tokens and with the encoder's cells or pixels, next to the single-step soft attention of ``ppv_amd.decoder.Attention``
(Image_Caption/models.py:57-90).

    out = multihead_attention(q, k, v, causal=..., q_lens=..., k_lens=...)

Scores and probabilities are never stored: the forward pass keeps one number per row (the log of the softmax's denominator), the backward
pass computes the probabilities again from it.  Products run on the matrix pipe in the operands' type (f32: exact f32 products) and
accumulate in f32; softmax statistics are f32.  Where probabilities and their gradients enter the next product they are rounded to the operands' type, or,
where that costs nothing (up to 32 rows or keys to a key head), given in two terms of it (csrc/attention_tiles.h two_terms).  No atomics: the same
bits every time.  No CPU path."""
import torch

from . import _lib
from .nn_ops import ELEM_TYPES


def _lens(name, t, B, T, device):
    if not torch.is_tensor(t) or t.dtype not in (torch.int32, torch.int64) or t.shape != (B,):
        raise ValueError(f"multihead_attention: {name} is an int32 or int64 tensor of shape ({B},)")
    if t.device != device:
        raise ValueError(f"multihead_attention: {name} is on {t.device}, q on {device}")
    return t.clamp(0, T).to(torch.int32) if t.dtype == torch.int64 else t.contiguous()


def _in_order(q, k, v):
    """What _refuse goes through one by one, as one expression: 7.8 us of a call's host time were these checks, 3 are."""
    t, on, ks = q.dtype, q.device, k.shape
    if not (q.dim() == 4 == len(ks) and v.shape == ks and t in ELEM_TYPES and k.dtype is t and v.dtype is t and k.device == on and v.device == on):
        return False
    (B, Tq, H, D), (Bk, Tk, Hkv, Dk) = q.shape, ks
    return (Bk == B and Dk == D and 1 <= D <= 128 and H >= 1 and Hkv >= 1 and H % Hkv == 0 and B * Hkv < 1 << 30 and Tq * H < 1 << 30 and Tk < 1 << 30)


def _refuse(q, k, v):
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
    if max(B * k.shape[2], Tq * H, k.shape[1]) >= 1 << 30:
        raise ValueError("multihead_attention: fewer than 2^30 rows, keys and (sequence, key head) pairs")
    if not 1 <= D <= 128:
        raise ValueError(f"multihead_attention: head dimension {D} is not in 1..128")


def multihead_attention(q, k, v, causal=False, q_lens=None, k_lens=None, scale=None):
    """softmax(scale q k^T) v for every head.

    q [B,Tq,H,D]; k, v [B,Tk,Hkv,D] with H a multiple of Hkv (query head h reads key head h // (H // Hkv)), D <= 128, all f32, bf16 or f16.  Any strides
    (pass ``x.transpose(1, 2)`` for [B,H,T,D]); views whose last axis is contiguous and whose other strides and address are multiples of
    16 bytes are read in place, others copied.  -> [B,Tq,H,D] of the same type, contiguous.

    q_lens, k_lens  int32 / int64 [B] on the same device (clamped to 0..Tq, 0..Tk): a sequence's queries and keys at or behind its length take
                    no part, whatever they hold; such queries give zeros, such queries and keys zero gradients.
    causal          row i of a sequence with n queries and m keys sees key j if j <= i + m - n: the last query sees every key, so a single new token
                    sees its whole history.  Rows that see nothing, or whose scores are all minus infinity, give zeros and zero
                    gradients.  (An infinite or NaN value in a key or row can reach, as zero times infinity, rows and keys of its
                    sequence that do not see it.)
    scale           > 0, D ** -0.5 by default.

    Fewer than 2^30 rows of a sequence (times heads), keys, and (sequence, key head) pairs; 2^24 tiles of 32 to 128 rows or keys in all.

    Gradients to q, k and v (once differentiable); those of shared key heads are the sums over their query heads."""
    if not _in_order(q, k, v):
        _refuse(q, k, v)
    B, Tq, _, D = q.shape
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < 1e30:
        raise ValueError("multihead_attention: scale > 0")
    if q_lens is not None:
        q_lens = _lens("q_lens", q_lens, B, Tq, q.device)
    if k_lens is not None:
        k_lens = _lens("k_lens", k_lens, B, k.shape[1], q.device)
    if not q.is_cuda:
        _lib.require_cuda(q)
    return _lib.torch_ops().attention(q, k, v, q_lens, k_lens, bool(causal), scale)
