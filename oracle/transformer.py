"""CPU oracles of the transformer operators (ppv_amd.nn_ops.layer_norm, ppv_amd.attention, ppv_amd.optim.AdamW): plain implementations from
the formulas, in the precision of their inputs (tests call the first two in f64).  AdamW's is f32 by definition: its 8-bit form is a
function of the f32 arithmetic, operation by operation."""
import math

import torch

BLOCK = 256


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    centred = x - x.mean(-1, keepdim=True)
    y = centred / torch.sqrt((centred * centred).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight
    return y if bias is None else y + bias


def visible(Tq, Tk, q_len, k_len, causal):
    """[Tq, Tk] truth values of one sequence: row i < q_len sees key j < k_len, where causal if j <= i + k_len - q_len."""
    i, j = torch.arange(Tq).view(-1, 1), torch.arange(Tk).view(1, -1)
    seen = (i < q_len) & (j < k_len)
    return seen & (j - i <= k_len - q_len) if causal else seen


def attention(q, k, v, causal=False, q_lens=None, k_lens=None, scale=None):
    """q [B,Tq,H,D], k, v [B,Tk,Hkv,D] -> (out [B,Tq,H,D], log-sum-exp [B,H,Tq]); rows that see nothing are zero (-inf).  A pair that is
    masked takes no part at all, whatever k and v hold there."""
    B, Tq, H, D = q.shape
    Tk, G = k.shape[1], H // k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    outs, lses = [], []
    for b in range(B):
        n = Tq if q_lens is None else int(q_lens[b])
        m = Tk if k_lens is None else int(k_lens[b])
        seen = visible(Tq, Tk, n, m, causal)
        kb = k[b, :m].repeat_interleave(G, 1)
        vb = v[b, :m].repeat_interleave(G, 1)
        qb = torch.cat([q[b, :n], torch.zeros_like(q[b, n:])])
        s = torch.einsum("qhd,khd->hqk", qb, kb) * scale
        s = torch.where(seen[None, :, :m], s, torch.full_like(s, -math.inf))
        some = seen[:, :m].any(1)
        lse = torch.full((H, Tq), -math.inf, dtype=q.dtype)
        out = torch.zeros((Tq, H, D), dtype=q.dtype)
        if bool(some.any()):
            p = torch.softmax(s[:, some], -1)
            out = out.index_put((some.nonzero().squeeze(1),), torch.einsum("hqk,khd->qhd", p, vb))
            lse[:, some] = torch.logsumexp(s[:, some], -1).detach()
        outs.append(out)
        lses.append(lse)
    return torch.stack(outs), torch.stack(lses)


# ---------------------------------------------------------------------------------------------------------------- AdamW, 8-bit moments

def block_scale(x):
    """2^(floor(log2 max) - 7) of every block of 256 elements of x (values that are not finite stay out of the maximum)."""
    a = x.reshape(-1).abs()
    a = torch.where(torch.isfinite(a), a, torch.zeros_like(a))
    a = torch.cat([a, a.new_zeros(-a.numel() % BLOCK)]).view(-1, BLOCK).amax(1)
    e = (a.view(torch.int32) >> 23).clamp(min=9)
    return ((e - 7) << 23).view(torch.float32)


def spread(scale, n):
    return scale.repeat_interleave(BLOCK)[:n]


def dither(seed, step, place, n):
    low = 0xFFFFFFFF
    key = (seed * 0x9E3779B1 + step * 0x85EBCA77 + place * 0xC2B2AE3D) & low
    h = (torch.arange(n) * 0x9E3779B1 + key) & low
    h = ((h ^ (h >> 16)) * 0x7FEB352D) & low
    h = ((h ^ (h >> 15)) * 0x846CA68B) & low
    h = h ^ (h >> 16)
    return h & 0xFFFF, h >> 16


def to_e4m3(x, scale, dith, keep):
    """Stochastic rounding of x / scale to e4m3 (as f32 values); keep: what is not zero does not become zero."""
    a = x.abs() / scale
    up = (dith * 16 + 8).to(torch.int32)
    normal = ((a.view(torch.int32) + up) >> 20 << 20).view(torch.float32)
    small = torch.floor(a * 512.0 + up.float() * 2.0 ** -20) / 512.0
    r = torch.where(a >= 2.0 ** -6, normal, small)
    if keep:
        r = torch.where((r == 0) & (a > 0), torch.full_like(r, 2.0 ** -9), r)
    r = torch.where(torch.isfinite(a), r, torch.full_like(r, math.nan))
    return torch.copysign(r, x)


def adamw_step(p, g, st, step, place=0, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, seed=0):
    """One step on flat f32 tensors; st holds "m", "v" (32 bits) or "m", "r" (e4m3 values as f32), "ms", "rs"; updated in place."""
    b1, b2 = betas
    n = p.numel()
    if "r" in st:
        m, r = st["m"] * spread(st["ms"], n), st["r"] * spread(st["rs"], n)
        v = r * r
    else:
        m, v = st["m"], st["v"]
    m = m + (g - m) * (1 - b1)
    v = v * b2 + (g * (1 - b2)) * g
    root = torch.sqrt(v.double()).float()       # correctly rounded (torch.sqrt of f32 on the CPU is not always: 0.6 % of values are an ulp off)
    p.copy_(p * (1 - lr * weight_decay) - (m / (root * (1 / math.sqrt(1 - b2 ** step)) + eps)) * (lr / (1 - b1 ** step)))
    if "r" not in st:
        st["m"], st["v"] = m, v
        return
    dm, dr = dither(seed, step, place, n)
    st["ms"], st["rs"] = block_scale(m), block_scale(root)
    st["m"] = to_e4m3(m, spread(st["ms"], n), dm, False)
    st["r"] = to_e4m3(root, spread(st["rs"], n), dr, True)
