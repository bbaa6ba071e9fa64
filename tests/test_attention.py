"""ppv_amd.attention.multihead_attention (csrc/attention.hip, csrc/attention_bwd.hip) against the formula in 64 bits: value and gradients over
types, head layouts, lengths, masks, strides; refusals.

Tolerances count roundings.  u = 2^-24 (f32 arithmetic), h = half a step of the operands' type (0 for f32 products, which are exact f32).
  S: D products accumulated in f32: off by at most (D + 2) u scale |q||k|; in the exponent that is a relative error of P.  The running
     maximum, exp2 and the saved log-sum-exp add (4 + |S| + log) u.  So P is off by eP = e_s + h relative, e_s = u (D + 2) max(scale |q||k|) + 32 u.
  O = sum P V: |dO_i| <= (eP + (Tk + 8) u ... a f32 chain over tiles, counted as 64 u + Tk / 32 u) sum P |V|, then rounded once: h |O|.
  dV = sum P dO likewise.  dS = P (dP - D) with dP, D off by (D + 2) u |dO||V| and, D being taken from the rounded O, h |dO| . |O|;
     rounded to the operands' type with the scale in it: h.  dQ and dK sum dS over keys and rows."""
import math

import pytest
import torch

from oracle import transformer as orc

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24


def _inputs(B, Tq, Tk, H, Hkv, D, dt, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: (torch.randn(*s, generator=g) * spread).to(dt)
    return r(B, Tq, H, D), r(B, Tk, Hkv, D), r(B, Tk, Hkv, D), r(B, Tq, H, D)


def _bounds(q, k, v, g, causal, q_lens, k_lens, scale):
    """(reference out, dq, dk, dv) in f64 with a bound for each."""
    dt = q.dtype
    h = 0.0 if dt == torch.float32 else torch.finfo(dt).eps / 2
    hr = torch.finfo(dt).eps / 2                       # the results' own rounding
    tiny = 0.0 if dt != torch.float16 else 2.0 ** -25  # f16: half a step of its subnormals
    B, Tq, H, D = q.shape
    Tk, G = k.shape[1], H // k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    qd, kd, vd = (t.double().requires_grad_(True) for t in (q, k, v))
    gd = g.double()
    out, _ = orc.attention(qd, kd, vd, causal, q_lens, k_lens, scale)
    dq, dk, dv = torch.autograd.grad(out, (qd, kd, vd), gd)
    out = out.detach()
    tol = [torch.zeros_like(t) for t in (out, dq, dk, dv)]
    for b in range(B):
        n = Tq if q_lens is None else min(max(int(q_lens[b]), 0), Tq)
        m = Tk if k_lens is None else min(max(int(k_lens[b]), 0), Tk)
        seen = orc.visible(Tq, Tk, n, m, causal)[:n, :m]
        if not bool(seen.any()):
            continue
        qb, gb, ob = (t[b, :n].detach().transpose(0, 1) for t in (qd, gd, out))                     # [H, n, D]
        kb, vb = (t[b, :m].detach().transpose(0, 1).repeat_interleave(G, 0) for t in (kd, vd))      # [H, m, D]
        s = qb @ kb.transpose(1, 2) * scale
        s = torch.where(seen, s, torch.full_like(s, -math.inf))
        some = seen.any(1)
        p = torch.zeros_like(s)
        p[:, some] = torch.softmax(s[:, some], -1)
        big = scale * qb.norm(dim=-1).amax() * kb.norm(dim=-1).amax()
        es = U * (D + 2) * big + 32 * U + 4 * U * big
        eP, eS = es + h, 64 * U + Tk / 32 * U
        o_sum = p @ vb.abs()
        tol[0][b, :n] += ((eP + eS) * o_sum + hr * ob.abs() + tiny).transpose(0, 1)
        dp = gb @ vb.transpose(1, 2)
        delta = (gb * ob).sum(-1, keepdim=True)
        e_dp = (D + 2) * U * gb.norm(dim=-1, keepdim=True) * vb.norm(dim=-1).amax()
        e_delta = (gb.abs() * (hr * ob.abs() + (eP + eS) * o_sum)).sum(-1, keepdim=True) + (D + 2) * U * (gb.abs() * ob.abs()).sum(-1, keepdim=True)
        e_ds = p * ((dp - delta).abs() * (es + h + 4 * U) + e_dp + e_delta) + tiny / scale           # (rounded with the scale in it)
        ds = (p * (dp - delta)).abs()
        rows = n * G
        eR = 64 * U + rows / 32 * U
        tol[1][b, :n] += (scale * ((e_ds + eS * ds) @ kb.abs()) + hr * dq[b, :n].transpose(0, 1).abs() + tiny).transpose(0, 1)
        tk_ = scale * ((e_ds + eR * ds).transpose(1, 2) @ qb.abs())
        tv_ = (p * (eP + eR) + tiny).transpose(1, 2) @ gb.abs()
        tol[2][b, :m] += tk_.view(-1, G, m, D).sum(1).transpose(0, 1) + hr * dk[b, :m].abs() + tiny
        tol[3][b, :m] += tv_.view(-1, G, m, D).sum(1).transpose(0, 1) + hr * dv[b, :m].abs() + tiny
    return (out, dq, dk, dv), tol


def _check(names, got, want, tol):
    for name, a, b, t in zip(names, got, want, tol):
        err = (a.cpu().double() - b).abs()
        over = (err > t * 1.001 + 1e-30)
        assert not bool(over.any()), f"{name}: {int(over.sum())} of {over.numel()} outside, first {over.nonzero()[0].tolist()}, error {err[over][0]:.3e} bound {t[over][0]:.3e}"


def _run(q, k, v, g, **kw):
    from ppv_amd.attention import multihead_attention
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    cu = {n: (x.cuda() if torch.is_tensor(x) else x) for n, x in kw.items()}
    out = multihead_attention(*leaves, **cu)
    grads = torch.autograd.grad(out, leaves, g.cuda())
    with torch.no_grad():
        assert torch.equal(multihead_attention(*leaves, **cu), out)          # without the saved statistics: the same numbers
    again = torch.autograd.grad(multihead_attention(*leaves, **cu), leaves, g.cuda())
    assert all(torch.equal(a, b) for a, b in zip(again, grads))              # the same bits every time
    return (out.detach(),) + tuple(grads)


NAMES = ("out", "dq", "dk", "dv")


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B,Tq,Tk,H,Hkv,D", [
    (1, 1, 1, 1, 1, 8), (2, 3, 5, 2, 2, 16), (1, 31, 33, 1, 1, 32), (2, 52, 52, 4, 4, 64), (1, 64, 65, 2, 1, 40), (1, 65, 64, 2, 2, 128),
    (1, 129, 200, 1, 1, 72), (2, 1, 77, 4, 2, 64), (1, 7, 130, 8, 1, 32), (1, 200, 40, 2, 2, 96), (1, 130, 257, 6, 2, 128), (3, 40, 1, 2, 2, 24),
    (1, 300, 300, 1, 1, 64)])
def test_attention_value_and_gradients(B, Tq, Tk, H, Hkv, D, causal, dt):
    q, k, v, g = _inputs(B, Tq, Tk, H, Hkv, D, DT[dt], B + Tq * 3 + Tk * 5 + D)
    want, tol = _bounds(q, k, v, g, causal, None, None, None)
    _check(NAMES, _run(q, k, v, g, causal=causal), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("G", [1, 3])
def test_attention_lengths_and_what_lies_behind_them(G, causal, dt):
    """Sequences of every length, empty ones and lengths out of range among them; behind each end NaN and infinities, which reach nothing; rows that
    see nothing (more queries than keys, causal) are exact zeros, as are the gradients behind the ends."""
    from ppv_amd.attention import multihead_attention
    B, Tq, Tk, H, D = 8, 70, 66, 2 * G, 64
    q, k, v, g = _inputs(B, Tq, Tk, H, 2, D, DT[dt], 77)
    q_lens = torch.tensor([70, 1, 0, 33, 64, 70, 99, -4], dtype=torch.int32)
    k_lens = torch.tensor([66, 66, 5, 0, 1, 31, 65, 40], dtype=torch.int64)
    want, tol = _bounds(q, k, v, g, causal, q_lens.clamp(0, Tq), k_lens.clamp(0, Tk), 0.11)
    for b in range(B):
        n, m = min(max(int(q_lens[b]), 0), Tq), min(int(k_lens[b]), Tk)
        q[b, n:], g[b, n:] = float("nan"), float("inf")
        k[b, m:], v[b, m:] = float("nan"), float("-inf")
    got = _run(q, k, v, g, causal=causal, q_lens=q_lens, k_lens=k_lens, scale=0.11)
    _check(NAMES, got, want, tol)
    for b in range(B):
        n, m = min(max(int(q_lens[b]), 0), Tq), min(int(k_lens[b]), Tk)
        empty = ~orc.visible(Tq, Tk, n, m, causal).any(1)
        for t in (got[0][b].cpu()[empty], got[1][b].cpu()[empty], got[2][b].cpu()[m:], got[3][b].cpu()[m:]):
            assert torch.equal(t, torch.zeros_like(t))
    one = multihead_attention(q[:, :1].cuda(), k.cuda(), v.cuda(), causal=causal, k_lens=k_lens.cuda(), scale=0.11)   # a new token each
    ref, _ = orc.attention(q[:, :1].nan_to_num(0.0).double(), k.double(), v.double(), causal, None, k_lens, 0.11)
    ok = [b for b in range(B) if torch.isfinite(q[b, 0]).all()]
    assert torch.isfinite(one[ok]).all() and (one[ok].cpu().double() - ref[ok]).abs().max() < 0.02


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,Tq,Tk,H,Hkv,D", [(1, 1, 5000, 1, 1, 64), (2, 1, 3001, 8, 2, 128), (1, 2, 1500, 8, 8, 32), (1, 17, 2049, 4, 2, 64),
                                             (1, 100, 4100, 1, 1, 128), (3, 1, 1296, 4, 4, 56)])
def test_attention_few_rows_against_many_keys(B, Tq, Tk, H, Hkv, D, dt):
    """Where the keys are split over workgroups and joined, ragged, causal; the gradients too."""
    q, k, v, g = _inputs(B, Tq, Tk, H, Hkv, D, DT[dt], Tk)
    k_lens = torch.tensor([Tk - 700 * b for b in range(B)], dtype=torch.int32)
    want, tol = _bounds(q, k, v, g, True, None, k_lens, None)
    _check(NAMES, _run(q, k, v, g, causal=True, k_lens=k_lens), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,Tq,Tk,H,Hkv,D", [(1, 900, 40, 4, 1, 64), (1, 40, 1500, 1, 1, 128), (1, 1100, 1100, 1, 1, 48), (2, 500, 130, 8, 2, 32)])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_gradients_where_the_walk_is_split(B, Tq, Tk, H, Hkv, D, causal, dt):
    """Few tiles own rows or keys: the other axis is split over workgroups, ragged, so that some splits have nothing to do."""
    q, k, v, g = _inputs(B, Tq, Tk, H, Hkv, D, DT[dt], Tq + D)
    q_lens = torch.tensor([Tq - 333 * b - 7 for b in range(B)], dtype=torch.int32)
    k_lens = torch.tensor([Tk - 90 * b for b in range(B)], dtype=torch.int32)
    want, tol = _bounds(q, k, v, g, causal, q_lens, k_lens, None)
    _check(NAMES, _run(q, k, v, g, causal=causal, q_lens=q_lens, k_lens=k_lens), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_attention_large_scores(dt):
    """Scores of several hundred: the softmax is a choice of one key; equal scores share; a lone enormous score wins without an overflow."""
    q, k, v, g = _inputs(1, 64, 96, 2, 2, 64, DT[dt], 5, spread=6.0)
    k[0, 50] = k[0, 51]
    q[0, 7] = 0.0
    k[0, 90] *= 40.0
    want, tol = _bounds(q, k, v, g, False, None, None, None)
    got = _run(q, k, v, g)
    _check(NAMES, got, want, tol)
    assert all(torch.isfinite(t).all() for t in got)


@pytest.mark.gpu
def test_attention_strides_and_layouts():
    """[B,H,T,D] seen as [B,T,H,D], heads cut out of one projection, one key sequence shared by a batch (stride 0), odd head dimensions and
    addresses off a 16-byte boundary (copied), a transposed gradient, an expanded gradient."""
    from ppv_amd.attention import multihead_attention
    gen = torch.Generator().manual_seed(8)
    for dt in DT.values():
        B, T, H, D = 2, 45, 2, 64
        qkv = torch.randn(B, T, 3, H, D, generator=gen).to(dt)
        q, k, v = qkv.unbind(2)
        g = torch.randn(B, H, T, D, generator=gen).to(dt).transpose(1, 2)
        want, tol = _bounds(q, k, v, g, True, None, None, None)
        qkv_g = qkv.cuda().requires_grad_(True)
        out = multihead_attention(*qkv_g.unbind(2), causal=True)
        dall, = torch.autograd.grad(out, qkv_g, g.cuda().transpose(1, 2).contiguous().transpose(1, 2))
        _check(NAMES, (out.detach(),) + tuple(dall.unbind(2)), want, tol)
        assert out.is_contiguous()
        # [B, H, T, D]
        qt, kt, vt = (t.transpose(1, 2).contiguous().cuda().transpose(1, 2).requires_grad_(True) for t in (q, k, v))
        out = multihead_attention(qt, kt, vt, causal=True)
        _check(NAMES, (out.detach(),) + torch.autograd.grad(out, (qt, kt, vt), g.cuda()), want, tol)
        # keys shared by the batch: their gradient is the sum over it
        ks, vs = k[:1], v[:1]
        want, tol = _bounds(q, ks.expand(B, T, H, D), vs.expand(B, T, H, D), g, False, None, None, None)
        leaves = [t.cuda().requires_grad_(True) for t in (q, ks, vs)]
        out = multihead_attention(leaves[0], *(t.expand(B, T, H, D) for t in leaves[1:]))
        got = (out.detach(),) + torch.autograd.grad(out, leaves, g.cuda())
        hr = torch.finfo(dt).eps / 2
        sums = [x.sum(0, keepdim=True) for x in want[2:]]
        _check(NAMES, got, list(want[:2]) + sums, list(tol[:2]) + [t.sum(0, keepdim=True) + hr * s.abs() for t, s in zip(tol[2:], sums)])
        # any head dimension, any address
        for D2, off in ((37, 0), (1, 0), (64, 1), (120, 3)):
            q, k, v, g = _inputs(1, 20, 33, 2, 1, D2, dt, D2)
            def moved(t):
                buf = torch.zeros(t.numel() + off, dtype=dt, device="cuda")
                buf[off:] = t.reshape(-1).cuda()
                return buf[off:].view(t.shape).requires_grad_(True)
            leaves = [moved(t) for t in (q, k, v)]
            out = multihead_attention(*leaves)
            ones = torch.ones((), dtype=dt)
            want, tol = _bounds(q, k, v, ones.expand(g.shape), False, None, None, None)
            _check(NAMES, (out.detach(),) + torch.autograd.grad(out.sum(), leaves), want, tol)


@pytest.mark.gpu
def test_attention_gradients_of_a_scaled_loss_in_f16():
    """dO of several thousand (a loss multiplied for f16): dO V^T leaves f16's range, the gradients do not."""
    q, k, v, g = _inputs(1, 70, 90, 2, 2, 128, torch.float16, 12)
    g = g * 3000.0
    v = v * 2.0
    want, tol = _bounds(q, k, v, g, False, None, None, None)
    got = _run(q, k, v, g)
    assert (g.double().view(70, 2, 128).transpose(0, 1) @ v.double().view(90, 2, 128).permute(1, 2, 0)).abs().max() > 65504
    assert all(torch.isfinite(t).all() for t in got)
    _check(NAMES, got, want, tol)


@pytest.mark.gpu
def test_attention_empty_sizes():
    from ppv_amd.attention import multihead_attention
    q = torch.randn(2, 3, 4, 16, device="cuda", requires_grad=True)
    k = torch.zeros(2, 0, 2, 16, device="cuda", requires_grad=True)
    out = multihead_attention(q, k, k)
    out.sum().backward()
    assert torch.equal(out, torch.zeros_like(out)) and torch.equal(q.grad, torch.zeros_like(q)) and k.grad.shape == k.shape
    assert multihead_attention(q[:, :0], k, k).shape == (2, 0, 4, 16)
    assert multihead_attention(q[:0], k[:0], k[:0]).shape == (0, 3, 4, 16)


@pytest.mark.gpu
def test_attention_gradient_against_differences():
    q, k, v, g = _inputs(1, 9, 14, 4, 2, 24, torch.float32, 3)
    _, dq, dk, dv = _run(q, k, v, g, causal=True)
    gen = torch.Generator().manual_seed(4)
    for i, grad in enumerate((dq, dk, dv)):
        d = torch.randn((q, k, v)[i].shape, generator=gen).double()
        def f(sign):
            x = [t.double() for t in (q, k, v)]
            x[i] = x[i] + sign * 1e-5 * d
            return (orc.attention(*x, causal=True)[0] * g.double()).sum()
        slope = (f(1) - f(-1)) / 2e-5
        assert abs((grad.cpu().double() * d).sum() - slope) <= 1e-5 * (grad.cpu().double() * d).abs().sum()


@pytest.mark.gpu
def test_attention_on_another_stream_and_in_a_graph():
    from ppv_amd.attention import multihead_attention
    q, k, v, g = (t.cuda() for t in _inputs(2, 52, 300, 4, 4, 64, torch.bfloat16, 6))
    tok = q[:, :1].clone()
    lens = torch.tensor([300, 120], dtype=torch.int32, device="cuda")
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(multihead_attention(*leaves, causal=True, k_lens=lens), leaves, g)
        one = multihead_attention(tok, k, v, k_lens=lens)
    side.synchronize()
    assert torch.equal(one, multihead_attention(tok, k, v, k_lens=lens))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = multihead_attention(*leaves, causal=True, k_lens=lens)
        grads = torch.autograd.grad(out, leaves, g)
        one = multihead_attention(tok, k, v, k_lens=lens)
    for n in (300, 77, 12):
        lens.fill_(n)                                          # the lengths are read when the graph runs
        with torch.no_grad():
            leaves[0].mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        fresh = [t.detach().clone().requires_grad_(True) for t in leaves]
        want = multihead_attention(*fresh, causal=True, k_lens=lens)
        assert torch.equal(out, want) and torch.equal(one, multihead_attention(tok, k, v, k_lens=lens))
        assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(want, fresh, g)))


def test_attention_refusals():
    from ppv_amd.attention import multihead_attention
    q, k = torch.zeros(2, 3, 4, 16), torch.zeros(2, 5, 2, 16)
    for bad, err in (((q, k, k), RuntimeError),                                    # no CPU path
                     ((q[0], k, k), ValueError), ((q, k[0], k), ValueError), ((q.double(), k.double(), k.double()), TypeError),
                     ((q, k.bfloat16(), k), TypeError), ((q, k, k[:, :4]), ValueError), ((q, k[:1], k[:1]), ValueError),
                     ((q, k[..., :8], k[..., :8]), ValueError), ((q, torch.zeros(2, 5, 3, 16), torch.zeros(2, 5, 3, 16)), ValueError),
                     ((q, k[:, :, :0], k[:, :, :0]), ValueError), ((torch.zeros(1, 1, 1, 129),) * 3, ValueError), ((torch.zeros(1, 1, 1, 0),) * 3, ValueError)):
        with pytest.raises(err):
            multihead_attention(*bad)
    for kw in ({"scale": 0.0}, {"scale": -1.0}, {"scale": float("nan")}, {"scale": float("inf")}, {"q_lens": torch.zeros(3, dtype=torch.int32)},
               {"k_lens": torch.zeros(2)}, {"k_lens": [1, 2]}, {"k_lens": torch.zeros(2, 1, dtype=torch.int32)}):
        with pytest.raises(ValueError):
            multihead_attention(q, k, k, **kw)


def test_attention_entry_points_refuse():
    import ctypes
    from ppv_amd import _lib
    L = _lib.lib()
    NULL, SIZE, WORK = _lib.PPV_ERR_NULL, _lib.PPV_ERR_BAD_SIZE, _lib.PPV_ERR_WORKSPACE

    def args(**kw):
        a = _lib.Attention()
        for n in ("q", "k", "v", "out", "lse", "dout", "dq", "dk", "dv", "workspace"):
            setattr(a, n, 64)
        for n in ("sqb", "sqt", "sqh", "skb", "skt", "skh", "svb", "svt", "svh", "sgb", "sgt", "sgh"):
            setattr(a, n, 64)
        a.B, a.H, a.Hkv, a.Tq, a.Tk, a.D, a.dtype, a.causal, a.scale = 1, 2, 1, 4, 4, 32, 1, 0, 1.0
        for n, x in kw.items():
            setattr(a, n, x)
        return a

    assert L.ppv_attention_fwd(None, None) == NULL and L.ppv_attention_bwd(None, None) == NULL
    for n in ("q", "k", "v", "out"):
        assert L.ppv_attention_fwd(args(**{n: None}), None) == NULL
    for n in ("lse", "dout", "dq", "dk", "dv"):
        assert L.ppv_attention_bwd(args(**{n: None}), None) == NULL
    assert L.ppv_attention_bwd(args(workspace=None), None) == WORK
    assert L.ppv_attention_fwd(args(Tk=100000, workspace=None), None) == WORK
    for kw in ({"B": 0}, {"H": 3, "Hkv": 2}, {"Hkv": 0}, {"Tq": 0}, {"Tk": -1}, {"D": 0}, {"D": 136}, {"D": 20}, {"dtype": 3}, {"scale": 0.0},
               {"scale": float("nan")}, {"sqt": 12}, {"skb": -64}, {"q": 72}, {"out": 68}):
        assert L.ppv_attention_fwd(args(**kw), None) == SIZE, kw
    for kw in ({"sgt": 12}, {"dout": 72}, {"dk": 8}):
        assert L.ppv_attention_bwd(args(**kw), None) == SIZE, kw
    assert L.ppv_attention_fwd_workspace_bytes(1, 3, 2, 1, 1, 8, 1) == 0 and L.ppv_attention_bwd_workspace_bytes(0, 1, 1, 1, 1, 8, 1) == 0


@pytest.mark.gpu
def test_attention_is_differentiable_once_and_keeps_what_it_needs():
    from ppv_amd.attention import multihead_attention
    q, k, v, g = (t.cuda() for t in _inputs(1, 5, 9, 2, 2, 16, torch.float32, 1))
    q.requires_grad_(True)
    want, = torch.autograd.grad(multihead_attention(q, k, v), q, g)
    dq, = torch.autograd.grad(multihead_attention(q, k, v), q, g, create_graph=True)
    assert torch.equal(dq, want)
    with pytest.raises(RuntimeError, match="differentiable once"):
        dq.sum().backward()
    lens = torch.tensor([4], dtype=torch.int32, device="cuda")
    out = multihead_attention(q, k, v, k_lens=lens)
    lens.fill_(9)                                                  # lengths are operands: changed under a pending backward pass, they are refused
    with pytest.raises(RuntimeError):
        out.sum().backward()


def test_attention_entry_points_refuse_more_than_a_launch_holds():
    """Workgroups beyond 2^24 (work items are counted in 32 bits), key tiles beyond 2^30, a workspace off 16 bytes: refused before anything is launched."""
    from ppv_amd import _lib
    L = _lib.lib()

    def args(**kw):
        a = _lib.Attention()
        for n in ("q", "k", "v", "out", "lse", "dout", "dq", "dk", "dv", "workspace"):
            setattr(a, n, 64)
        a.B, a.H, a.Hkv, a.Tq, a.Tk, a.D, a.dtype, a.causal, a.scale = 1, 1, 1, 1, 1, 8, 1, 0, 1.0
        for n, x in kw.items():
            setattr(a, n, x)
        return a

    for kw in ({"B": 1 << 24}, {"B": (1 << 24) - 7}, {"B": 1 << 20, "Tq": 2048}, {"B": 200, "Tk": 1 << 28}):
        assert L.ppv_attention_fwd(args(**kw), None) == _lib.PPV_ERR_BAD_SIZE, kw
        assert L.ppv_attention_bwd(args(**kw), None) == _lib.PPV_ERR_BAD_SIZE, kw
    assert L.ppv_attention_bwd(args(B=1 << 20, Tk=2048), None) == _lib.PPV_ERR_BAD_SIZE
    assert L.ppv_attention_fwd(args(Tk=100000, workspace=72), None) == _lib.PPV_ERR_BAD_SIZE


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("Tq", [1, 130])
def test_attention_reads_a_cache_whose_offsets_pass_32_bits(Tq, dt):
    """A cache [T, layers * heads * D ...] read in place through its token stride: the same bits as from a packed copy."""
    from ppv_amd.attention import multihead_attention
    T, D, step = 4200, 64, 1 << 20                              # offsets up to 4.4e9 elements
    store = torch.empty(T * step, dtype=dt, device="cuda")
    gen = torch.Generator().manual_seed(7)
    wide = store.view(1, T, step)
    k, v = wide[..., :2 * D].unflatten(2, (2, D)), wide[..., step - 2 * D:].unflatten(2, (2, D))
    packed = [torch.randn(1, T, 2, D, generator=gen).to(dt).cuda() for _ in range(2)]
    k.copy_(packed[0])
    v.copy_(packed[1])
    assert (k.stride(1), v.stride(1)) == (step, step)
    q, g = (torch.randn(1, Tq, 4, D, generator=gen).to(dt).cuda() for _ in range(2))
    runs = []
    for a, b in ((k, v), packed):
        leaves = [t.detach().requires_grad_(True) for t in (q, a, b)]
        out = multihead_attention(*leaves, causal=True)
        runs.append((out,) + torch.autograd.grad(out, leaves, g))
    assert all(torch.equal(x, y) for x, y in zip(*runs))
    far = wide[:, ::8, :2 * D].unflatten(2, (2, D))            # a token stride of 2^23: copied
    assert torch.equal(multihead_attention(q, far, far), multihead_attention(q, far.contiguous(), far.contiguous()))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B,Tq,Tk,H,Hkv,D", [(2, 1, 3001, 8, 2, 80), (1, 40, 1500, 1, 1, 96), (1, 900, 40, 4, 1, 88), (1, 300, 300, 2, 2, 96),
                                             (4, 52, 130, 8, 4, 80), (64, 130, 70, 4, 4, 72)])
def test_attention_of_head_dimensions_between_64_and_96(B, Tq, Tk, H, Hkv, D, causal, dt):
    """Staged in rows of 128, multiplied as 96: with the keys split, the backward walks split, neither, and whole tiles of every direction."""
    q, k, v, g = _inputs(B, Tq, Tk, H, Hkv, D, DT[dt], Tq + D)
    k_lens = torch.tensor([max(0, Tk - 5 * b) for b in range(B)], dtype=torch.int32)
    want, tol = _bounds(q, k, v, g, causal, None, k_lens, None)
    _check(NAMES, _run(q, k, v, g, causal=causal, k_lens=k_lens), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,Tq,Tk,H", [(8, 100, 4096, 32), (8, 40, 4096, 32), (64, 1, 8192, 8), (1, 1, 60000, 1)])
def test_attention_of_one_large_score_among_many_small_ones(B, Tq, Tk, H, dt):
    """One key whose weight is 2^25.2 times each other's, in a value of 0 among values of 1: what is left is the sum of the small weights, w = (Tk - 1)
    e^-17.5.  As numbers of f16 beside a largest of 1 each of them would round to zero; beside one of 2^7 they are 2^-18.2, off by at most 2^-25, 2^-6.8 of
    their value if all the same way.  bf16: half a step, 2^-8.  The values' sum is exact in f32 but for a chain of Tk / 32 additions."""
    from ppv_amd.attention import multihead_attention
    D, t = 16, DT[dt]
    q, k, v = torch.zeros(B, Tq, H, D), torch.zeros(B, Tk, H, D), torch.ones(B, Tk, H, D)
    q[..., 0], k[:, 0, :, 0], v[:, 0] = 1.0, 17.5, 0.0
    q, k, v = (x.to(t).cuda() for x in (q, k, v))
    w = (Tk - 1) * math.exp(-17.5)
    want = w / (1.0 + w)
    rel = {"f32": 0.0, "bf16": 2.0 ** -8, "f16": 2.0 ** -6.8}[dt] + torch.finfo(t).eps / 2 + (Tk / 32 + 64 + 16 * 17.5) * U
    with torch.no_grad():
        out = multihead_attention(q, k, v, scale=1.0)
        first = multihead_attention(q, k.flip(1), v.flip(1), scale=1.0)          # the large one last
    for o in (out, first):
        assert ((o.double() - want).abs() <= want * rel + (2.0 ** -25 if dt == "f16" else 0.0)).all(), (float(o.min()), float(o.max()), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("Tq,Tk,H,Hkv", [(1500, 300, 2, 2), (700, 200, 16, 2), (64, 64, 32, 1), (3000, 20, 1, 1)])
def test_attention_gradient_of_values_with_small_weights(Tq, Tk, H, Hkv, dt):
    """Every row gives one key e^17.5 times each other's weight (2^-25.2); their dV is the sum of it over the rows, w = rows e^-17.5 / (1 + (Tk - 1) e^-17.5): a
    scaled loss would not help numbers of f16 that round to zero beside 1; beside 2^12 they are 2^-13.2, no subnormal ones.  dQ and dK are 0: V is the same for all keys."""
    D, t = 16, DT[dt]
    q, k, v, g = torch.zeros(1, Tq, H, D), torch.zeros(1, Tk, Hkv, D), torch.ones(1, Tk, Hkv, D), torch.ones(1, Tq, H, D)
    q[..., 0], k[:, 7, :, 0] = 1.0, 17.5
    out, dq, dk, dv = _run(*(x.to(t) for x in (q, k, v, g)), scale=1.0)
    rows = Tq * H // Hkv
    w = rows * math.exp(-17.5) / (1.0 + (Tk - 1) * math.exp(-17.5))
    h = torch.finfo(t).eps / 2
    rel = h + (0.0 if dt == "f32" else h) + (rows / 32 + 64 + 16 * 17.5 + 32) * U
    small = torch.cat([dv[:, :7], dv[:, 8:]], 1).double()
    assert ((small - w).abs() <= w * rel + (2.0 ** -25 if dt == "f16" else 0.0)).all(), (float(small.min()), float(small.max()), w)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("Tq,Tk,H,Hkv", [(40, 33, 2, 2), (200, 300, 4, 2), (1, 3000, 1, 1)])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_rows_whose_scores_all_overflow(Tq, Tk, H, Hkv, causal, dt):
    """A row that gives every key it sees a score of minus infinity (products of 1e25 and -1e25) is like one that sees nothing: zeros, and it takes no part in the
    gradients.  The other rows and the keys are as without it."""
    D = 32
    q, k, v, g = _inputs(1, Tq, Tk, H, Hkv, D, DT[dt], Tq + Tk)
    row = Tq // 2
    q[..., 0], k[..., 0] = 0.0, -1e25
    q[0, row, :, 0] = 1e25
    out, dq, dk, dv = _run(q, k, v, g, causal=causal)
    for t in (out[0, row], dq[0, row]):
        assert torch.equal(t, torch.zeros_like(t))
    assert all(torch.isfinite(t).all() for t in (out, dq, dk, dv))
    k2, g2, q2 = k.clone(), g.clone(), q.clone()
    k2[..., 0], g2[0, row], q2[0, row] = 0.0, 0.0, 0.0
    want, tol = _bounds(q2, k2, v, g2, causal, None, None, None)
    keep = [i for i in range(Tq) if i != row]
    # (dq of the row's first dimension is a sum of dS times -1e25: not finite in general, left out for the others, as is dk's, a sum of dS times 0 or 1e25)
    _check(("out", "dq", "dk", "dv"), (out[:, keep], dq[:, keep, :, 1:], dk[..., 1:], dv),
           (want[0][:, keep], want[1][:, keep, :, 1:], want[2][..., 1:], want[3]), (tol[0][:, keep], tol[1][:, keep, :, 1:], tol[2][..., 1:], tol[3]))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("B,Tq,Tk,H,Hkv,D", [(2, 1, 700, 4, 2, 64), (3, 5, 300, 8, 2, 128), (1, 32, 2000, 2, 2, 96), (2, 9, 9, 4, 1, 80), (2, 100, 30, 2, 2, 64), (1, 300, 300, 2, 1, 8),
                                             (2, 70, 200, 3, 3, 32), (1, 4, 5000, 1, 1, 40)])
def test_attention_of_few_rows_or_keys_rounds_its_results_alone(B, Tq, Tk, H, Hkv, D, dt):
    """Where the matrix products are not what takes the time (up to 32 rows to a key head: value and dQ; up to 32 keys: dK and dV; D up to 32: dQ) P and dS enter them in two
    terms of the 16-bit type, off by h^2 of their value (f16 also by half a step of its subnormals, 2^-25, beside a P of at least 2^7 in the value's product,
    2^12 P in dV's and dS itself in dQ's and dK's).  The rest is that of f32 operands, and the result's one rounding."""
    t = DT[dt]
    q, k, v, g = _inputs(B, Tq, Tk, H, Hkv, D, t, Tq + 7 * Tk + D)
    want, tol = _bounds(q.float(), k.float(), v.float(), g.float(), False, None, None, None)
    h, tiny, G, scale = torch.finfo(t).eps / 2, 2.0 ** -25 if dt == "f16" else 0.0, H // Hkv, D ** -0.5
    qh, gh = (x.double().transpose(1, 2) for x in (q, g))                                          # [B, H, Tq, D]
    kh, vh = (x.double().transpose(1, 2).repeat_interleave(G, 1) for x in (k, v))
    p = torch.softmax(qh @ kh.transpose(2, 3) * scale, -1)
    ds = (p * (gh @ vh.transpose(2, 3) - (gh * (p @ vh)).sum(-1, keepdim=True)) * scale).abs()
    heads = lambda x: x.view(B, Hkv, G, Tk, D).sum(2)
    few, keys = Tq * G <= 32, Tk <= 32
    # D = rowsum(dO O) is the forward pass' O, whose P has one term where there are more rows: off by h sum |dO| sum P |V|, and dS by P times that
    d_off = 0.0 if few else h * scale * p * (gh.abs() * (p @ vh.abs())).sum(-1, keepdim=True)
    two = [(h * h * p + 2.0 ** -7 * tiny) @ vh.abs(), (h * h * ds + d_off + tiny) @ kh.abs(), heads((h * h * ds + d_off + tiny).transpose(2, 3) @ qh.abs()),
           heads((h * h * p + 2.0 ** -12 * tiny).transpose(2, 3) @ gh.abs())]
    got = _run(q, k, v, g)
    for name, a, b, s, x, on in zip(NAMES, got, want, tol, two, (few, few or D <= 32, keys, keys)):
        if on:
            _check((name,), (a,), (b,), (s + x.transpose(1, 2) + h * b.abs() + tiny,))
