"""Cases and plain forms of the transformer operators that stand next to the captioner: layer norm, multi-head attention (both with
their backward passes) and an AdamW step over a list of tensors with its states in 32 or in 8 bits.

``run`` computes a case in elementary torch operations in 32 bits, or, where ``own`` is true, through ``ppv_amd``'s entry points;
``exact`` computes it in 64 bits from the definitions, written apart from ``run``."""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
F32, F64 = torch.float32, torch.float64

# hyper-parameters of the optimiser cases: a usual AdamW run, some steps after its start
LR, BETAS, EPS, DECAY, STEP0, SEED = 4e-4, (0.9, 0.999), 1e-8, 1e-2, 20, 7
BLOCK = 256               # elements of a tensor that share a scale in the 8-bit states
MIN_8BIT = 4096           # smaller tensors (biases, norm weights) keep 32-bit states


# ---------------------------------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one decoding step of a beam search over 5 hypotheses, width 512 (the captioner's): what it costs to call at all
        {"name": "norm_token", "op": "norm", "rows": 5, "cols": 512, "dtype": "f32", "train": False},
        # a batch of 128 captions padded to 52 tokens, width 512
        {"name": "norm_captions", "op": "norm", "rows": 128 * 52, "cols": 512, "dtype": "bf16", "train": True},
        # the 36 x 36 pixels of 128 encoded images, 2048 channels
        {"name": "norm_pixels", "op": "norm", "rows": 128 * 1296, "cols": 2048, "dtype": "bf16", "train": True},
        # rows that start at odd addresses and end inside a vector
        {"name": "norm_ragged", "op": "norm", "rows": 4099, "cols": 1367, "dtype": "f16", "train": True},
        # one token of 5 hypotheses looks at the 1296 pixels of an image
        {"name": "attend_token", "op": "attend", "B": 5, "Tq": 1, "Tk": 1296, "H": 8, "Hkv": 8, "D": 64, "dtype": "bf16",
         "causal": False, "ragged": False, "train": False},
        # one new token against a long history, key and value heads shared by four query heads
        {"name": "attend_history", "op": "attend", "B": 4, "Tq": 1, "Tk": 65536, "H": 32, "Hkv": 8, "D": 128, "dtype": "bf16",
         "causal": True, "ragged": True, "train": False},
        # captions attend to themselves in training: short, padded, 1024 (image, head) pairs
        {"name": "attend_captions", "op": "attend", "B": 128, "Tq": 52, "Tk": 52, "H": 8, "Hkv": 8, "D": 64, "dtype": "bf16",
         "causal": True, "ragged": True, "train": True},
        # captions attend to the pixels of their images in the decoder's own precision
        {"name": "attend_pixels", "op": "attend", "B": 32, "Tq": 52, "Tk": 1296, "H": 8, "Hkv": 8, "D": 64, "dtype": "f32",
         "causal": False, "ragged": False, "train": True},
        # the 64 x 64 positions of a 512 x 512 image's feature map attend in raster order
        {"name": "attend_raster", "op": "attend", "B": 2, "Tq": 4096, "Tk": 4096, "H": 16, "Hkv": 16, "D": 128, "dtype": "bf16",
         "causal": True, "ragged": False, "train": True},
        # a head's few small tensors: the launch is the cost
        {"name": "adamw_head", "op": "adamw", "bits": 32, "tensors": "head"},
        # the captioner's decoder, 32-bit states
        {"name": "adamw_decoder", "op": "adamw", "bits": 32, "tensors": "decoder"},
        # ResNet-101 and the decoder together, 8-bit states
        {"name": "adamw_caption_8bit", "op": "adamw", "bits": 8, "tensors": "resnet101+decoder"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["norm", "attend", "attend", "adamw"])
    if op == "norm":
        cols = _log(rng, 8, 12000)               # (under four columns a row's gradient is its rounding)
        rows = _log(rng, 1, min(200000, 300000000 // cols))
        return {"op": "norm", "rows": rows, "cols": cols, "dtype": rng.choice(["f32", "bf16", "f16"]), "train": rng.random() < 0.7}
    if op == "adamw":
        return {"op": "adamw", "bits": rng.choice([8, 32]),
                "tensors": "random:%d:%d:%d" % (_log(rng, 1, 300), _log(rng, 16, 4000000), rng.randrange(1 << 30))}
    train = rng.random() < 0.6
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    D = rng.choice([8, 24, 32, 40, 64, 64, 80, 96, 128, 128])
    group = rng.choice([1, 1, 1, 2, 4, 8])
    Hkv = rng.choice([1, 2, 4, 8])
    H = Hkv * group
    if train:
        Tk = _log(rng, 8, 2600)                  # (with one key to see, the gradients of scores are their rounding)
        Tq = Tk if rng.random() < 0.5 else _log(rng, 1, 2600)
        most = 500000000
    else:
        Tq = rng.choice([1, 1, 1, _log(rng, 2, 16), _log(rng, 1, 2600)])
        Tk = _log(rng, 1, 60000)
        most = 250000000
    B = _log(rng, 1, 128)
    while B > 1 and (B * H * Tq * Tk > most or B * Hkv * Tk * D > 200000000):
        B = (B + 1) // 2
    while H * Tq * Tk > most:
        Tq = (Tq + 1) // 2
    return {"op": "attend", "B": B, "Tq": Tq, "Tk": Tk, "H": H, "Hkv": Hkv, "D": D, "dtype": dtype, "causal": rng.random() < 0.5,
            "ragged": rng.random() < 0.5, "train": train}


def _shapes(spec):
    """The tensors of an optimiser case, as element counts."""
    if spec.startswith("random:"):
        count, largest, seed = (int(v) for v in spec.split(":")[1:])
        r = random.Random(seed)
        return [_log(r, 1, largest) for _ in range(count)]
    got = []
    for part in spec.split("+"):
        if part == "head":                       # two norms, a projection's bias and a small projection
            got += [512, 512, 512, 512, 512, 512 * 64, 64]
        elif part == "decoder":                  # soft-attention LSTM captioner: 512 / 512 / 512, 2048 channels, 9490 words
            got += [512 * 2048, 512, 512 * 512, 512, 512, 1, 9490 * 512, 2048 * 2560, 2048 * 512, 2048, 2048, 512 * 2048, 512,
                    512 * 2048, 512, 2048 * 512, 2048, 9490 * 512, 9490]
        elif part == "resnet101":
            got += [64 * 3 * 49, 64, 64]
            width = 64
            for planes, blocks in ((64, 3), (128, 4), (256, 23), (512, 3)):
                for b in range(blocks):
                    got += [planes * width, planes, planes, planes * planes * 9, planes, planes, 4 * planes * planes, 4 * planes, 4 * planes]
                    if b == 0:
                        got += [4 * planes * width, 4 * planes, 4 * planes]
                    width = 4 * planes
    return got


def _lengths(case):
    """(query lengths, key lengths) of an attention case, as lists: spread evenly from a quarter of the longest to the longest."""
    B, Tq, Tk = case["B"], case["Tq"], case["Tk"]
    if not case["ragged"]:
        return [Tq] * B, [Tk] * B
    def even(T):
        lo = (T + 3) // 4
        return [lo + (T - lo) * (i + 1) // B for i in range(B)]
    return even(Tq), even(Tk)


def _pairs(case):
    """(query, key) pairs of one head that the mask leaves."""
    total = 0
    for n, m in zip(*_lengths(case)):
        if not case["causal"]:
            total += n * m
        else:                                    # row i sees m - n + i + 1 keys, where that is positive
            first = m - n + 1
            skip = max(0, -first + 1)
            rows = max(0, n - skip)
            a = first + skip
            total += rows * a + rows * (rows - 1) // 2
    return total


def work(case):
    if case["op"] == "norm":
        n, size = case["rows"] * case["cols"], SIZE[case["dtype"]]
        passes = 2 + (2 if case["train"] else 0)               # x, y; and g, dx
        return {"bytes": n * size * passes + case["cols"] * (16 if case["train"] else 8), "flops": n * (18 if case["train"] else 8)}
    if case["op"] == "adamw":
        bytes_, flops = 0, 0
        for n in _shapes(case["tensors"]):
            eight = case["bits"] == 8 and n >= MIN_8BIT
            bytes_ += n * (16 if eight else 28) + (16 * -(-n // BLOCK) if eight else 0)
            flops += n * (40 if eight else 15)
        return {"bytes": bytes_, "flops": flops}
    qs, ks = _lengths(case)
    size = SIZE[case["dtype"]]
    rows = sum(qs) * case["H"] * case["D"] * size
    keys = sum(ks) * case["Hkv"] * case["D"] * size
    whole = case["B"] * case["Tq"] * case["H"] * case["D"] * size
    whole_k = case["B"] * case["Tk"] * case["Hkv"] * case["D"] * size
    product = 2 * _pairs(case) * case["H"] * case["D"]
    if not case["train"]:
        return {"bytes": rows + 2 * keys + whole, "flops": 2 * product}
    return {"bytes": 2 * rows + 2 * keys + 2 * whole + 2 * whole_k, "flops": 7 * product}


# --------------------------------------------------------------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def prepare(case, seed):
    gen = _gen(seed)

    def normal(*shape, dtype=F32, scale=1.0):
        return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)

    if case["op"] == "norm":
        dt = DTYPES[case["dtype"]]
        rows, cols, train = case["rows"], case["cols"], case["train"]
        x = normal(rows, cols) * (0.5 + torch.rand((rows, 1), generator=gen, device="cuda")) + normal(rows, 1)
        state = {"case": case, "x": x.to(dt), "weight": 1.0 + normal(cols, scale=0.1), "bias": normal(cols, scale=0.1)}
        if train:
            state["g"] = normal(rows, cols, dtype=dt)
            for k in ("x", "weight", "bias"):
                state[k].requires_grad_(True)
        return state
    if case["op"] == "attend":
        dt = DTYPES[case["dtype"]]
        B, Tq, Tk, H, Hkv, D = (case[k] for k in ("B", "Tq", "Tk", "H", "Hkv", "D"))
        state = {"case": case, "q": normal(B, Tq, H, D, dtype=dt), "k": normal(B, Tk, Hkv, D, dtype=dt), "v": normal(B, Tk, Hkv, D, dtype=dt),
                 "q_lens": None, "k_lens": None}
        if case["ragged"]:
            order = torch.randperm(B, generator=torch.Generator().manual_seed(int(seed)))
            qs, ks = _lengths(case)
            state["q_lens"] = torch.tensor(qs, dtype=torch.int32)[order].cuda()
            state["k_lens"] = torch.tensor(ks, dtype=torch.int32)[order].cuda()
        if case["train"]:
            state["g"] = normal(B, Tq, H, D, dtype=dt)
            for k in "qkv":
                state[k].requires_grad_(True)
        return state
    counts = _shapes(case["tensors"])
    total = sum(counts)
    flat_p, flat_g = normal(total, scale=0.05), normal(total, scale=1e-3)
    m, root = normal(total, scale=3e-4), (normal(total, scale=1e-3).abs() + 1e-6)
    state = {"case": case, "step": STEP0, "p": flat_p, "g": flat_g, "params": [], "moments": []}
    small = sum(n for n in counts if case["bits"] == 32 or n < MIN_8BIT)
    large = total - small
    blocks = sum(-(-n // BLOCK) for n in counts if not (case["bits"] == 32 or n < MIN_8BIT))
    if small:
        state["m32"], state["v32"] = torch.empty(small, device="cuda"), torch.empty(small, device="cuda")
    if large:
        state["m8"], state["r8"] = (torch.empty(large, dtype=torch.float8_e4m3fn, device="cuda") for _ in range(2))
        state["m8_scale"], state["r8_scale"] = torch.empty(blocks, device="cuda"), torch.empty(blocks, device="cuda")
    at = at_s = at_l = at_b = 0
    for n in counts:
        p = flat_p[at:at + n].requires_grad_(True)
        p.grad = flat_g[at:at + n]
        state["params"].append(p)
        if case["bits"] == 32 or n < MIN_8BIT:
            mom = {"m": state["m32"][at_s:at_s + n], "v": state["v32"][at_s:at_s + n]}
            mom["m"].copy_(m[at:at + n])
            mom["v"].copy_(root[at:at + n].square())
            at_s += n
        else:
            b = -(-n // BLOCK)
            mom = {"m": state["m8"][at_l:at_l + n], "r": state["r8"][at_l:at_l + n],
                   "ms": state["m8_scale"][at_b:at_b + b], "rs": state["r8_scale"][at_b:at_b + b]}
            for name, x in (("m", m), ("r", root)):
                x = x[at:at + n]
                scale = _block_scale(x)
                mom[name].copy_((x / _spread(scale, n)).to(torch.float8_e4m3fn))
                mom[name + "s"].copy_(scale)
            at_l, at_b = at_l + n, at_b + b
        state["moments"].append(mom)
        at += n
    return state


# ----------------------------------------------------------------------------------------------------------------------- plain forms

def _norm(state):
    x, w, b = (state[k].detach().float() for k in ("x", "weight", "bias"))
    dt = state["x"].dtype
    centred = x - x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + 1e-5)
    hat = centred * rstd
    y = (hat * w + b).to(dt)
    if "g" not in state:
        return {"y": y}
    g = state["g"].float()
    gw = g * w
    dx = rstd * (gw - gw.mean(1, keepdim=True) - hat * (gw * hat).mean(1, keepdim=True))
    return {"y": y, "dx": dx.to(dt), "dweight": (g * hat).sum(0), "dbias": g.sum(0)}


def _visible(case, q_lens, k_lens):
    """[B or 1, Tq, Tk] truth values, or None where every pair counts: row i of a sequence with n queries and m keys sees key j < m if
    i < n and, where causal, j <= i + m - n."""
    if q_lens is None and not case["causal"]:
        return None
    i = torch.arange(case["Tq"], device="cuda").view(1, -1, 1)
    j = torch.arange(case["Tk"], device="cuda").view(1, 1, -1)
    n = q_lens.view(-1, 1, 1).long() if q_lens is not None else torch.full((1, 1, 1), case["Tq"], device="cuda")
    m = k_lens.view(-1, 1, 1).long() if k_lens is not None else torch.full((1, 1, 1), case["Tk"], device="cuda")
    seen = (i < n) & (j < m)
    return seen & (j - i <= m - n) if case["causal"] else seen


def _attend(state):
    case = state["case"]
    B, Tq, Tk, H, Hkv, D = (case[k] for k in ("B", "Tq", "Tk", "H", "Hkv", "D"))
    G, dt, scale = H // Hkv, state["q"].dtype, D ** -0.5

    def heads(x):                                # [B, T, H, D] -> [B * Hkv, G * T, D] in 32 bits
        x = x.detach().float()
        return x.view(B, x.shape[1], Hkv, -1, D).permute(0, 2, 3, 1, 4).reshape(B * Hkv, -1, D)

    def back(x, T):
        return x.view(B, Hkv, -1, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, -1, D).to(dt)

    q, k, v = heads(state["q"]), heads(state["k"]), heads(state["v"])
    s = torch.bmm(q, k.transpose(1, 2).contiguous()) * scale
    seen = _visible(case, state["q_lens"], state["k_lens"])
    if seen is not None:
        s = s.view(B, Hkv * G, Tq, Tk)
        s = torch.where(seen.unsqueeze(1), s, float("-inf")).view(B * Hkv, G * Tq, Tk)
    top = s.amax(2, keepdim=True)
    p = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(2, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = torch.bmm(p, v)
    if "g" not in state:
        return {"out": back(out, Tq)}
    g = heads(state["g"])
    dv = torch.bmm(p.transpose(1, 2).contiguous(), g)
    dp = torch.bmm(g, v.transpose(1, 2).contiguous())
    ds = p * (dp - (g * out).sum(2, keepdim=True)) * scale
    dq = torch.bmm(ds, k)
    dk = torch.bmm(ds.transpose(1, 2).contiguous(), q)
    return {"out": back(out, Tq), "dq": back(dq, Tq), "dk": back(dk, Tk), "dv": back(dv, Tk)}


def _block_scale(x):
    """Power-of-two scales of the blocks of 256 elements of x: 2 ** (floor(log2(largest magnitude)) - 7)."""
    n = x.numel()
    padded = torch.zeros(-(-n // BLOCK) * BLOCK, device=x.device)
    padded[:n] = x.abs()
    exponent = (padded.view(-1, BLOCK).amax(1).view(torch.int32) >> 23) - 127
    return ((exponent.clamp(min=-118) - 7 + 127) << 23).view(F32)


def _spread(scale, n):
    return scale.repeat_interleave(BLOCK)[:n]


def _dither(step, tensor, n):
    """Two 16-bit numbers for each of a tensor's n elements in this step: a 32-bit integer hash of the element's place."""
    low = 0xFFFFFFFF
    key = (SEED * 0x9E3779B1 + step * 0x85EBCA77 + tensor * 0xC2B2AE3D) & low
    h = (torch.arange(n, device="cuda") * 0x9E3779B1 + key) & low
    h = ((h ^ (h >> 16)) * 0x7FEB352D) & low
    h = ((h ^ (h >> 15)) * 0x846CA68B) & low
    h = h ^ (h >> 16)
    return h & 0xFFFF, h >> 16


def _eight_bits(x, scale, dither):
    """x / scale as the e4m3 value below or above it, the upper one with the probability of its nearness: 20 bits of the mantissa go."""
    a = x.abs() / scale                          # exact: scales are powers of two
    up = (dither * 16 + 8).to(torch.int32)
    normal = ((a.view(torch.int32) + up) >> 20 << 20).view(F32)
    small = torch.floor(a * 512.0 + up.to(F32) * 2.0 ** -20) / 512.0
    return torch.copysign(torch.where(a >= 2.0 ** -6, normal, small), x)


def _adamw(state):
    state["step"] += 1
    t, (b1, b2) = state["step"], BETAS
    rate, undo = LR / (1 - b1 ** t), 1 / math.sqrt(1 - b2 ** t)

    def one(i, p, mom):
        p, g, n = p.detach(), p.grad, p.numel()
        eight = "r" in mom
        if eight:
            m = mom["m"].float() * _spread(mom["ms"], n)
            root = mom["r"].float() * _spread(mom["rs"], n)
            v = root * root
        else:
            m, v = mom["m"], mom["v"]
        m = m + (g - m) * (1 - b1)
        v = v * b2 + (g * (1 - b2)) * g
        root = torch.sqrt(v)
        p.copy_(p * (1 - LR * DECAY) - (m / (root * undo + EPS)) * rate)
        if not eight:
            mom["m"].copy_(m)
            mom["v"].copy_(v)
            return
        for_m, for_r = _dither(t, i, n)
        mom["ms"].copy_(_block_scale(m))
        mom["rs"].copy_(_block_scale(root))
        mom["m"].copy_(_eight_bits(m, _spread(mom["ms"], n), for_m).to(torch.float8_e4m3fn))
        r = _eight_bits(root, _spread(mom["rs"], n), for_r)
        mom["r"].copy_(torch.where((r == 0) & (root > 0), 2.0 ** -9, r).to(torch.float8_e4m3fn))

    [one(i, p, mom) for i, (p, mom) in enumerate(zip(state["params"], state["moments"]))]
    return {k: state[k] for k in ("p", "m32", "v32", "m8", "m8_scale", "r8", "r8_scale") if k in state}


# ------------------------------------------------------------------------------------------------------------------------------- run

def run(state):
    op = state["case"]["op"]
    if not own:
        return {"norm": _norm, "attend": _attend, "adamw": _adamw}[op](state)
    import ppv_amd  # noqa: F401
    if op == "norm":
        from ppv_amd.nn_ops import layer_norm
        x, w, b = state["x"], state["weight"], state["bias"]
        y = layer_norm(x, w, b, eps=1e-5)
        if "g" not in state:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (x, w, b), state["g"])
        return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}
    if op == "attend":
        from ppv_amd.attention import multihead_attention
        q, k, v = state["q"], state["k"], state["v"]
        out = multihead_attention(q, k, v, causal=state["case"]["causal"], q_lens=state["q_lens"], k_lens=state["k_lens"])
        if "g" not in state:
            return {"out": out}
        dq, dk, dv = torch.autograd.grad(out, (q, k, v), state["g"])
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    if "optimiser" not in state:                 # a program makes its optimiser once and keeps it
        from ppv_amd.optim import AdamW
        opt = AdamW(state["params"], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=state["case"]["bits"], min_8bit_size=MIN_8BIT,
                    seed=SEED)
        for p, mom in zip(state["params"], state["moments"]):
            names = {"m": "exp_avg", "v": "exp_avg_sq", "r": "exp_avg_sq_root", "ms": "exp_avg_scale", "rs": "exp_avg_sq_root_scale"}
            opt.state[p].update({"step": float(state["step"]), **{names[k]: x for k, x in mom.items()}})
        state["optimiser"] = opt
    state["optimiser"].step()
    return {k: state[k] for k in ("p", "m32", "v32", "m8", "m8_scale", "r8", "r8_scale") if k in state}


# ------------------------------------------------------------------------------------------------------------- 64 bits, from the definition

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "norm":
        x, w, b = (state[k].detach().double().requires_grad_(True) for k in ("x", "weight", "bias"))
        mean = x.mean(1, keepdim=True)
        y = (x - mean) / torch.sqrt(x.var(1, unbiased=False, keepdim=True) + 1e-5) * w + b
        if not case["train"]:
            return {"y": y.detach()}
        dx, dw, db = torch.autograd.grad(y, (x, w, b), state["g"].double())
        return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}
    if case["op"] == "attend":
        return _exact_attend(case, state)
    return _exact_adamw(case, state)


def _exact_attend(case, state):
    G = case["H"] // case["Hkv"]
    outs = {"out": []}
    for b in range(case["B"]):                   # a sequence at a time: scores of one are what the card holds easily
        n = case["Tq"] if state["q_lens"] is None else int(state["q_lens"][b])
        m = case["Tk"] if state["k_lens"] is None else int(state["k_lens"][b])
        q, k, v = (state[x].detach()[b].double().requires_grad_(case["train"]) for x in "qkv")
        with torch.set_grad_enabled(case["train"]):
            qh = q[:n].transpose(0, 1).contiguous()                                      # [H, n, D]
            kh = k[:m].transpose(0, 1).repeat_interleave(G, 0).contiguous()
            vh = v[:m].transpose(0, 1).repeat_interleave(G, 0).contiguous()
            s = torch.bmm(qh, kh.transpose(1, 2).contiguous()) / math.sqrt(case["D"])
            first = 0                                                                    # rows before it see nothing
            if case["causal"]:
                first = min(n, max(0, n - m))
                s = s + torch.triu(torch.full((n, m), float("-inf"), dtype=F64, device="cuda"), diagonal=m - n + 1)
            o = torch.bmm(torch.softmax(s[:, first:], 2), vh).transpose(0, 1)            # [n - first, H, D]
            out = torch.zeros((case["Tq"], case["H"], case["D"]), dtype=F64, device="cuda")
            out = torch.cat([out[:first], o, out[n:]])
        outs["out"].append(out.detach())
        if case["train"]:
            for name, x in zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), state["g"][b].double())):
                outs.setdefault(name, []).append(x)
    return {k: torch.stack(x) for k, x in outs.items()}


def _exact_adamw(case, state):
    t, (b1, b2) = STEP0 + 1, BETAS
    got = {}

    def note(name, x):
        got.setdefault(name, []).append(x)

    for i, (p, mom) in enumerate(zip(state["params"], state["moments"])):
        w, g, n = p.detach().double(), p.grad.double(), p.numel()
        if "r" in mom:
            m = mom["m"].double() * mom["ms"].double().repeat_interleave(BLOCK)[:n]
            v = (mom["r"].double() * mom["rs"].double().repeat_interleave(BLOCK)[:n]) ** 2
        else:
            m, v = mom["m"].double(), mom["v"].double()
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
        w = w - LR * DECAY * w - LR * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + EPS)
        note("p", w)
        if "r" not in mom:
            note("m32", m)
            note("v32", v)
            continue
        for name, x, dither in zip(("m8", "r8"), (m, v.sqrt()), _dither(t, i, n)):
            whole = torch.cat([x.abs(), torch.zeros(-n % BLOCK, dtype=F64, device="cuda")]).view(-1, BLOCK).amax(1)
            scale = torch.exp2(torch.floor(torch.log2(whole)).clamp(min=-118) - 7)
            a = x.abs() / scale.repeat_interleave(BLOCK)[:n]
            ulp = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
            code = torch.floor(a / ulp + (dither.double() + 0.5) / 65536) * ulp
            if name == "r8":
                code = torch.where((code == 0) & (x > 0), 2.0 ** -9, code)
            note(name, code * x.sign())
            note(name + "_scale", scale)
    return {k: torch.cat(x) for k, x in got.items()}
