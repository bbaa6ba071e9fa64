"""ppv_amd.optim.AdamW (csrc/adamw.hip), moments in 32 and in 8 bits.  The step is a stated sequence of f32 operations, so the oracle's values
(oracle/transformer.py, f32 on the CPU) are reproduced bit for bit; against 64 bits the bounds count roundings."""
import copy
import math
import pickle

import pytest
import torch

from oracle import transformer as orc

U = 2.0 ** -24
SIZES = [(64,), (5,), (4095,), (4096,), (4099,), (64, 3, 7, 7), (300, 257), (1,), (12288,), (7, 4096)]


def _tensors(seed, sizes, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g) * scale for s in sizes]


def _oracle_state(n, eight):
    z = lambda k: torch.zeros(k)
    b = -(-n // 256)
    return {"m": z(n), "r": z(n), "ms": z(b), "rs": z(b)} if eight else {"m": z(n), "v": z(n)}


def _same(opt, p, st):
    got = opt.state[p]
    if "r" in st:
        pairs = [(got["exp_avg"].float(), st["m"]), (got["exp_avg_sq_root"].float(), st["r"]), (got["exp_avg_scale"], st["ms"]),
                 (got["exp_avg_sq_root_scale"], st["rs"])]
    else:
        pairs = [(got["exp_avg"], st["m"]), (got["exp_avg_sq"], st["v"])]
    for a, b in pairs:
        a = a.cpu().reshape(-1)
        assert torch.equal(torch.nan_to_num(a, nan=-12345.0), torch.nan_to_num(b, nan=-12345.0))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("wd,betas", [(0.0, (0.9, 0.999)), (1e-2, (0.8, 0.95))])
def test_adamw_reproduces_the_oracle_bit_for_bit(bits, wd, betas):
    from ppv_amd.optim import AdamW
    ref = [t.reshape(-1) for t in _tensors(0, SIZES)]
    got = [torch.nn.Parameter(t.cuda()) for t in _tensors(0, SIZES)]
    st = [_oracle_state(r.numel(), bits == 8 and r.numel() >= 4096) for r in ref]
    count = [0] * len(ref)
    opt = AdamW(got, lr=1e-2, betas=betas, weight_decay=wd, state_bits=bits, seed=11)
    flat = torch.zeros(sum(r.numel() for r in ref) + 3, device="cuda")             # gradients are slices of one buffer, few of them aligned
    for step in range(6):
        grads = _tensors(100 + step, SIZES, scale=10.0 ** (-step))                 # (the blocks' maxima move through powers of two)
        grads[4][:] = 0.0 if step < 2 else grads[4]                                # no gradient at all at first
        off = 1
        for i, (q, g) in enumerate(zip(got, grads)):
            view = flat[off:off + g.numel()].view_as(g)
            view.copy_(g)
            off += g.numel()
            q.grad = None if (step == 3 and i in (3, 6)) else view                # a parameter without a gradient keeps its own count
        opt.step()
        for i, (r, g) in enumerate(zip(ref, grads)):
            if got[i].grad is None:
                continue
            count[i] += 1
            orc.adamw_step(r, g.reshape(-1), st[i], count[i], place=i, lr=1e-2, betas=betas, weight_decay=wd, seed=11)
            assert opt.state[got[i]]["step"] == count[i]
            _same(opt, got[i], st[i])
            assert torch.equal(got[i].detach().cpu().reshape(-1), r), (step, i)
    assert (bits == 8) == any(s.get("exp_avg_scale") is not None for s in opt.state.values())


@pytest.mark.gpu
@pytest.mark.parametrize("wd", [0.0, 1e-2])
def test_adamw_32_against_64_bits_and_torch(wd):
    """Five steps from zero moments against the formula in f64.  A step rounds m and v at most 3 times each on operands no larger than
    |m| + |g| (v: 3 |v|), the errors shrink by the betas: after t steps at most 4 t u (|m| + max|g|) and 4 t u v.  The update lr m / r^ inherits
    their relative errors plus 8 of its own roundings; p is rounded twice per step."""
    from ppv_amd.optim import AdamW
    p0 = _tensors(1, [(513,), (70, 70)])
    got = [torch.nn.Parameter(t.cuda()) for t in p0]
    tor = [torch.nn.Parameter(t.double()) for t in p0]
    opt, ref = AdamW(got, lr=1e-2, weight_decay=wd), torch.optim.AdamW(tor, lr=1e-2, weight_decay=wd, foreach=False)
    for step in range(5):
        for q, t, g in zip(got, tor, _tensors(50 + step, [(513,), (70, 70)])):
            q.grad, t.grad = g.cuda(), g.double()
        opt.step()
        ref.step()
    t = 5
    for q, r in zip(got, tor):
        a, b = opt.state[q], ref.state[r]
        assert ((a["exp_avg"].cpu().double() - b["exp_avg"]).abs() <= 4 * t * U * (b["exp_avg"].abs() + 5.0)).all()
        assert ((a["exp_avg_sq"].cpu().double() - b["exp_avg_sq"]).abs() <= 4 * t * U * b["exp_avg_sq"] + 1e-30).all()
        # |update| <= lr * 10 (|m^| <= sqrt(v^) / sqrt(1 - b1 ...) of a few steps), m's absolute error seen through 1 / r^ >= 1 / 5
        small = torch.sqrt(b["exp_avg_sq"] / (1 - 0.999 ** t)).clamp(min=1e-3)
        tol = 2 * t * U * r.detach().abs() + t * 1e-2 * (16 * t * U * 10 + 4 * t * U * 10 / small)
        assert ((q.detach().cpu().double() - r.detach()).abs() <= tol).all()


@pytest.mark.gpu
def test_adamw_loads_aligned_or_not_and_leaves_the_neighbours():
    """Parameters that are slices of a buffer at every offset: the elements between them are not touched."""
    from ppv_amd.optim import AdamW
    buf, grad = torch.randn(40000, device="cuda"), torch.randn(40000, device="cuda")
    before = buf.clone()
    spans = [(1, 4096), (4099, 5000), (9103, 1), (9106, 8192), (17299, 12287), (29589, 9000)]
    ps = []
    for at, n in spans:
        p = buf[at:at + n].requires_grad_(True)
        p.grad = grad[at:at + n]
        ps.append(p)
    AdamW(ps, lr=1e-2, state_bits=8).step()
    inside = torch.zeros(40000, dtype=torch.bool)
    for at, n in spans:
        inside[at:at + n] = True
    b, a = before.cpu(), buf.detach().cpu()
    assert torch.equal(a[~inside], b[~inside]) and (a[inside] != b[inside]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_state_survives_reload_and_pickle(bits):
    """Rolled back to a saved state the same steps give the same bits; the saved state is not what later steps write to."""
    from ppv_amd.optim import AdamW
    sizes = [(300,), (64, 128), (4099,)]
    got = [torch.nn.Parameter(t.cuda()) for t in _tensors(0, sizes)]
    opt = AdamW(got, lr=1e-2, state_bits=bits, seed=3)

    def run(o, a, b):
        for s in range(a, b):
            for q, g in zip(got, _tensors(200 + s, sizes)):
                q.grad = g.cuda()
            o.step()

    run(opt, 0, 2)
    sd = opt.state_dict()
    kept = copy.deepcopy(sd)
    w = [q.detach().clone() for q in got]
    run(opt, 2, 5)
    want = [q.detach().clone() for q in got]
    fresh = AdamW(got, lr=1e-2, state_bits=bits, seed=3)
    for o in (opt, fresh, pickle.loads(pickle.dumps(AdamW([torch.nn.Parameter(torch.zeros(1))], state_bits=bits, seed=3)))):
        if o is not opt and o is not fresh:
            assert (o.state_bits, o.seed, o.min_8bit_size) == (bits, 3, 4096) and o._tables == {}
            continue
        with torch.no_grad():
            for q, x in zip(got, w):
                q.copy_(x)
        o.load_state_dict(kept)
        run(o, 2, 5)
        assert all(torch.equal(a, b.detach()) for a, b in zip(want, got))
    again = copy.deepcopy(opt.state_dict())                    # `kept` itself is as it was saved
    assert kept["state"][0]["step"] == 2.0 and again["state"][0]["step"] == 5.0
    if bits == 8:
        st = kept["state"][1]
        assert st["exp_avg"].dtype == torch.float8_e4m3fn and st["exp_avg"].shape == (64, 128) and st["exp_avg_scale"].shape == (32,)
        assert opt.state[got[1]]["exp_avg"].dtype == torch.float8_e4m3fn
    else:
        t = torch.optim.AdamW(got, lr=1e-2)
        t.load_state_dict(kept)                                # interchangeable with torch's
        back = AdamW(got, lr=1e-2)
        back.load_state_dict(t.state_dict())
        assert torch.equal(back.state[got[2]]["exp_avg_sq"], kept["state"][2]["exp_avg_sq"])


@pytest.mark.gpu
def test_adamw_8bit_values_that_are_not_finite_stay_where_they_are():
    from ppv_amd.optim import AdamW
    n = 8192
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    opt = AdamW([p], lr=1e-2, state_bits=8, seed=1)
    ref, st = torch.zeros(n), _oracle_state(n, True)
    for step in range(3):
        g = torch.randn(n, generator=torch.Generator().manual_seed(step))
        if step == 1:
            g[5], g[700], g[4000] = math.inf, math.nan, -math.inf
        p.grad = g.cuda()
        opt.step()
        orc.adamw_step(ref, g, st, step + 1, lr=1e-2, seed=1)
        _same(opt, p, st)
    bad = ~torch.isfinite(p.detach().cpu())
    assert bad.nonzero().squeeze(1).tolist() == [5, 700, 4000]
    assert torch.equal(p.detach().cpu()[~bad], ref[~bad])


@pytest.mark.gpu
def test_adamw_on_two_streams_and_with_moving_gradients():
    """The descriptor table follows the stream and the gradients' addresses."""
    from ppv_amd.optim import AdamW
    sizes = [(5000,), (64, 64)]
    a = [torch.nn.Parameter(t.cuda()) for t in _tensors(0, sizes)]
    b = [torch.nn.Parameter(t.cuda()) for t in _tensors(0, sizes)]
    oa, ob = AdamW(a, lr=1e-2, state_bits=8), AdamW(b, lr=1e-2, state_bits=8)
    side, keep = torch.cuda.Stream(), []
    for step in range(6):
        grads = [g.cuda() for g in _tensors(step, sizes)]
        keep.append(grads)                                      # new addresses every step
        for p, g in zip(a, grads):
            p.grad = g
        oa.step()
        for p, g in zip(b, grads):
            p.grad = g.clone()
        torch.cuda.synchronize()
        if step % 2:
            with torch.cuda.stream(side):
                ob.step()
            side.synchronize()
        else:
            ob.step()
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and len(ob._tables) == 1


def test_8bit_second_moment_follows_a_constant_gradient():
    """Why the rounding is stochastic (the format alone, on the CPU): with g = 1 and beta2 = 0.999 the second moment is 1 - 0.999^t.  A step of the
    root is at most 2^-3 of it and moves it by at most its own share d <= 0.5e-3 / r^2, so rounding adds at most (2^-3 r) (d r) per step to
    E[r^2], against a decay of 1e-3: at most 6.3 % too much in v.  To the nearest, the root stops where half a step of e4m3 (>= 2^-5 of it)
    is more than an update: below 0.2."""
    n, steps = 2048, 2500
    for nearest in (False, True):
        st, p, g = _oracle_state(n, True), torch.zeros(n), torch.ones(n)
        if nearest:
            keep = orc.dither
            orc.dither = lambda seed, step, place, k: (torch.full((k,), 32767), torch.full((k,), 32767))
        try:
            for t in range(1, steps + 1):
                orc.adamw_step(p, g, st, t, lr=0.0)
        finally:
            if nearest:
                orc.dither = keep
        v = ((st["r"] * orc.spread(st["rs"], n)).double() ** 2).mean().item()
        want = 1 - 0.999 ** steps
        if nearest:
            assert v < 0.2
        else:
            assert 0.98 * want <= v <= 1.063 * want + 0.02


def test_adamw_refusals():
    from ppv_amd.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(4))
    for kw in ({"amsgrad": True}, {"maximize": True}, {"capturable": True}):
        with pytest.raises(NotImplementedError):
            AdamW([p], **kw)
    for kw in ({"state_bits": 16}, {"lr": -1.0}, {"betas": (1.0, 0.9)}, {"betas": (0.9, -0.1)}, {"eps": -1e-8}, {"weight_decay": -0.1},
               {"min_8bit_size": -1}):
        with pytest.raises(ValueError):
            AdamW([p], **kw)
    with pytest.raises(TypeError):
        AdamW([p], nesterov=True)
    o = AdamW([p])
    o.step()                                                    # nothing has a gradient: nothing to do
    p.grad = torch.zeros(4)
    with pytest.raises(NotImplementedError):
        o.step()                                                # no CPU path


def test_adamw_entry_point_refuses():
    import ctypes
    from ppv_amd import _lib
    L, p = _lib.lib(), ctypes.c_void_p(64)
    NULL, SIZE = _lib.PPV_ERR_NULL, _lib.PPV_ERR_BAD_SIZE
    hyper = (1e-3, 0.9, 0.999, 1e-8, 0.0)
    assert L.ppv_adamw_multi(None, 1, 1, *hyper, 1.0, 0, None) == NULL
    assert L.ppv_adamw_multi(p, 0, 1, *hyper, 1.0, 0, None) == SIZE
    assert L.ppv_adamw_multi(p, 1, 0, *hyper, 1.0, 0, None) == SIZE
    assert L.ppv_adamw_multi(p, 1, 1, *hyper, 0.0, 0, None) == SIZE
    assert L.ppv_adamw_multi(p, 1, 1, 1e-3, 1.0, 0.999, 1e-8, 0.0, 1.0, 0, None) == SIZE
    assert L.ppv_adamw_multi(p, 1, 1, 1e-3, 0.9, 1.5, 1e-8, 0.0, 1.0, 0, None) == SIZE


@pytest.mark.gpu
def test_adamw_refuses_on_the_gpu():
    from ppv_amd.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(8, 8, device="cuda"))
    p.grad = torch.zeros(8, 8, device="cuda").t()
    with pytest.raises(NotImplementedError):
        AdamW([p]).step()
    p.grad = torch.zeros(8, 8, device="cuda")
    o = AdamW([p])
    o.step()
    o.state[p]["exp_avg"] = torch.zeros(3, device="cuda")
    with pytest.raises(ValueError):
        o.step()
    e = torch.nn.Parameter(torch.zeros(0, device="cuda"))
    e.grad = torch.zeros(0, device="cuda")
    o = AdamW([e])
    o.step()
    assert o.state[e]["step"] == 1.0
    q = torch.nn.Parameter(torch.zeros(8, device="cuda"))
    q.grad = torch.ones(8, device="cuda")
    o = AdamW([q])
    o.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    refused = False
    with torch.cuda.graph(graph):
        scratch = torch.empty(4, device="cuda").zero_()         # (a capture that holds something)
        try:
            o.step()
        except RuntimeError:
            refused = True
    assert refused and o.state[q]["step"] == 1.0 and scratch.numel() == 4


def test_adamw_refuses_a_group_that_asks_for_more():
    """amsgrad and maximize of a single group, or of a state that was another optimiser's: refused, not left out."""
    from ppv_amd.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.ones(4)
    for name in ("amsgrad", "maximize"):
        with pytest.raises(NotImplementedError, match="maximize"):
            AdamW([{"params": [p], name: True}]).step()
        o = AdamW([p])
        o.load_state_dict(torch.optim.AdamW([p], **{name: True}).state_dict())
        with pytest.raises(NotImplementedError, match="maximize"):
            o.step()


@pytest.mark.filterwarnings("ignore")
def test_adamw_refuses_a_parameter_twice():
    from ppv_amd.optim import AdamW
    p, q = torch.nn.Parameter(torch.zeros(4)), torch.nn.Parameter(torch.zeros(4))
    with pytest.raises(ValueError, match="twice"):
        AdamW([p, q, p])
    o = AdamW([p])
    with pytest.raises(ValueError):
        o.add_param_group({"params": [q, q]})
    assert len(o.param_groups) == 1
    with pytest.raises(ValueError):
        o.add_param_group({"params": [q, p]})                   # (torch's own check)


@pytest.mark.gpu
def test_adamw_refuses_parameters_that_share_memory():
    from ppv_amd.optim import AdamW
    x = torch.zeros(100, device="cuda")
    a, b, c = torch.nn.Parameter(x[:60]), torch.nn.Parameter(x[59:90]), torch.nn.Parameter(x[60:])
    for t in (a, b, c):
        t.grad = torch.ones_like(t)
    with pytest.raises(ValueError, match="share memory"):
        AdamW([c, a, b]).step()
    AdamW([c, a], lr=0.5, weight_decay=0.0).step()              # neighbours
    assert (x + 0.5).abs().max() < 1e-6


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_of_a_tensor_beyond_32_bits(bits):
    from ppv_amd.optim import AdamW
    n = (1 << 32) + 4099
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    p.grad = torch.ones(n, device="cuda")
    AdamW([p], lr=0.5, weight_decay=0.0, state_bits=bits).step()
    lo, hi = p.detach().aminmax()
    assert lo == hi and abs(float(lo) + 0.5) < 1e-6


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_steps_that_start_from_the_last_one_are_those_that_do_not(bits):
    """A step that finds everything as the last one left it goes a shorter way: the same bits as an optimiser that forgets, whatever is changed in between:
    a gradient that is missing or comes, a replaced moment or state, a changed number, a new group, other memory behind a parameter."""
    from ppv_amd.optim import AdamW
    gen = torch.Generator().manual_seed(3)
    first = [torch.randn(n, generator=gen) for n in (300, 5, 5000, 64)]
    grads = [[torch.randn(len(t), generator=gen) for t in first] for _ in range(12)]

    def run(forget):
        ps = [torch.nn.Parameter(t.clone().cuda()) for t in first]
        o = AdamW(ps[:3], lr=1e-2, state_bits=bits, seed=5)
        for k in range(12):
            for p, g in zip(ps, grads[k]):
                p.grad = g.cuda()
            if k in (3, 4):
                ps[1].grad = None                               # its count stays behind: two launches from here on
            if k == 6:
                o.state[ps[1]]["step"] = o.state[ps[0]]["step"] # one again
            if k == 7:
                o.state[ps[0]]["exp_avg"] = o.state[ps[0]]["exp_avg"].clone()
                o.state[ps[0]][list(o.state[ps[0]])[1]].copy_(o.state[ps[0]]["exp_avg"])
            if k == 8:
                o.state[ps[2]] = {n: (t.clone() if torch.is_tensor(t) else t) for n, t in o.state[ps[2]].items()}
                o.add_param_group({"params": [ps[3]], "lr": 1e-3})
            if k == 9:
                ps[0].data = ps[0].data.clone()
                o.param_groups[0]["lr"] = 3e-3
            if k == 10:
                del o.param_groups[0]["params"][1]
                for st in (o.state[ps[0]], o.state[ps[2]]):
                    st["step"] = 20.0
            if forget:
                o._last.clear()
                o._tables.clear()
            o.step()
        return [p.detach() for p in ps] + [t for p in ps for t in o.state[p].values()]

    for a, b in zip(run(False), run(True)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)) if torch.is_tensor(a) else a == b


@pytest.mark.gpu
def test_adamw_refuses_a_state_whose_memory_was_swapped():
    from ppv_amd.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(64, device="cuda"))
    p.grad = torch.ones(64, device="cuda")
    o = AdamW([p])
    o.step()
    o.state[p]["exp_avg_sq"].data = torch.zeros(3, device="cuda")
    with pytest.raises(ValueError):
        o.step()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_raises_the_version_of_what_it_writes(bits):
    """Parameters and moments are written through their addresses; autograd's check of saved tensors and every cache of a weight's layout go by the
    version counter.  The short way of a step counts too; what a step does not write keeps its version."""
    from ppv_amd.optim import AdamW
    ps = [torch.nn.Parameter(t.cuda()) for t in _tensors(0, [(300,), (64, 128), (5,), (0,)])]
    opt = AdamW(ps, lr=1e-2, state_bits=bits)
    for step in range(4):
        for p in ps[:2] + ps[3:]:
            p.grad = torch.ones_like(p)
        was = [p._version for p in ps]
        held = [(t, t._version) for p in ps for t in opt.state[p].values() if torch.is_tensor(t)] if step else []
        opt.step()
        assert ps[0]._version > was[0] and ps[1]._version > was[1] and ps[2]._version == was[2]
        assert all(t._version > v for t, v in held if t.numel()) and all(p.grad is None or p.grad._version == 0 for p in ps)
        assert len(held) == (0 if step == 0 else 2 + 2 + (4 if bits == 8 else 2))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_modules_follow_adamw(bits):
    """Two steps on a block whose convolutions keep their weights' layouts: value and gradients are those of a new block with the same weights."""
    from ppv_amd.optim import AdamW
    from ppv_amd.stargan_blocks import ResBlk
    torch.manual_seed(0)
    blk = ResBlk(64, 128, normalize=True, downsample=True).cuda()
    x = torch.randn(2, 64, 16, 16, device="cuda", requires_grad=True)
    opt = AdamW(blk.parameters(), lr=3e-2, state_bits=bits, min_8bit_size=256)
    seen = []
    for step in range(3):
        out = blk(x)
        new = copy.deepcopy(blk)                                # its parameters are other tensors: no layout of theirs is kept
        for q in new.parameters():
            q.grad = None
        want = new(x)
        assert torch.equal(out, want), step
        assert all(not torch.equal(out, s) for s in seen)
        seen.append(out.detach())
        g = torch.autograd.grad(out.square().sum(), [x] + list(blk.parameters()))
        h = torch.autograd.grad(want.square().sum(), [x] + list(new.parameters()))
        assert all(torch.equal(a, b) for a, b in zip(g, h)), step
        for p, d in zip(blk.parameters(), g[1:]):
            p.grad = d
        opt.step()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_between_forward_and_backward_is_an_error(bits):
    """The backward pass would mix the weights of two steps."""
    from ppv_amd.nn_ops import layer_norm
    from ppv_amd.optim import AdamW
    x, w = torch.randn(6, 512, device="cuda", requires_grad=True), torch.nn.Parameter(torch.ones(512, device="cuda"))
    opt = AdamW([w], lr=1e-2, state_bits=bits, min_8bit_size=256)
    for _ in range(2):
        w.grad = torch.ones_like(w)
        y = layer_norm(x, w)
        opt.step()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_adamw_loads_a_state_that_knows_neither_amsgrad_nor_maximize():
    """A state written before a group had these names (torch.optim.AdamW fills them in on loading, too)."""
    from ppv_amd.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(4))
    for drop in (["amsgrad"], ["maximize"], ["amsgrad", "maximize"]):
        o, sd = AdamW([p]), AdamW([p], lr=0.25).state_dict()
        for name in drop:
            del sd["param_groups"][0][name]
        o.load_state_dict(sd)
        o.step()                                                # (nothing has a gradient)
        assert o.param_groups[0]["lr"] == 0.25 and not o.param_groups[0]["amsgrad"] and not o.param_groups[0]["maximize"]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_refused_step_leaves_the_list_as_it_was(bits):
    """A moment's memory is swapped, the step refused, the memory put back: the next step is the one that would have come."""
    from ppv_amd.optim import AdamW
    runs = []
    for swap in (False, True):
        ps = [torch.nn.Parameter(t.cuda()) for t in _tensors(0, [(300,), (64, 128), (70,)])]
        o = AdamW(ps, lr=1e-2, state_bits=bits, min_8bit_size=256)
        for step in range(3):
            for p in ps:
                p.grad = torch.full_like(p, 0.5 + step) if step == 0 else p.grad
            if swap and step == 2:
                st = o.state[ps[1]]["exp_avg"]
                keep = st.data
                st.data = torch.zeros(3, device="cuda")
                with pytest.raises(ValueError):
                    o.step()
                st.data = keep
            o.step()
        runs.append([p.detach() for p in ps])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_refuses_a_state_that_became_shorter_or_another_type_in_its_place(bits):
    """The same address does not make it the same tensor: a shorter one may lie where the old one lay."""
    from ppv_amd.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(1024, device="cuda"))
    p.grad = torch.ones(1024, device="cuda")
    o = AdamW([p], state_bits=bits, min_8bit_size=256)
    o.step()
    for name, t in list(o.state[p].items()):
        if not torch.is_tensor(t):
            continue
        keep = t.data
        for other in (keep[:3], keep.view(torch.uint8)[:keep.numel()].view(torch.bool), keep.as_strided(keep.shape, (0,))):
            t.data = other
            assert t.data_ptr() == keep.data_ptr()
            with pytest.raises(ValueError, match="does not belong"):
                o.step()
            t.data = keep
    o.step()
    assert o.state[p]["step"] == 2.0


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_refuses_memory_that_comes_to_be_shared(bits):
    """Tensors of one launch that overlap would be written by two workgroups in any order: refused at the first step and at any later one that finds other
    addresses, parameters, moments and scales alike; so is a gradient that lies in what the launch writes, but for a parameter's own."""
    from ppv_amd.optim import AdamW
    buf = torch.zeros(4096, device="cuda")
    ps = [torch.nn.Parameter(torch.zeros(1024, device="cuda")) for _ in range(3)]
    o = AdamW(ps, lr=1e-2, weight_decay=0.0, state_bits=bits, min_8bit_size=256)
    for p in ps:
        p.grad = torch.ones_like(p)
    o.step()
    names = [n for n, t in o.state[ps[0]].items() if torch.is_tensor(t)]
    assert len(names) == (4 if bits == 8 else 2)

    def refused(put, back):
        put()
        for _ in range(2):
            with pytest.raises(ValueError, match="share memory"):
                o.step()
        back()

    keep = [p.data for p in ps]
    def two(a, b):
        ps[0].data, ps[2].data = a, b
    def own():
        for p, t in zip(ps, keep):
            p.data = t
    refused(lambda: two(buf[:1024], buf[1023:2047]), own)
    refused(lambda: two(buf[1:1025], buf[:1024]), own)
    for n in names:                                             # one moment for two parameters
        st = o.state[ps[2]]
        mine = st[n]
        refused(lambda: st.__setitem__(n, o.state[ps[0]][n]), lambda: st.__setitem__(n, mine))
    g = [p.grad for p in ps]
    refused(lambda: setattr(ps[1], "grad", ps[0].data), lambda: setattr(ps[1], "grad", g[1]))
    two(buf[:1024], keep[2])
    refused(lambda: setattr(ps[0], "grad", buf[1:1025]), lambda: setattr(ps[0], "grad", g[0]))
    own()
    ps[1].grad = g[0]                                           # one gradient for two, neighbours, a gradient that is the parameter: in order
    two(buf[:1024], buf[1024:2048])
    o.step()
    before = ps[0].detach().clone()
    ps[0].grad = ps[0].data
    o.step()
    assert o.state[ps[0]]["step"] == 3.0 and torch.isfinite(ps[0]).all() and not torch.equal(ps[0], before)
    assert torch.equal(buf[2048:], torch.zeros(2048, device="cuda"))
