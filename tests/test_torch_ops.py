"""The autograd nodes of lib/ppv_torch.so (csrc/torch/torch_ops.cpp) behind layer_norm and multihead_attention: what torch does with an operator
besides calling it.  Their kernels go by addresses, so each of these is refused, never left out of the result.  (The refusals come before
anything else in the native functions: they are tested there without a GPU, and through the public entry points with one.)"""
import pytest
import torch
import torch.autograd.forward_ad as fw


def _native():
    from ppv_amd import _lib
    T = _lib.torch_ops()
    return (lambda x, w=None, b=None: T.layer_norm(x, w, b, 1e-5)), (lambda q, k, v: T.attention(q, k, v, None, None, False, 0.25))


def _public():
    from ppv_amd.attention import multihead_attention
    from ppv_amd.nn_ops import layer_norm
    return layer_norm, multihead_attention


WHERE = [("cpu", _native), pytest.param("cuda", _public, marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device,entries", WHERE)
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_tangents_are_refused(device, entries, grad):
    norm, attend = entries()
    x, w = torch.ones(4, 64, device=device, requires_grad=grad), torch.ones(64, device=device)
    q = torch.ones(1, 4, 2, 16, device=device, requires_grad=grad)
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))
        for call in (lambda: norm(dual(x)), lambda: norm(x, dual(w)), lambda: norm(x, w, dual(w)), lambda: norm(x, None, dual(w)),
                     lambda: attend(dual(q), q, q), lambda: attend(q, dual(q), q), lambda: attend(q, q, dual(q))):
            with torch.no_grad() if not grad else torch.enable_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call()


@pytest.mark.gpu
def test_forward_mode_tangents_of_the_gradient_are_refused():
    """Forward over reverse: a tangent that comes in with the gradient of the result."""
    norm, attend = _public()
    x, q = torch.ones(4, 64, device="cuda", requires_grad=True), torch.ones(1, 4, 2, 16, device="cuda", requires_grad=True)
    for leaf, y in ((x, norm(x)), (q, attend(q, q, q))):
        with fw.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(y, leaf, fw.make_dual(torch.ones_like(y), torch.ones_like(y)))
        with fw.dual_level():                                   # a level without tangents changes nothing
            want, = torch.autograd.grad((attend(q, q, q) if leaf is q else norm(x)).sum(), leaf)
        assert torch.isfinite(want).all()


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("device,entries", WHERE)
@pytest.mark.parametrize("grad", [False, True])
def test_what_records_calls_is_refused(device, entries, grad):
    """A trace would hold the allocation of the result and nothing else: replayed, whatever lay in that memory."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    norm, attend = entries()
    x, q = torch.ones(4, 64, device=device, requires_grad=grad), torch.ones(1, 4, 2, 16, device=device, requires_grad=grad)
    for call, t in ((lambda a: norm(a), x), (lambda a: attend(a, a, a), q)):
        with pytest.raises(NotImplementedError, match="torch.jit.trace"):
            torch.jit.trace(call, (t,), check_trace=False)
        for pre in (False, True):
            with pytest.raises(NotImplementedError, match="does not see the kernel"):
                make_fx(call, pre_dispatch=pre)(t)
        with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(NotImplementedError, match="does not see the kernel"):
            call(t)


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore")
def test_compiled_callers_run_the_operators_themselves():
    """torch.compile breaks its graph at the operators: the same numbers, value and gradient."""
    norm, attend = _public()
    torch.manual_seed(0)
    x = torch.randn(3, 5, 2, 32, device="cuda", requires_grad=True)
    f = lambda a: attend(norm(a * 2.0), a, a, causal=True) + 1.0
    g = torch.compile(f, backend="eager")
    for _ in range(2):
        want, got = f(x), g(x)
        assert torch.equal(want, got)
        assert torch.equal(*(torch.autograd.grad(y.square().sum(), x)[0] for y in (want, got)))


class _Logged(torch.Tensor):
    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("device,entries", WHERE)
def test_tensors_that_stand_for_others_are_refused(device, entries):
    norm, attend = entries()
    x, q = torch.ones(4, 64, device=device), torch.ones(2, 1, 4, 2, 16, device=device)
    for call in (lambda: torch.vmap(lambda a: norm(a.view(1, 64)))(x), lambda: torch.func.grad(lambda a: norm(a).sum())(x),
                 lambda: torch.func.jvp(lambda a: norm(a), (x,), (x,)), lambda: torch.vmap(lambda a: attend(a, a, a))(q),
                 lambda: torch.vmap(lambda a: attend(q[0], a, q[0]))(q), lambda: torch.func.vjp(lambda a: attend(a, a, a), q[0]),
                 lambda: norm(x.as_subclass(_Logged)), lambda: norm(x, x[0].as_subclass(_Logged)), lambda: attend(q[0], q[0], q[0].as_subclass(_Logged))):
        with pytest.raises(NotImplementedError, match="do not reach the kernel"):
            call()


@pytest.mark.gpu
def test_negations_still_to_be_done_are_done():
    """z.conj().imag and the like are the old memory with a note to negate it: as argument, parameter and gradient."""
    from ppv_amd.optim import AdamW
    norm, attend = _public()
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen).cuda()
    x, w, b, q, k, v = r(5, 64), r(64), r(64), r(1, 5, 2, 16), r(1, 7, 2, 16), r(1, 7, 2, 16)
    neg = lambda t: torch._neg_view(t)
    assert neg(x).is_neg() and neg(x).data_ptr() == x.data_ptr()
    col = torch.complex(r(6, 1), r(6, 1))                       # (one column: every stride fits)
    for got, want in ((norm(neg(x), neg(w), neg(b)), norm(-x, -w, -b)), (norm(neg(x.view(1, 5, 64))), norm(-x.view(1, 5, 64))),
                      (attend(neg(q), neg(k), neg(v)), attend(-q, -k, -v)), (norm(x, None, neg(b)), norm(x, None, -b)),
                      (norm(col.conj().imag, None, b[:1]), norm((-col.imag).clone(), None, b[:1]))):
        assert torch.equal(got, want)
    for run in (lambda f: torch.autograd.grad(norm(f(xl), wl), (xl, wl), f(x)), lambda f: torch.autograd.grad(attend(ql, k, v), ql, f(q)),
                lambda f: torch.autograd.grad(attend(f(ql), k, v), ql, q)):
        xl, wl, ql = x.clone().requires_grad_(True), w.clone().requires_grad_(True), q.clone().requires_grad_(True)
        assert all(torch.equal(a, c) for a, c in zip(run(neg), run(lambda t: -t)))
    zero = torch._efficientzerotensor((5, 64), device="cuda")
    xl = x.clone().requires_grad_(True)
    assert torch.equal(norm(zero, w, b), b.expand(5, 64)) and torch.equal(torch.autograd.grad(norm(xl), xl, zero)[0], torch.zeros_like(x))
    p = torch.nn.Parameter(r(64))
    p.grad = neg(b)
    with pytest.raises(NotImplementedError):
        AdamW([p]).step()


def test_a_library_of_another_build_is_refused():
    import types
    from ppv_amd import _lib
    mod = _lib.torch_ops()
    names = ("abi_version", "attention_bytes", "torch_version")
    _lib._check_torch_ops(mod)
    for name, other in zip(names, (mod.abi_version - 1, mod.attention_bytes + 8, "1.0.0")):
        with pytest.raises(RuntimeError, match="stale build"):
            _lib._check_torch_ops(types.SimpleNamespace(**{**{n: getattr(mod, n) for n in names}, name: other}))
    with pytest.raises(RuntimeError, match="stale build"):
        _lib._check_torch_ops(types.SimpleNamespace())          # from before it said what it was made for


@pytest.mark.parametrize("version", ["", "a0+git1234567", ".dev20260101+rocm7.0", "+rocm7.0"])
def test_builds_of_one_torch_release_are_one(version, monkeypatch):
    from ppv_amd import _lib
    mod = _lib.torch_ops()
    monkeypatch.setattr(torch, "__version__", mod.torch_version + version)
    _lib._check_torch_ops(mod)
    monkeypatch.setattr(torch, "__version__", mod.torch_version + "7" + version)
    with pytest.raises(RuntimeError, match="stale build"):
        _lib._check_torch_ops(mod)


def _train_step(norm, attend, x, w, q, k, v, lens):
    leaves = [t.clone().requires_grad_(True) for t in (x, w, q, k, v)]
    y = norm(leaves[0], leaves[1])
    o = attend(*leaves[2:], causal=True, q_lens=lens, k_lens=lens)
    return (y.detach(), o.detach()) + torch.autograd.grad((y, o), leaves, (torch.cos(y.detach()), torch.cos(o.detach())))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_saved_tensors_may_go_away_and_come_back(dt):
    """Through host memory, in another order of memory, at another alignment: the same bits.  What comes back on another device, in another size or type is an
    error, never an address for a kernel."""
    norm, attend = _public()
    gen = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=gen).cuda().to(dt)
    args = (r(7, 40), r(40), r(3, 9, 4, 20), r(3, 11, 2, 20), r(3, 11, 2, 20), torch.tensor([9, 4, 0], dtype=torch.int32, device="cuda"))
    want = _train_step(norm, attend, *args)

    def backwards(t):                                           # the same values, memory in the reversed order of axes
        return t.permute(*reversed(range(t.dim()))).contiguous().permute(*reversed(range(t.dim())))

    def off(t):                                                 # one element behind a multiple of 16 bytes
        f = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape)
        return f.copy_(t)

    hooks = torch.autograd.graph.saved_tensors_hooks
    for ctx in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.save_on_cpu(pin_memory=True), hooks(backwards, lambda t: t), hooks(off, lambda t: t)):
        with ctx:
            got = _train_step(norm, attend, *args)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    for wrong in (lambda t: t.cpu(), lambda t: t.double() if t.is_floating_point() else t.long(), lambda t: t[:-1], lambda t: t[None]):
        for call, leaf in ((lambda a: norm(a, args[1]), args[0]), (lambda a: attend(a, args[3], args[4], q_lens=args[5]), args[2])):
            a = leaf.clone().requires_grad_(True)
            with hooks(wrong, lambda t: t):
                y = call(a)
            with pytest.raises(RuntimeError, match="came back from its hooks"):
                y.sum().backward()
