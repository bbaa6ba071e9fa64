"""ppv_amd.nn_ops.layer_norm (csrc/layernorm.hip) against the formula in 64 bits: value, gradients to x, weight and bias, strides, odd
and long rows, refusals."""
import pytest
import torch

from oracle import transformer as orc

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24


def _half_step(dt):
    return torch.finfo(dt).eps / 2


def _case(rows, cols, dt, wdt, seed, offset=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, cols, generator=g) * 1.5 + offset * torch.randn(rows, 1, generator=g)).to(dt)
    w = (1 + 0.1 * torch.randn(cols, generator=g)).to(wdt)
    b = (0.1 * torch.randn(cols, generator=g)).to(wdt)
    dy = torch.randn(rows, cols, generator=g).to(dt)
    return x, w, b, dy


def _check(x, w, b, dy, y, dx, dw, db, eps):
    """Bounds by counting roundings: a sum over a row is at most 32 additions in a lane and 16 across lanes (rows that are longer than the
    registers: C / 256 in a lane), a row's mean is off by at most K u max|x| with K = 48 + C / 256, and so is x - mean; h = (x - mean) rstd
    is off by E = K u max|x| rstd plus 3 u |h|, and rstd's own error is of the same order.  Each result is rounded once to its type."""
    rows, C = x.shape
    dt, wdt = y.dtype, (w.dtype if w is not None else torch.float32)
    xd, dyd = x.double().requires_grad_(True), dy.double()
    wd = (torch.ones(C) if w is None else w).double().requires_grad_(True)
    bd = (torch.zeros(C) if b is None else b).double().requires_grad_(True)
    ref = orc.layer_norm(xd, wd, bd, eps)
    gx, gw, gb = torch.autograd.grad(ref, (xd, wd, bd), dyd)
    xd, ref, wd = xd.detach(), ref.detach(), wd.detach()
    K = 48 + C / 256
    rstd = 1 / torch.sqrt(xd.var(1, unbiased=False, keepdim=True) + eps)
    h = (xd - xd.mean(1, keepdim=True)) * rstd
    E = K * U * (xd.abs().amax(1, keepdim=True) * rstd + h.abs()) + K * U * h.abs().amax(1, keepdim=True)
    tol_y = _half_step(dt) * ref.abs() + wd.abs() * 2 * E + 4 * U * (ref.abs() + bd.detach().abs())
    assert ((y.cpu().double() - ref).abs() <= tol_y * 1.0001 + 1e-30).all()
    if dx is None:
        return
    G = (dyd * wd).abs().amax(1, keepdim=True)
    H = h.abs().amax(1, keepdim=True)
    tol_dx = _half_step(dt) * gx.abs() + rstd * G * (1 + H) * (1 + H) * 2 * (3 * K * U + 2 * E)
    assert ((dx.cpu().double() - gx).abs() <= tol_dx * 1.0001 + 1e-30).all()
    chain = rows / 64 + 128                       # additions one after another in a column's sum
    for got, ref_, terms in ((dw, gw, (dyd * h).abs().sum(0)), (db, gb, dyd.abs().sum(0))):
        if got is not None:
            tol = _half_step(wdt) * ref_.abs() + chain * U * terms + (dyd.abs() * 2 * E).sum(0)
            assert ((got.cpu().double() - ref_).abs() <= tol * 1.0001 + 1e-30).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt,wdt", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f16", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (5, 7), (17, 64), (9, 65), (33, 127), (6, 512), (300, 513), (7, 1367), (5, 2048), (3, 2049),
                                       (4, 4100), (3, 8192), (2, 8201), (2, 16384), (3, 16391), (1, 40000), (4099, 24), (2500, 520)])
def test_layer_norm_value_and_gradients(rows, cols, dt, wdt):
    from ppv_amd.nn_ops import layer_norm
    x, w, b, dy = _case(rows, cols, DT[dt], DT[wdt], rows * 7 + cols)
    xg, wg, bg = (t.cuda().requires_grad_(True) for t in (x, w, b))
    y = layer_norm(xg, wg, bg, eps=1e-5)
    dx, dw, db = torch.autograd.grad(y, (xg, wg, bg), dy.cuda())
    assert y.dtype == x.dtype and dx.dtype == x.dtype and dw.dtype == w.dtype and db.dtype == b.dtype
    _check(x, w, b, dy, y.detach(), dx, dw, db, 1e-5)
    with torch.no_grad():
        assert torch.equal(layer_norm(xg, wg, bg, eps=1e-5), y)                     # the form without statistics: the same numbers
    y2 = layer_norm(xg, wg, bg, eps=1e-5)
    again = torch.autograd.grad(y2, (xg, wg, bg), dy.cuda())
    assert all(torch.equal(a, c) for a, c in zip(again, (dx, dw, db)))              # and the same bits every time


@pytest.mark.gpu
@pytest.mark.parametrize("has_w,has_b", [(False, False), (True, False), (False, True)])
def test_layer_norm_without_parameters(has_w, has_b):
    from ppv_amd.nn_ops import layer_norm
    x, w, b, dy = _case(40, 260, torch.float32, torch.float32, 3)
    xg = x.cuda().requires_grad_(True)
    wg = w.cuda().requires_grad_(True) if has_w else None
    bg = b.cuda().requires_grad_(True) if has_b else None
    y = layer_norm(xg, wg, bg)
    y.backward(dy.cuda())
    _check(x, w if has_w else None, b if has_b else None, dy, y.detach(), xg.grad, wg.grad if has_w else None, bg.grad if has_b else None, 1e-5)


@pytest.mark.gpu
def test_layer_norm_strides_and_shapes():
    """Rows inside a wider buffer (a row stride that is no multiple of 16 bytes), a start off any 16-byte boundary, transposed and expanded
    inputs, leading dimensions, an expanded gradient, an empty batch."""
    from ppv_amd.nn_ops import layer_norm
    g = torch.Generator().manual_seed(5)
    for dt in DT.values():
        wide = torch.randn(21, 331, generator=g).to(dt)
        w, b = torch.randn(200, generator=g), torch.randn(200, generator=g)
        for view in (lambda t: t[:, 3:203], lambda t: t[::2, 131:331], lambda t: t[:, :200].unsqueeze(1).expand(21, 2, 200),
                     lambda t: t[:20, :200].t().contiguous().t(), lambda t: t[:1, :200]):
            x = view(wide)
            xg = view(wide.cuda()).requires_grad_(True)
            y = layer_norm(xg, w.cuda(), b.cuda())
            dy = torch.ones((), dtype=dt).expand(x.shape)                          # a gradient without a stride
            dx, = torch.autograd.grad(y, xg, dy.cuda().expand(x.shape))
            assert y.shape == x.shape and dx.shape == x.shape
            _check(x.reshape(-1, 200), w, b, dy.reshape(-1, 200), y.detach().reshape(-1, 200), dx.reshape(-1, 200), None, None, 1e-5)
    e = torch.zeros(0, 16, device="cuda", requires_grad=True)
    we = torch.ones(16, device="cuda", requires_grad=True)
    y = layer_norm(e, we, None)
    y.sum().backward()
    assert y.shape == (0, 16) and torch.equal(we.grad, torch.zeros(16, device="cuda"))
    one = torch.randn(16, device="cuda")
    assert layer_norm(one).shape == (16,)


@pytest.mark.gpu
def test_layer_norm_keeps_rows_apart_and_what_lies_around_them():
    """A NaN or infinite row poisons itself alone (its share of the weight gradient aside); rows far from zero keep their variance; nothing is
    written outside the result."""
    from ppv_amd.nn_ops import layer_norm
    x, w, b, _ = _case(70, 513, torch.float32, torch.float32, 9)
    x[3, 100] = float("nan")
    x[64, 0] = float("inf")
    x[10] = 30000.0 + 0.01 * torch.arange(513)                  # (the spacing of f32 there is 0.002)
    y = layer_norm(x.cuda(), w.cuda(), b.cuda()).cpu()
    bad = torch.zeros(70, dtype=torch.bool)
    bad[[3, 64]] = True
    assert torch.isnan(y[bad]).any(1).all() and torch.isfinite(y[~bad]).all()
    ok = ~bad
    _check(x[ok], w, b, torch.zeros_like(x[ok]), y[ok], None, None, None, 1e-5)


@pytest.mark.gpu
def test_layer_norm_gradient_against_differences():
    from ppv_amd.nn_ops import layer_norm
    x, w, b, dy = _case(6, 37, torch.float32, torch.float32, 21)
    xg = x.cuda().requires_grad_(True)
    dx, = torch.autograd.grad(layer_norm(xg, w.cuda(), b.cuda()), xg, dy.cuda())
    d = torch.randn(x.shape, generator=torch.Generator().manual_seed(1)).double()
    h = 1e-5
    f = lambda t: (orc.layer_norm(t, w.double(), b.double()) * dy.double()).sum()
    slope = (f(x.double() + h * d) - f(x.double() - h * d)) / (2 * h)
    assert abs((dx.cpu().double() * d).sum() - slope) <= 1e-5 * (dx.cpu().double() * d).abs().sum()


@pytest.mark.gpu
def test_layer_norm_on_another_stream_and_in_a_graph():
    from ppv_amd.nn_ops import layer_norm
    x, w, b, dy = (t.cuda() for t in _case(130, 512, torch.bfloat16, torch.float32, 2))
    want = layer_norm(x, w, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    xs = x.clone().requires_grad_(True)
    ws = w.clone().requires_grad_(True)
    with torch.cuda.stream(side):
        for _ in range(3):
            torch.autograd.grad(layer_norm(xs, ws, b), (xs, ws), dy)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer_norm(xs, ws, b)
        dx, dw = torch.autograd.grad(y, (xs, ws), dy)
    for k in range(3):
        with torch.no_grad():
            xs.copy_(x * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        xe, we = xs.detach().clone().requires_grad_(True), ws.detach().clone().requires_grad_(True)
        ye = layer_norm(xe, we, b)
        de = torch.autograd.grad(ye, (xe, we), dy)
        assert torch.equal(y, ye) and torch.equal(dx, de[0]) and torch.equal(dw, de[1])
        if k == 0:
            assert torch.equal(y, want)


def test_layer_norm_refusals():
    """Raised before anything is launched: no GPU is needed."""
    from ppv_amd.nn_ops import layer_norm
    x = torch.zeros(3, 8)
    with pytest.raises(RuntimeError):
        layer_norm(x)                                           # no CPU path
    with pytest.raises(TypeError):
        layer_norm(x.double())
    with pytest.raises(ValueError):
        layer_norm(torch.zeros(3, 0))
    with pytest.raises(ValueError):
        layer_norm(torch.zeros(()))
    with pytest.raises(ValueError):
        layer_norm(x, torch.ones(7))
    with pytest.raises(ValueError):
        layer_norm(x, None, torch.ones(1, 8))
    with pytest.raises(TypeError):
        layer_norm(x, torch.ones(8), torch.ones(8).bfloat16())
    with pytest.raises(TypeError):
        layer_norm(x, torch.ones(8, dtype=torch.float64))
    with pytest.raises(ValueError):
        layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError):
        layer_norm(x, eps=float("nan"))


def test_layer_norm_entry_points_refuse():
    import ctypes
    from ppv_amd import _lib
    L = _lib.lib()
    p = ctypes.c_void_p(64)
    NULL, SIZE = _lib.PPV_ERR_NULL, _lib.PPV_ERR_BAD_SIZE
    assert L.ppv_layernorm_fwd(None, 8, p, p, p, p, p, 1, 8, 0, 0, 1e-5, None) == NULL
    assert L.ppv_layernorm_fwd(p, 8, p, p, None, p, p, 1, 8, 0, 0, 1e-5, None) == NULL
    assert L.ppv_layernorm_fwd(p, 8, p, p, p, p, None, 1, 8, 0, 0, 1e-5, None) == NULL
    assert L.ppv_layernorm_fwd(p, 8, p, p, p, p, p, 0, 8, 0, 0, 1e-5, None) == SIZE
    assert L.ppv_layernorm_fwd(p, 8, p, p, p, p, p, 1, 0, 0, 0, 1e-5, None) == SIZE
    assert L.ppv_layernorm_fwd(p, 8, p, p, p, p, p, 1, 8, 3, 0, 1e-5, None) == SIZE
    assert L.ppv_layernorm_fwd(p, 8, p, p, p, p, p, 1, 8, 0, -1, 1e-5, None) == SIZE
    assert L.ppv_layernorm_bwd(p, 8, p, 8, p, p, p, p, p, p, None, 1, 8, 0, 0, None) == NULL
    assert L.ppv_layernorm_bwd(p, 8, p, 8, p, None, p, p, p, p, p, 1, 8, 0, 0, None) == NULL
    assert L.ppv_layernorm_bwd(p, 8, p, 8, p, p, p, p, p, p, p, 1, 8, 0, 5, None) == SIZE
    assert L.ppv_layernorm_bwd_workspace_bytes(0, 8, 0) == 0
    assert L.ppv_layernorm_bwd_workspace_bytes(10, 8, 0) >= 2 * 8 * 4


@pytest.mark.gpu
def test_layer_norm_is_differentiable_once():
    """A graph of the backward pass can be asked for; differentiating through it is an error, not a silent zero."""
    from ppv_amd.nn_ops import layer_norm
    x, w, b, dy = (t.cuda() for t in _case(6, 40, torch.float32, torch.float32, 4))
    x.requires_grad_(True)
    want, = torch.autograd.grad(layer_norm(x, w, b), x, dy)
    dx, = torch.autograd.grad(layer_norm(x, w, b), x, dy, create_graph=True)
    assert torch.equal(dx, want)
    with pytest.raises(RuntimeError, match="differentiable once"):
        dx.sum().backward()


@pytest.mark.gpu
def test_captured_backward_over_a_living_eager_graph_is_refused():
    """The engine would hand the gradient to the default stream, where the leaf's accumulation lives, in the middle of the capture: an error that says so
    comes first, the capture stays whole and so does the eager graph.  Once the eager graph is gone, or where its leaf is not asked for, capturing works."""
    from ppv_amd.attention import multihead_attention
    from ppv_amd.nn_ops import layer_norm
    torch.manual_seed(5)
    x = torch.randn(6, 64, device="cuda", requires_grad=True)
    w = torch.randn(64, device="cuda", requires_grad=True)
    g = torch.randn(6, 64, device="cuda")
    want = torch.autograd.grad(layer_norm(x, w), (x, w), g)
    eager = layer_norm(x.view(6, 64), w) * 1.0
    for run, what in ((lambda: torch.autograd.grad(layer_norm(x.view(6, 64), None), x, g), "layer norm"),
                      (lambda: torch.autograd.grad(multihead_attention(*(x.view(1, 6, 1, 64),) * 3), x, g.view(1, 6, 1, 64)), "attention")):
        graph, refused = torch.cuda.CUDAGraph(), ""
        with torch.cuda.graph(graph):
            scratch = torch.empty(4, device="cuda").zero_()     # (a capture that holds something)
            try:
                run()
            except RuntimeError as e:
                refused = str(e)
        assert "eager graph" in refused and scratch.numel() == 4, what
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(eager, (x, w), g), want))
    eager = layer_norm(g, w)                                    # of w alone: x's graph is gone, w's is not asked for
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dx, = torch.autograd.grad(layer_norm(x, w), x, g)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dx, want[0]) and eager.requires_grad


@pytest.mark.gpu
def test_layer_norm_of_rows_whose_offsets_pass_32_bits():
    from ppv_amd.nn_ops import layer_norm
    rows, C, step = 4200, 200, 1 << 20                          # offsets up to 4.4e9 elements
    x, w, b, dy = (t.cuda() for t in _case(rows, C, torch.bfloat16, torch.float32, 3))
    far = torch.empty(rows * step, dtype=torch.bfloat16, device="cuda").view(rows, step)[:, 5:5 + C]
    far.copy_(x)
    runs = []
    for t in (far, x):
        leaf = t.detach().requires_grad_(True)
        y = layer_norm(leaf, w, b)
        runs.append((y,) + torch.autograd.grad(y, leaf, dy))
    assert all(torch.equal(p, q) for p, q in zip(*runs))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,C", [(2, 1 << 27), (70000, 8193)])
def test_layer_norm_of_more_columns_or_long_rows_than_a_launch_has_along_one_axis(rows, C):
    """Weight gradients of 2^27 columns (2^28 sums, 16 to a workgroup of 256: 2^32 work items) and 70000 rows that are read in passes.  Rows of +-1 with gradients
    of small whole numbers: every sum is exact.  The mean is 0 (or 1 / C), h = +-rstd within 2 / C: u / 4 and 3 roundings; a gradient of w adds its
    rows' products one by one (70000 rows in 64 shares: 1100 additions of at most 2, and 16)."""
    from ppv_amd.nn_ops import layer_norm
    i = torch.arange(C, device="cuda")
    x = (1.0 - 2.0 * (i % 2)).expand(rows, C).contiguous().requires_grad_(True)
    dy = ((i * 7) % 5 - 2).float()
    w, b = torch.ones(C, device="cuda", requires_grad=True), torch.zeros(C, device="cuda", requires_grad=True)
    y = layer_norm(x, w, b, eps=0.0)
    off = 0.0 if C % 2 == 0 else 4.0 / C
    assert ((y.detach() - x.detach()).abs().amax()) <= off + 8 * U
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy.expand(rows, C))
    assert torch.equal(db, dy * rows)
    assert ((dw - dy * x.detach()[0] * rows).abs() <= rows * 2 * (off + 8 * U) + (0 if rows == 2 else 1116 * U * 2 * rows)).all()
    s1, s2 = dy.double().mean(), (dy * x.detach()[0]).double().mean()
    want = dy.double() - s1 - x.detach()[0].double() * s2
    for r in (0, rows // 2, rows - 1):
        assert ((dx[r].double() - want).abs() <= 16 * off + 64 * U).all()


def test_layer_norm_entry_points_refuse_more_long_rows_than_they_count():
    import ctypes
    from ppv_amd import _lib
    L, p = _lib.lib(), ctypes.c_void_p(64)
    assert L.ppv_layernorm_fwd(p, 9000, p, p, p, p, p, 1 << 31, 9000, 0, 0, 1e-5, None) == _lib.PPV_ERR_BAD_SIZE
    assert L.ppv_layernorm_bwd(p, 9000, p, 9000, p, p, p, p, p, p, p, 1 << 31, 9000, 0, 0, None) == _lib.PPV_ERR_BAD_SIZE
