"""Linear cross entropy (vrs_linear_cross_entropy_*, vector_cuda.ops): loss and
gradients against the formulas in 64 bits, differences, refusals.

Tolerances. Products of 16-bit operands are exact in 32 bits; a score's sum of
d of them is off by at most (d + 2) 2^-22 sum|x_i w_i| scale (4 ulps a term, so
that a truncating accumulator is allowed). e_z, the largest of these in a row,
bounds the error of lse up to the 32-bit exponentials and sums: 2^-20 relative
in the sum, 2^-22 of |lse|. A probability is then off by the factor
2 e_z + 2^-20. The gradient of a score is an operand of the tensor cores in 16
bits: half an ulp (h = 2^-11 or 2^-8) of |g|, in f16 also 2^-38 of the largest
(its scaled range ends there). With d_g = h + 2^-20 + 2 e_z, taken
for both the probability and the whole gradient:
  |dx - exact| <= d_g |g| |table| + (classes + 2) 2^-22 |g| |table|, and likewise
  dtable over rows, each plus half an ulp of the result."""
import ctypes

import pytest

HALF = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def _make(rows, classes, d, dtype, ignored=0.0, spread=1.5, seed=0, unit=False):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 7 + classes * 3 + d)
    t = torch.randint(0, classes, (rows,), generator=g, device="cuda")
    w = torch.randn(classes, d, generator=g, device="cuda") * (spread / d ** 0.5)
    x = torch.randn(rows, d, generator=g, device="cuda") + w[t]
    if unit:
        w /= w.norm(dim=1, keepdim=True)
        x /= x.norm(dim=1, keepdim=True)
    if ignored:
        t = torch.where(torch.rand(rows, generator=g, device="cuda") < ignored, -1 - t, t)
    dl = torch.rand(rows, generator=g, device="cuda") + 0.25
    dt = getattr(torch, dtype)
    return x.to(dt), w.to(dt), t, dl


def _check(x, w, t, dl, scale=1.0, dtype=None):
    import torch
    from vector_cuda import ops
    h = HALF[str(x.dtype).replace("torch.", "")]
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    classes, d = w.shape
    taken = (t >= 0) & (t < classes)
    X, W = torch.where(taken[:, None], x.double(), 0.0), w.double()
    z = scale * (X @ W.t())
    ez = (d + 2) * 2.0 ** -22 * scale * (X.abs() @ W.abs().t()).amax(1)
    lse64 = torch.logsumexp(z, 1)
    zt = z.gather(1, t.clamp(0, classes - 1)[:, None])[:, 0]
    loss, lse = ops.linear_cross_entropy_forward(x, w, t, scale)
    assert loss.dtype == lse.dtype == torch.float32 and loss.shape == t.shape
    assert not loss[~taken].any() and not lse[~taken].any()
    tol = ez + 2.0 ** -20 + 2.0 ** -22 * lse64.abs()
    assert ((lse.double() - lse64).abs() <= tol)[taken].all()
    assert ((loss.double() - (lse64 - zt)).abs() <= tol + ez + 2.0 ** -22 * zt.abs())[taken].all()
    p = torch.exp(z - lse64[:, None])
    hot = torch.zeros_like(p).scatter_(1, t.clamp(0, classes - 1)[:, None], 1.0)
    up = torch.where(taken, dl.double() * scale, 0.0)[:, None]
    g = (p - hot) * up
    ga = (p + hot) * up.abs()  # |g|, and what its error is relative to
    rel = 2.0 ** -20 + 2 * ez[:, None]
    ge = h * 1.01 * g.abs() + rel * ga + (2.0 ** -38 * up.abs().max() if tiny else 0.0) * taken[:, None]
    dx, dw = ops.linear_cross_entropy_backward(dl, x, w, t, lse, scale)
    assert dx.shape == x.shape and dw.shape == w.shape and dx.dtype == dw.dtype == x.dtype
    for got, want, e, a in ((dx, g @ W, ge @ W.abs() + (classes + 2) * 2.0 ** -22 * (ga @ W.abs()), "dx"),
                            (dw, g.t() @ X, ge.t() @ X.abs() + (len(t) + 2) * 2.0 ** -22 * (ga.t() @ X.abs()), "dtable")):
        off = (got.double() - want).abs()
        lim = e + 1.01 * h * want.abs() + tiny
        assert (off <= lim).all(), f"{a}: {int((off > lim).sum())} of {off.numel()} off, worst {(off / lim).max().item():.3g}x"
    assert not dx[~taken].any()
    return loss, lse, dx, dw


# Rows: one, both sides of the 128- and 256-row tiles. Classes: one, both sides
# of the 256-class tiles, primes. Widths: one, odd, both sides of 64.
SIZES = [(1, 1, 1), (1, 2, 8), (3, 5, 7), (1, 1000, 64), (7, 255, 65), (64, 256, 63), (127, 257, 128), (128, 300, 100),
         (129, 511, 96), (255, 512, 256), (256, 513, 72), (257, 1031, 200), (300, 70, 513), (1000, 31, 40),
         (19, 4099, 500), (2100, 129, 64), (5, 20011, 24), (513, 2500, 501)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,classes,d", SIZES)
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_matches_formula(gpu, rows, classes, d, dtype):
    _check(*_make(rows, classes, d, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("ignored", [0.05, 0.5, 0.97, 1.1])
@pytest.mark.parametrize("rows", [5, 300, 1025])
def test_rows_without_target(gpu, rows, ignored, dtype):
    _check(*_make(rows, 700, 136, dtype, ignored=ignored))


@pytest.mark.gpu
def test_targets_outside_on_both_sides(gpu):
    import torch
    x, w, t, dl = _make(40, 100, 64, "bfloat16")
    t[::4] = 100
    t[1::4] = 2 ** 40
    t[2::8] = -(2 ** 62)
    _check(x, w, t, dl)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_values_of_rows_that_take_no_part(gpu, dtype):
    """Infinities and NaN in rows without a target, in their dloss too, reach nothing."""
    import torch
    from vector_cuda import ops
    x, w, t, dl = _make(150, 333, 72, dtype, ignored=0.4)
    clean = _check(x, w, t, dl)
    off = t < 0
    x[off] = float("nan")
    x[off.nonzero()[0, 0], ::2] = float("inf")
    dl[off] = float("nan")
    loss, lse = ops.linear_cross_entropy_forward(x, w, t)
    got = (loss, lse, *ops.linear_cross_entropy_backward(dl, x, w, t, lse))
    assert all(torch.equal(p, q) for p, q in zip(clean, got))


@pytest.mark.gpu
def test_infinite_and_nan_scores(gpu):
    """A row whose scores are NaN or +inf has a loss that says so; its
    neighbours' losses do not change. A score of -inf has probability 0."""
    import torch
    from vector_cuda import ops
    x, w, t, dl = _make(140, 300, 64, "bfloat16")
    a, _ = ops.linear_cross_entropy_forward(x, w, t)
    x[3, 0] = float("nan")
    x[7] = float("inf")
    b, _ = ops.linear_cross_entropy_forward(x, w, t)
    assert not torch.isfinite(b[3]) and not torch.isfinite(b[7])
    keep = [i for i in range(140) if i not in (3, 7)]
    assert torch.equal(a[keep], b[keep])
    x, w, t, dl = _make(20, 300, 64, "float16")
    x[:, 0] = 1.0
    w[::2, 0] = -float("inf")
    t = t // 2 * 2 + 1 - 2 * (t == 299)  # odd classes keep finite scores
    want = torch.logsumexp(x.double() @ w.double().t(), 1)
    _, lse = ops.linear_cross_entropy_forward(x, w, t)
    assert ((lse - want).abs() < 1e-3).all()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-3, 0.37, 20.0, 100.0])
def test_scale(gpu, scale):
    _check(*_make(200, 900, 128, "bfloat16", unit=True), scale=scale)
    _check(*_make(200, 900, 128, "float16", unit=True), scale=scale)


@pytest.mark.gpu
def test_large_scores(gpu):
    """Scores of some thousands: the running maximum has to carry them."""
    _check(*_make(64, 2000, 64, "bfloat16", spread=600.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** 10])
def test_gradients_of_any_size(gpu, size, dtype):
    """dloss far from 1 (with 16-bit floats 2^-20 is below their normal range)."""
    x, w, t, dl = _make(130, 500, 64, dtype)
    _check(x, w, t, dl * size)


@pytest.mark.gpu
def test_rows_of_very_different_weight(gpu):
    x, w, t, dl = _make(130, 500, 64, "float16")
    dl[::2] *= 2.0 ** -12
    dl[5] = 0.0
    dl[7] *= -1.0
    _check(x, w, t, dl)


@pytest.mark.gpu
@pytest.mark.parametrize("xs,xo,ws,wo", [(136, 0, 128, 0), (131, 1, 128, 0), (128, 0, 136, 0), (128, 0, 133, 0),
                                         (128, 0, 136, 4), (200, 3, 129, 5)])
def test_strided_rows(gpu, xs, xo, ws, wo):
    """Rows and tables inside wider buffers, on and off 16-byte boundaries."""
    import torch
    x, w, t, dl = _make(70, 310, 128, "bfloat16")

    def inside(m, stride, offset):
        b = torch.full((m.shape[0] * stride + offset,), float("nan"), dtype=m.dtype, device="cuda")
        v = b[offset:].view(m.shape[0], stride)[:, :m.shape[1]]
        v.copy_(m)
        return v

    _check(inside(x, xs, xo), inside(w, ws, wo), t, dl)


@pytest.mark.gpu
def test_gradients_into_wider_buffers(gpu, vc):
    """C entry: dx and dtable with strides and offsets of their own; what lies
    between their rows is left alone. Either alone gives the same bits."""
    import torch
    from vector_cuda import ops
    x, w, t, dl = _make(70, 310, 104, "float16", ignored=0.2)
    _, lse = ops.linear_cross_entropy_forward(x, w, t)
    dx, dw = ops.linear_cross_entropy_backward(dl, x, w, t, lse)
    a, none = ops.linear_cross_entropy_backward(dl, x, w, t, lse, need_dtable=False)
    assert none is None and torch.equal(a, dx)
    none, b = ops.linear_cross_entropy_backward(dl, x, w, t, lse, need_dx=False)
    assert none is None and torch.equal(b, dw)
    L, n = vc.lib(), ctypes.c_int64(0)
    for stride, offset in ((112, 8), (107, 3)):
        bx = torch.full((70 * stride + offset,), 7.0, dtype=x.dtype, device="cuda")
        bw = torch.full((310 * stride + offset,), 7.0, dtype=x.dtype, device="cuda")
        assert L.vrs_linear_cross_entropy_workspace(70, 310, 104, 1, 1, int(stride % 8 == 0), ctypes.byref(n)) == 0
        ws = torch.empty(n.value, dtype=torch.uint8, device="cuda")
        st = L.vrs_linear_cross_entropy_backward(dl.data_ptr(), x.data_ptr(), 104, 70, w.data_ptr(), 104, 310, 104, 1,
                                                 t.data_ptr(), 1.0, lse.data_ptr(), bx.data_ptr() + 2 * offset, stride,
                                                 bw.data_ptr() + 2 * offset, stride, ws.data_ptr(), n.value, None)
        assert st == 0, L.vrs_last_error()
        torch.cuda.synchronize()
        for buf, want, rows in ((bx, dx, 70), (bw, dw, 310)):
            v = buf[offset:].view(rows, stride)
            assert torch.equal(v[:, :104], want) and (v[:, 104:] == 7.0).all() and (buf[:offset] == 7.0).all()


@pytest.mark.gpu
def test_many_pieces(gpu):
    """Classes enough for several pieces of the backward pass."""
    import torch
    from vector_cuda import ops
    x, w, t, dl = _make(1100, 300000, 16, "bfloat16", ignored=0.3)
    loss, lse = ops.linear_cross_entropy_forward(x, w, t)
    dx, dw = ops.linear_cross_entropy_backward(dl, x, w, t, lse)
    # a stretch of classes across the middle, and every row's loss, in 64 bits
    taken = t >= 0
    z = x.double() @ w.double().t()
    want = torch.logsumexp(z, 1)
    assert ((lse.double() - want).abs() <= 1e-4)[taken].all()
    g = torch.exp(z - want[:, None])
    g.scatter_add_(1, t.clamp(min=0)[:, None], -torch.ones_like(want)[:, None])
    g *= torch.where(taken, dl.double(), 0.0)[:, None]
    h = HALF["bfloat16"]
    ga = g.abs()
    lim = 1.01 * (h + 1e-4) * (ga @ w.double().abs()) + h * 1.01 * (g @ w.double()).abs() + 1e-12
    assert ((dx.double() - g @ w.double()).abs() <= lim).all()
    want = g.t() @ x.double()
    lim = 1.01 * (h + 1e-4) * (ga.t() @ x.double().abs()) + h * 1.01 * want.abs() + 1e-12
    assert ((dw.double() - want).abs() <= lim).all()


# Tiles enough for several turns of the CTAs (up to 128 rows) and of the pairs,
# with last turns that are full, half full and shorter.
@pytest.mark.gpu
@pytest.mark.parametrize("rows,classes,d", [(64, 38000, 24), (65, 50000, 40), (128, 39000, 72), (129, 20000, 33),
                                            (200, 38100, 64), (256, 19000, 130), (257, 9700, 64), (700, 6500, 320)])
def test_several_turns(gpu, rows, classes, d):
    _check(*_make(rows, classes, d, "bfloat16", ignored=0.1))


# More rows than a block counts by itself (8,192), with pieces of the classes.
@pytest.mark.gpu
@pytest.mark.parametrize("rows,classes,d,ignored", [(8193, 600, 40, 0.0), (9500, 700, 96, 0.5), (20000, 9000, 16, 0.2),
                                                    (12345, 3, 264, 0.9)])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_many_rows(gpu, rows, classes, d, ignored, dtype):
    _check(*_make(rows, classes, d, dtype, ignored=ignored))


@pytest.mark.gpu
@pytest.mark.parametrize("d", [8, 9, 15, 127, 129, 500, 1001])
def test_alignments_of_rows(gpu, d):
    """Every start of a row within 16 bytes: contiguous odd widths, and tables
    that begin off a 16-byte boundary."""
    import torch
    x, w, t, dl = _make(150, 400, d, "float16", ignored=0.2)
    for o in range(0, 8, 3):
        bx = torch.zeros(x.numel() + o, dtype=x.dtype, device="cuda")
        bw = torch.zeros(w.numel() + o, dtype=x.dtype, device="cuda")
        vx, vw = bx[o:].view_as(x), bw[o:].view_as(w)
        vx.copy_(x)
        vw.copy_(w)
        _check(vx, vw, t, dl)


@pytest.mark.gpu
def test_repeatable_and_empty(gpu):
    import torch
    from vector_cuda import ops
    x, w, t, dl = _make(700, 5000, 264, "bfloat16", ignored=0.1)
    loss, lse = ops.linear_cross_entropy_forward(x, w, t)
    first = (loss, lse, *ops.linear_cross_entropy_backward(dl, x, w, t, lse))
    for _ in range(3):
        loss, lse = ops.linear_cross_entropy_forward(x, w, t)
        again = (loss, lse, *ops.linear_cross_entropy_backward(dl, x, w, t, lse))
        assert all(torch.equal(p, q) for p, q in zip(first, again))
    loss, lse = ops.linear_cross_entropy_forward(x[:0], w, t[:0])
    assert loss.shape == (0,)
    dx, dw = ops.linear_cross_entropy_backward(dl[:0], x[:0], w, t[:0], lse)
    assert dx.shape == (0, 264) and dw.shape == w.shape and not dw.any()


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_autograd(gpu, reduction):
    import torch
    from vector_cuda import ops
    x, w, t, _ = _make(90, 400, 80, "float16", ignored=0.3)
    x, w = x.view(9, 10, 80).requires_grad_(True), w.requires_grad_(True)
    t = t.view(9, 10)
    loss = ops.linear_cross_entropy(x, w, t, 2.0, reduction)
    c = torch.linspace(1.0, 2.0, 90, device="cuda").view(9, 10) if reduction == "none" else torch.tensor(1.0, device="cuda")
    (loss * c).sum().backward()
    taken = t >= 0
    z = 2.0 * (x.detach().double() @ w.detach().double().t())
    l64 = torch.where(taken, torch.logsumexp(z, 2) - z.gather(2, t.clamp(min=0)[..., None])[..., 0], 0.0)
    want = {"mean": l64.sum() / taken.sum(), "sum": l64.sum(), "none": l64}[reduction]
    assert ((loss.double() - want).abs() <= 1e-4 * (1 + want.abs())).all()
    up = (c if reduction == "none" else torch.ones(9, 10, device="cuda") / (taken.sum() if reduction == "mean" else 1)).double()
    g = (torch.softmax(z, 2) - torch.nn.functional.one_hot(t.clamp(min=0), 400)) * torch.where(taken, 2.0 * up, 0.0)[..., None]
    for got, exact in ((x.grad, g @ w.detach().double()), (w.grad, torch.einsum("abv,abd->vd", g, x.detach().double()))):
        assert (got.double() - exact).norm() <= 2.0 ** -9 * exact.norm() + 2.0 ** -25 * got.numel() ** 0.5


@pytest.mark.gpu
def test_nothing_takes_part(gpu):
    import torch
    from vector_cuda import ops
    x, w, t, _ = _make(30, 50, 16, "bfloat16")
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    loss = ops.linear_cross_entropy(x, w, torch.full_like(t, -100))
    loss.backward()
    assert loss.item() == 0.0 and not x.grad.any() and not w.grad.any()


@pytest.mark.gpu
def test_gradients_against_differences(gpu):
    """Directional differences of the 32-bit loss: operands move along exact
    16-bit steps, so the difference is of the operator itself. The step's
    second-order term and the loss's rounding (1e-6 over a step of 2^-5)
    stay under 2 % of the gradient's norm along the step."""
    import torch
    from vector_cuda import ops
    x, w, t, dl = _make(6, 40, 16, "float16", spread=1.0)
    lse = ops.linear_cross_entropy_forward(x, w, t)[1]
    dx, dw = ops.linear_cross_entropy_backward(dl, x, w, t, lse)
    g = torch.Generator(device="cuda").manual_seed(3)
    for which, grad in ((0, dx), (1, dw)):
        for _ in range(4):
            v = (torch.randint(0, 2, grad.shape, generator=g, device="cuda") * 2 - 1).to(x.dtype) * 2.0 ** -6
            a, b = [x, w], [x, w]
            a[which], b[which] = a[which] + v, b[which] - v
            fa = (ops.linear_cross_entropy_forward(a[0], a[1], t)[0].double() * dl.double()).sum()
            fb = (ops.linear_cross_entropy_forward(b[0], b[1], t)[0].double() * dl.double()).sum()
            step = (a[which].double() - b[which].double())
            want = (grad.double() * step).sum()
            assert abs((fa - fb - want).item()) <= 0.02 * (grad.double().norm() * step.norm()).item()


@pytest.mark.gpu
def test_on_another_stream(gpu):
    import torch
    from vector_cuda import ops
    x, w, t, dl = _make(600, 9000, 256, "bfloat16")
    loss, lse = ops.linear_cross_entropy_forward(x, w, t)
    want = (loss, *ops.linear_cross_entropy_backward(dl, x, w, t, lse))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        z = torch.zeros_like(x)
        for _ in range(5):
            z.copy_(x)
            loss, lse = ops.linear_cross_entropy_forward(z, w, t)
            got = (loss, *ops.linear_cross_entropy_backward(dl, z, w, t, lse))
            z.zero_()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(want, got))


@pytest.mark.gpu
def test_in_a_graph(gpu):
    """Nothing is allocated or waited for inside a call: it can be captured."""
    import torch
    from vector_cuda import ops
    x, w, t, dl = _make(200, 3000, 128, "bfloat16")
    loss, lse = ops.linear_cross_entropy_forward(x, w, t)
    want = (loss, *ops.linear_cross_entropy_backward(dl, x, w, t, lse))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        l2, e2 = ops.linear_cross_entropy_forward(x, w, t)
        got = (l2, *ops.linear_cross_entropy_backward(dl, x, w, t, e2))
    for o in got:
        o.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))


# ---------------------------------------------------------------- refusals


def _forward(vc, **k):
    a = dict(x=4096, xs=64, rows=4, w=4096, ws=64, v=10, d=64, dt=2, t=4096, scale=1.0, loss=4096, lse=4096, wsp=4096,
             n=1 << 40)
    a.update(k)
    return vc.lib().vrs_linear_cross_entropy_forward(a["x"], a["xs"], a["rows"], a["w"], a["ws"], a["v"], a["d"],
                                                     a["dt"], a["t"], a["scale"], a["loss"], a["lse"], a["wsp"],
                                                     a["n"], None)


@pytest.mark.parametrize("change", [dict(dt=0), dict(dt=3), dict(rows=-1), dict(v=0), dict(d=0), dict(d=65537),
                                    dict(rows=2 ** 31), dict(v=2 ** 31), dict(scale=0.0), dict(scale=-1.0),
                                    dict(scale=float("inf")), dict(scale=float("nan")), dict(x=None), dict(w=None),
                                    dict(t=None), dict(loss=None), dict(lse=None), dict(wsp=None), dict(n=0),
                                    dict(xs=63), dict(ws=63), dict(wsp=4097)])
def test_forward_refuses(vc, change):
    """Refused on the host, before any device work (the pointers are never used)."""
    assert _forward(vc, **change) == 5
    assert b"vrs_linear_cross_entropy_forward" in vc.lib().vrs_last_error()


def _backward(vc, **k):
    a = dict(dl=4096, x=4096, xs=64, rows=4, w=4096, ws=64, v=10, d=64, dt=2, t=4096, scale=1.0, lse=4096, dx=4096,
             dxs=64, dw=4096, dws=64, wsp=4096, n=1 << 40)
    a.update(k)
    return vc.lib().vrs_linear_cross_entropy_backward(a["dl"], a["x"], a["xs"], a["rows"], a["w"], a["ws"], a["v"],
                                                      a["d"], a["dt"], a["t"], a["scale"], a["lse"], a["dx"],
                                                      a["dxs"], a["dw"], a["dws"], a["wsp"], a["n"], None)


@pytest.mark.parametrize("change", [dict(dt=0), dict(rows=-1), dict(v=0), dict(d=0), dict(scale=0.0), dict(dl=None),
                                    dict(x=None), dict(w=None), dict(t=None), dict(lse=None), dict(wsp=None),
                                    dict(n=0), dict(dxs=63), dict(dws=63), dict(xs=1), dict(ws=1), dict(wsp=4097)])
def test_backward_refuses(vc, change):
    assert _backward(vc, **change) == 5
    assert b"vrs_linear_cross_entropy_backward" in vc.lib().vrs_last_error()


def test_workspace_refuses(vc):
    n = ctypes.c_int64(0)
    f = vc.lib().vrs_linear_cross_entropy_workspace
    for bad in ((-1, 10, 64, 2), (4, 0, 64, 2), (4, 10, 0, 2), (4, 10, 64, 0)):
        assert f(*bad, 1, 1, ctypes.byref(n)) == 5
    assert f(4, 10, 64, 2, 1, 1, None) == 5


@pytest.mark.gpu
def test_python_refusals(gpu):
    import torch
    from vector_cuda import ops
    x, w, t, dl = _make(8, 20, 16, "bfloat16")
    for a in ((x.float(), w.float(), t), (x.half(), w, t), (x, w[:, :8], t), (x, w, t[:7]), (x, w, t.int()),
              (x, w[:0], t), (x, w, t.cpu()), (x, w[0], t)):
        with pytest.raises(ValueError):
            ops.linear_cross_entropy_forward(*a)
    for s in (0.0, -2.0, float("nan")):
        with pytest.raises(ValueError):
            ops.linear_cross_entropy_forward(x, w, t, s)
    with pytest.raises(ValueError):
        ops.linear_cross_entropy(x, w, t, 1.0, "median")
    with pytest.raises(ValueError):
        ops.linear_cross_entropy_backward(dl.half(), x, w, t, dl)


# ------------------------------------------------ rows that are predicted well


def _sure(rows, classes, d, dtype, noise, seed=0, offset=0):
    """Unit rows near their targets, as a trained encoder gives them; `offset`
    elements off a 16-byte boundary."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 7 + classes * 3 + d)
    t = torch.randint(0, classes, (rows,), generator=g, device="cuda")
    w = torch.randn(classes, d, generator=g, device="cuda")
    w /= w.norm(dim=1, keepdim=True)
    x = w[t] + torch.randn(rows, d, generator=g, device="cuda") * (noise / d ** 0.5)
    x /= x.norm(dim=1, keepdim=True)

    def placed(m):
        b = torch.zeros(m.numel() + offset, dtype=getattr(torch, dtype), device="cuda")
        return b[offset:].view_as(m).copy_(m)

    return placed(x), placed(w), t


def _sure64(x, w, t, scale):
    """In 64 bits: loss, the score gradients (the target's without a difference)
    and a bound on the relative error of the other classes' weight r = sum of
    e^(z - z[target]) in 32 bits: two scores' errors (as at the head of this file),
    the rounding of the target's score and of both exponents (2^-22 of the score
    each), and the exponentials and sums."""
    import torch
    X, W = x.double(), w.double()
    at = t[:, None]
    z = scale * (X @ W.t())
    zt = z.gather(1, at)
    q = torch.exp(z - zt).scatter_(1, at, 0.0)
    r = q.sum(1, keepdim=True)
    g = (q / (1 + r)).scatter_(1, at, -r / (1 + r))
    ez = (x.shape[1] + 2) * 2.0 ** -22 * scale * (X.abs() @ W.abs().t()).amax(1)
    rel = 2 * ez + 3 * 2.0 ** -22 * zt[:, 0].abs() + 2.0 ** -20
    return torch.log1p(r)[:, 0], g, rel


SURE = [(90, 1000, 64, 0.5, 20.0, 0), (90, 1000, 65, 0.5, 20.0, 0), (300, 700, 33, 0.2, 20.0, 3), (64, 1000, 64, 0.3, 100.0, 0),
        (40, 300, 71, 0.7, 100.0, 1), (300, 20, 512, 1.0, 20.0, 0), (5, 2, 16, 0.1, 20.0, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,classes,d,noise,scale,offset", SURE)
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_small_losses_keep_their_digits(gpu, rows, classes, d, noise, scale, offset, dtype):
    """The loss of a row whose target clearly wins, relative to itself:
    log(1 + r) errs by at most r's relative error and a rounding (2^-22 with
    the logarithm's); below 2^-120 32 bits hold no more digits."""
    from vector_cuda import ops
    x, w, t = _sure(rows, classes, d, dtype, noise, offset=offset)
    want, _, rel = _sure64(x, w, t, scale)
    assert want.median() < 0.02  # (what the case is for)
    loss, lse = ops.linear_cross_entropy_forward(x, w, t, scale)
    off = (loss.double() - want).abs()
    assert (off <= (rel + 2.0 ** -22) * want + 2.0 ** -120).all(), f"worst {(off / want).max().item():.3g} of the loss"


def _sure_gradients(x, w, t, dl, scale, dx, dw):
    """dx and dtable of sure rows against 64 bits, relative to what they are made
    of: score gradients in 16 bits (half an ulp; in f16 2^-38 of the largest
    dloss at least, where their range ends) with r's relative error, against the
    other operand, the sums' own error, and the result's half ulp."""
    import torch
    h = HALF[str(x.dtype).replace("torch.", "")]
    f16 = x.dtype == torch.float16
    X, W = x.double(), w.double()
    _, g, rel = _sure64(x, w, t, scale)
    up = dl.double()[:, None] * scale
    g = g * up
    ge = (1.01 * h + 2 * rel[:, None]) * g.abs() + (2.0 ** -38 * up.abs().max() if f16 else 0.0)
    for got, want, e, what in ((dx, g @ W, ge @ W.abs() + (len(w) + 2) * 2.0 ** -22 * (g.abs() @ W.abs()), "dx"),
                               (dw, g.t() @ X, ge.t() @ X.abs() + (len(t) + 2) * 2.0 ** -22 * (g.abs().t() @ X.abs()), "dtable")):
        lim = e + 1.01 * h * want.abs() + (2.0 ** -25 if f16 else 0.0) + 2.0 ** -120
        off = (got.double() - want).abs()
        assert (off <= lim).all(), f"{what}: {int((off > lim).sum())} of {off.numel()} off, worst {(off / lim).max().item():.3g}x"


@pytest.mark.gpu
@pytest.mark.parametrize("rows,classes,d,noise,scale,offset", SURE)
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_gradients_of_small_losses(gpu, rows, classes, d, noise, scale, offset, dtype):
    """Through autograd. (f16 with a loss scale, as its training has.)"""
    import torch
    from vector_cuda import ops
    x, w, t = _sure(rows, classes, d, dtype, noise, offset=offset)
    dl = torch.full((rows,), 1024.0 if dtype == "float16" else 1.0, device="cuda")
    leaves = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    (ops.linear_cross_entropy(*leaves, t, scale, "none") * dl).sum().backward()
    _sure_gradients(x, w, t, dl, scale, leaves[0].grad, leaves[1].grad)


@pytest.mark.gpu
def test_backward_takes_the_loss(gpu):
    """The pass by itself, given the loss, is autograd's; without it the target's
    gradient comes from lse - z, off by no more than half of lse's last place
    (2^-24 of it) and what sure rows lose otherwise."""
    import torch
    from vector_cuda import ops
    x, w, t = _sure(200, 900, 65, "bfloat16", 0.5)
    dl = torch.ones(200, device="cuda")
    leaves = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    ops.linear_cross_entropy(*leaves, t, 20.0, "sum").backward()
    loss, lse = ops.linear_cross_entropy_forward(x, w, t, 20.0)
    dx, dw = ops.linear_cross_entropy_backward(dl, x, w, t, lse, 20.0, loss=loss)
    assert torch.equal(dx, leaves[0].grad) and torch.equal(dw, leaves[1].grad)
    dx, _ = ops.linear_cross_entropy_backward(dl, x, w, t, lse, 20.0, need_dtable=False)
    h = HALF["bfloat16"]
    _, g, rel = _sure64(x, w, t, 20.0)
    ge = (1.01 * h + 2 * rel[:, None]) * g.abs()
    ge.scatter_add_(1, t[:, None], 2.0 ** -24 * lse.double().abs()[:, None])
    want = 20.0 * (g @ w.double())
    lim = 20.0 * ((ge + 902 * 2.0 ** -22 * g.abs()) @ w.double().abs()) + 1.01 * h * want.abs()
    assert ((dx.double() - want).abs() <= lim).all()


@pytest.mark.gpu
def test_losses_changed_in_place(gpu):
    """reduction "none" hands the losses out; what becomes of them does not
    reach the gradients."""
    import torch
    from vector_cuda import ops
    x, w, t = _sure(50, 300, 64, "bfloat16", 0.5)
    grads = []
    for change in (False, True):
        leaf = x.detach().requires_grad_(True)
        loss = ops.linear_cross_entropy(leaf, w, t, 20.0, "none")
        if change:
            loss *= 1.0
            loss += 3.0
        loss.sum().backward()
        grads.append(leaf.grad)
    assert torch.equal(*grads)


@pytest.mark.parametrize("change", [dict(dl=None), dict(lse=None), dict(loss=None, lse=None), dict(scale=0.0), dict(dws=63)])
def test_backward_with_loss_refuses(vc, change):
    a = dict(dl=4096, scale=1.0, lse=4096, loss=4096, dws=64)
    a.update(change)
    assert vc.lib().vrs_linear_cross_entropy_backward_with_loss(
        a["dl"], 4096, 64, 4, 4096, 64, 10, 64, 2, 4096, a["scale"], a["lse"], a["loss"], 4096, 64, 4096, a["dws"], 4096,
        1 << 40, None) == 5
    assert b"vrs_linear_cross_entropy_backward" in vc.lib().vrs_last_error()


@pytest.mark.gpu
def test_python_refuses_another_loss(gpu):
    import torch
    from vector_cuda import ops
    x, w, t, dl = _make(8, 20, 16, "bfloat16")
    for loss in (dl[:7], dl.double(), dl.cpu(), 3.0):
        with pytest.raises(ValueError):
            ops.linear_cross_entropy_backward(dl, x, w, t, dl, loss=loss)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [60, 700, 9000])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_one_row_of_no_finite_weight(gpu, rows, dtype, bad):
    """An infinite or NaN dloss stays in its row of dx: the other rows are
    rounded and scaled as if that row had weight 0."""
    import torch
    from vector_cuda import ops
    x, w, t, dl = _make(rows, 500, 64, dtype, ignored=0.1)
    dl *= 1024.0
    at = int((t >= 0).nonzero()[3])
    _, lse = ops.linear_cross_entropy_forward(x, w, t)
    dl[at] = 0.0
    want, _ = ops.linear_cross_entropy_backward(dl, x, w, t, lse, need_dtable=False)
    dl[at] = bad
    got, _ = ops.linear_cross_entropy_backward(dl, x, w, t, lse, need_dtable=False)
    assert not torch.isfinite(got[at]).any()
    got[at] = want[at]
    assert torch.isfinite(got).all() and torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,classes,d", [(8, 1398, 75), (1, 1000, 64), (1, 30011, 768), (3, 20000, 500), (64, 5000, 130), (64, 5000, 60),
                                            (1, 300000, 64), (3, 100000, 72), (40, 9000, 264)])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_table_gradients_of_few_rows(gpu, rows, classes, d, dtype):
    """A row of dtable is a sum over rows: with few of them the 16-bit rounding of
    the score gradients has little to average with, so it must not be there: only
    the square of half an ulp (what two 16-bit parts leave), the scores' errors,
    and the result's own half ulp."""
    _few_terms(rows, classes, d, dtype, False)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,classes,d", [(8, 1398, 75), (1000, 2, 64), (5000, 3, 600), (300, 64, 1000), (20000, 17, 130)])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_row_gradients_of_few_classes(gpu, rows, classes, d, dtype):
    """And a row of dx is a sum over classes."""
    _few_terms(rows, classes, d, dtype, True)


def _few_terms(rows, classes, d, dtype, dx):
    import torch
    from vector_cuda import ops
    x, w, t, dl = _make(rows, classes, d, dtype)
    loss, lse = ops.linear_cross_entropy_forward(x, w, t)
    leaves = x.detach().requires_grad_(dx), w.detach().requires_grad_(not dx)
    (ops.linear_cross_entropy(*leaves, t, 1.0, "none") * dl).sum().backward()
    got = leaves[0].grad if dx else leaves[1].grad
    h, f16 = HALF[dtype], dtype == "float16"
    X, W = x.double(), w.double()
    _, g, rel = _sure64(x, w, t, 1.0)
    up = dl.double()[:, None]
    g = g * up
    ge = (1.01 * h * h + 2 * rel[:, None]) * g.abs() + (2.0 ** -38 * up.max() if f16 else 0.0)
    e = (ge + (len(w if dx else t) + 2) * 2.0 ** -22 * g.abs())
    want, e = (g @ W, e @ W.abs()) if dx else (g.t() @ X, e.t() @ X.abs())
    lim = e + 1.01 * h * want.abs() + (2.0 ** -25 if f16 else 0.0)
    off = (got.double() - want).abs()
    assert (off <= lim).all(), f"{int((off > lim).sum())} of {off.numel()} off, worst {(off / lim).max().item():.3g}x"


@pytest.mark.gpu
@pytest.mark.parametrize("which,rows,classes,d", [("dtable", 60, 2000, 300), ("dtable", 64, 5000, 130), ("dtable", 60, 700, 100),
                                                  ("dx", 2000, 40, 300), ("dx", 200, 500, 100), ("dx", 3000, 64, 100)])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_few_terms_in_the_mean(gpu, which, rows, classes, d, dtype):
    """The error's norm over the result's. Rounding values of a normal distribution
    to the nearest gives 0.43 half ulps; score gradients rounded likewise would
    add as much again, 0.6 in all. Half is between."""
    import torch
    from vector_cuda import ops
    x, w, t, dl = _make(rows, classes, d, dtype)
    dl *= 1024.0
    leaves = x.detach().requires_grad_(which == "dx"), w.detach().requires_grad_(which == "dtable")
    (ops.linear_cross_entropy(*leaves, t, 1.0, "none") * dl).sum().backward()
    _, g, _ = _sure64(x, w, t, 1.0)
    g = g * dl.double()[:, None]
    got, want = (leaves[0].grad, g @ w.double()) if which == "dx" else (leaves[1].grad, g.t() @ x.double())
    assert (got.double() - want).norm() <= 0.5 * HALF[dtype] * want.norm()


@pytest.mark.parametrize("backward", [0, 1])
@pytest.mark.parametrize("aligned", [0, 1])
def test_workspace_grows_with_every_size(vc, backward, aligned):
    """A workspace for the largest sizes serves every smaller call: the answer
    never falls as a size grows."""
    import math
    import random
    n = ctypes.c_int64(0)

    def size(rows, classes, d):
        assert vc.lib().vrs_linear_cross_entropy_workspace(rows, classes, d, 2, backward, aligned, ctypes.byref(n)) == 0
        return n.value

    rng = random.Random(3)
    pairs = [((2048, 48000, 1024), (4096, 48000, 1024)), ((1, 1000000, 16), (1, 1000000, 17)),
             ((64, 70000, 64), (65, 70000, 64)), ((256, 70000, 64), (257, 70000, 64)), ((300, 64, 500), (300, 65, 500))]
    for _ in range(4000):
        most = (2 ** 20, 2 ** 21, 2 ** 14)
        a = [round(2 ** rng.uniform(0, math.log2(m))) for m in most]
        b = [max(v, min(m, round(v * 2 ** rng.choice([0, 0, rng.uniform(0, 0.2), rng.uniform(0, 6)])) + rng.choice([0, 0, 1])))
             for v, m in zip(a, most)]
        pairs.append((tuple(a), tuple(b)))
    for a, b in pairs:
        assert size(*a) <= size(*b), f"{a} needs {size(*a)}, {b} {size(*b)}"
