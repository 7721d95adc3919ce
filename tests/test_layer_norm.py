"""Layer norm (vrs_layer_norm_*, vector_cuda.ops): forward and backward passes
against the formulas in 64 bits, gradients against differences, refusals.

Tolerances. With u = 2^-24: a 32-bit sum of the kernel adds at most 32 terms a
thread, then 5 + 3 + 3 levels over lanes, warps and blocks, so its error is
under 48 u sum|terms|. That bounds the mean's error by 48 u mean|x|, and
every element of the normalised row by K u (|xh| + rstd mean|x| + 1) with
K = 160 (three such sums and the roundings of each step). Outputs in 16 bits
add half an ulp. Column sums over R rows add at most R/(blocks) + blocks terms
in order: (R + 64) u sum|terms| bounds them whatever the split."""
import ctypes

import numpy as np
import pytest

U = 2.0 ** -24


def _half_ulp(t):
    import torch
    return {torch.float32: U, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[t]


def _tiny(t):
    """Half the spacing of subnormals."""
    import torch
    return {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}[t]


def _close(got, want, tol, what):
    import torch
    got = got.double()
    tol = torch.as_tensor(tol, dtype=torch.float64, device=got.device)
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {(got - want).abs().max().item():.3g}"


def _check(x, w, b, dy, eps=1e-5):
    import torch
    from vector_cuda import ops
    d = x.shape[-1]
    X = x.double().reshape(-1, d)
    W = torch.ones(d, dtype=torch.float64, device=x.device) if w is None else w.double()
    B = torch.zeros_like(W) if b is None else b.double()
    mean = X.mean(1, keepdim=True)
    rstd = ((X - mean).square().mean(1, keepdim=True) + eps).rsqrt()
    xh = (X - mean) * rstd
    e = 160 * U * (xh.abs() + rstd * X.abs().mean(1, keepdim=True) + 1.0)  # of xh
    y, m, r = ops.layer_norm_forward(x, w, b, eps)
    assert y.shape == x.shape and y.dtype == x.dtype and m.shape == x.shape[:-1] and r.dtype == torch.float32
    want = xh * W + B
    o = _half_ulp(x.dtype)
    _close(y.reshape(-1, d), want, e * W.abs() + 4 * U * want.abs() + o * want.abs() * 1.01 + _tiny(x.dtype), "y")
    _close(m.reshape(-1, 1), mean, 50 * U * X.abs().mean(1, keepdim=True), "mean")
    _close(r.reshape(-1, 1), rstd, 160 * U * rstd * (1 + rstd * X.abs().mean(1, keepdim=True)), "rstd")
    if dy is None:
        return
    D = dy.double().reshape(-1, d)
    G = D * W
    m0, m1 = G.mean(1, keepdim=True), (G * xh).mean(1, keepdim=True)
    dx, dw, db = ops.layer_norm_backward(dy, x, w, m, r)
    want = rstd * (G - m0 - xh * m1)
    a0, a1 = G.abs().mean(1, keepdim=True), (G * xh).abs().mean(1, keepdim=True)
    ea = e.amax(1, keepdim=True) * a0
    er = 160 * U * (1 + rstd * X.abs().mean(1, keepdim=True)) * want.abs()
    tol = rstd * (8 * U * (G.abs() + a0 + xh.abs() * a1) + 48 * U * (a0 + xh.abs() * a1) + e * a1 + xh.abs() * ea) + er
    _close(dx.reshape(-1, d), want, tol + o * want.abs() * 1.01 + _tiny(x.dtype), "dx")
    n = X.shape[0]
    p = _half_ulp(dw.dtype)
    sw, sb = (D * xh).sum(0), D.sum(0)
    _close(dw, sw, (n + 64) * U * (D * xh).abs().sum(0) + (D.abs() * e).sum(0) + p * sw.abs() * 1.01 + _tiny(dw.dtype),
           "dweight")
    _close(db, sb, (n + 64) * U * D.abs().sum(0) + p * sb.abs() * 1.01 + _tiny(db.dtype), "dbias")


def _make(rows, d, dtype, ptype, seed=0, shift=1.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed + rows * 131 + d)
    x = (torch.randn(rows, d, generator=g, device="cuda") * 1.5 + shift).to(dtype)
    w = (1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(ptype)
    b = (0.2 * torch.randn(d, generator=g, device="cuda")).to(ptype)
    dy = torch.randn(rows, d, generator=g, device="cuda").to(dtype)
    return x, w, b, dy


TYPES = [("float32", "float32"), ("float16", "float16"), ("float16", "float32"), ("bfloat16", "bfloat16"),
         ("bfloat16", "float32")]

# One element to the widest row; both sides of every split of a row (512,
# 1024, 2048, 4096, 8192 elements), odd widths, rows fewer and more than blocks.
SIZES = [(1, 1), (3, 2), (5, 7), (1, 384), (9, 512), (7, 513), (33, 1000), (300, 1024), (17, 1025), (1000, 96),
         (5, 2048), (21, 2056), (4, 4096), (3, 4104), (37, 5001), (2, 8192), (3, 8200), (2, 20011), (1, 32768),
         (4000, 64), (2500, 771)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,d", SIZES)
@pytest.mark.parametrize("dtype,ptype", TYPES)
def test_matches_formula(gpu, rows, d, dtype, ptype):
    import torch
    x, w, b, dy = _make(rows, d, getattr(torch, dtype), getattr(torch, ptype))
    _check(x, w, b, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
def test_without_parameters(gpu, weight, bias):
    import torch
    x, w, b, dy = _make(70, 200, torch.bfloat16, torch.bfloat16)
    _check(x, w if weight else None, b if bias else None, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("d,stride,offset", [(256, 264, 0), (256, 300, 0), (256, 257, 0), (255, 256, 0), (256, 264, 1),
                                             (256, 264, 8), (6000, 6001, 3)])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_strided_rows(gpu, d, stride, offset, dtype):
    """Rows inside a wider buffer, on and off 16-byte boundaries; what lies
    between them is not touched and does not count."""
    import torch
    t = getattr(torch, dtype)
    x, w, b, dy = _make(45, d, t, t)
    buf = torch.full((46 * stride + offset,), float("nan"), dtype=t, device="cuda")
    v = buf[offset:offset + 45 * stride].view(45, stride)[:, :d]
    v.copy_(x)
    buf2 = buf.clone()
    v2 = buf2[offset:offset + 45 * stride].view(45, stride)[:, :d]
    v2.copy_(dy)
    _check(v, w, b, v2)


@pytest.mark.gpu
def test_other_layouts(gpu):
    """Leading dimensions, transposed and broadcast inputs."""
    import torch
    x, w, b, dy = _make(60, 128, torch.float32, torch.float32)
    _check(x.view(3, 4, 5, 128), w, b, dy.view(3, 4, 5, 128))
    _check(x.t().contiguous().t(), w, b, dy)
    _check(x[:1].expand(60, 128), w, b, dy[:1].expand(60, 128))
    _check(x[0], w, b, dy[0])


@pytest.mark.gpu
def test_hard_values(gpu):
    """A mean far above the spread, rows without spread, large and infinite
    values (which stay within their row)."""
    import torch
    x, w, b, dy = _make(64, 300, torch.float32, torch.float32, shift=1000.0)
    _check(x, w, b, dy)
    from vector_cuda import ops
    x[3] = 7.0
    x[5, 2] = float("inf")
    x[6, 1] = float("nan")
    y, m, r = ops.layer_norm_forward(x, w, b)
    assert torch.equal(y[3], b) and m[3] == 7.0
    assert not torch.isfinite(y[5]).any() and torch.isnan(y[6]).all()
    keep = [i for i in range(64) if i not in (3, 5, 6)]
    y0, _, _ = ops.layer_norm_forward(x[keep], w, b)
    assert torch.equal(y[keep], y0)


@pytest.mark.gpu
def test_empty_and_repeatable(gpu):
    import torch
    from vector_cuda import ops
    x, w, b, dy = _make(5000, 769, torch.bfloat16, torch.float32)
    y, m, r = ops.layer_norm_forward(x[:0], w, b)
    assert y.shape == (0, 769) and m.shape == (0,)
    dx, dw, db = ops.layer_norm_backward(dy[:0], x[:0], w, m, r)
    assert dx.shape == (0, 769) and not dw.any() and not db.any()
    y, m, r = ops.layer_norm_forward(x, w, b)
    first = ops.layer_norm_backward(dy, x, w, m, r)
    for _ in range(3):
        assert all(torch.equal(p, q) for p, q in zip(first, ops.layer_norm_backward(dy, x, w, m, r)))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,d", [(3, 5), (4, 600)])
def test_gradients_against_differences(gpu, rows, d):
    """f(x, w, b) = sum c y in 32 bits along a random direction: the central
    difference with step h errs by O(h^2) and rounding over h; h = 2^-6 keeps
    both under 1 % of the largest directional derivative here."""
    import torch
    from vector_cuda import ops
    x, w, b, c = _make(rows, d, torch.float32, torch.float32)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    (ops.layer_norm(*leaves) * c).sum().backward()
    g = torch.Generator(device="cuda").manual_seed(9)
    for i, leaf in enumerate(leaves):
        v = torch.randn(leaf.shape, generator=g, device="cuda")
        v /= v.norm()
        h = 2.0 ** -6
        args = [[t.detach() for t in leaves] for _ in range(2)]
        args[0][i] = args[0][i] + h * v
        args[1][i] = args[1][i] - h * v
        f = [(ops.layer_norm_forward(*a)[0].double() * c.double()).sum() for a in args]
        diff = ((f[0] - f[1]) / (2 * h)).item()
        want = (leaf.grad.double() * v.double()).sum().item()
        assert abs(diff - want) <= 0.01 * leaf.grad.norm().item() + 1e-3


@pytest.mark.gpu
def test_stream_and_in_use(gpu):
    """Work goes to the current stream: results are ready to that stream's
    later work without any synchronisation."""
    import torch
    from vector_cuda import ops
    x, w, b, _ = _make(4000, 1024, torch.float32, torch.float32)
    want = ops.layer_norm_forward(x, w, b)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        z = torch.zeros_like(x)
        for _ in range(20):
            z.copy_(x)
            y = ops.layer_norm_forward(z, w, b)[0]
            z.zero_()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, want)


def _forward_status(vc, **k):
    a = dict(x=4096, xs=64, rows=4, d=64, dtype=0, w=None, b=None, pt=0, eps=1e-5, y=4096, ys=64)
    a.update(k)
    return vc.lib().vrs_layer_norm_forward(a["x"], a["xs"], a["rows"], a["d"], a["dtype"], a["w"], a["b"], a["pt"],
                                           a["eps"], a["y"], a["ys"], None, None, None)


@pytest.mark.parametrize("change", [dict(dtype=3), dict(dtype=-1), dict(dtype=1, pt=2), dict(rows=-1), dict(d=0),
                                    dict(d=32769), dict(eps=-1.0), dict(eps=float("nan")), dict(x=None), dict(y=None),
                                    dict(xs=63), dict(ys=10)])
def test_forward_refuses(vc, change):
    """Refused on the host, before any device work (the pointers are never used)."""
    assert _forward_status(vc, **change) == 5
    assert b"vrs_layer_norm_forward" in vc.lib().vrs_last_error()


def test_backward_refuses(vc):
    L = vc.lib()
    n = ctypes.c_int64(0)
    assert L.vrs_layer_norm_backward_workspace(4, 0, ctypes.byref(n)) == 5
    assert L.vrs_layer_norm_backward_workspace(4, 64, None) == 5

    def call(dy=4096, x=4096, rows=4, d=64, dtype=0, pt=0, mean=4096, dx=4096, dxs=64):
        return L.vrs_layer_norm_backward(dy, 64, x, 64, rows, d, dtype, None, pt, mean, 4096, dx, dxs, None, None, None,
                                         0, None)

    for bad in (dict(dy=None), dict(x=None), dict(mean=None), dict(dx=None), dict(dxs=63), dict(dtype=9),
                dict(dtype=1, pt=2), dict(d=40000), dict(rows=-5)):
        assert call(**bad) == 5
        assert b"vrs_layer_norm_backward" in L.vrs_last_error()


def test_python_refuses_cpu_tensors():
    torch = pytest.importorskip("torch")
    from vector_cuda import ops
    with pytest.raises(ValueError, match="CUDA"):
        ops.layer_norm_forward(torch.zeros(3, 4))


@pytest.mark.gpu
def test_python_refusals(gpu):
    import torch
    from vector_cuda import ops
    x = torch.zeros(4, 64, device="cuda")
    one = torch.ones(64, device="cuda")
    for bad in (lambda: ops.layer_norm_forward(x.double()), lambda: ops.layer_norm_forward(x, one[:63]),
                lambda: ops.layer_norm_forward(x, one.half()), lambda: ops.layer_norm_forward(x, one.cpu()),
                lambda: ops.layer_norm_forward(x[:, :0])):
        with pytest.raises(ValueError):
            bad()
    y, m, r = ops.layer_norm_forward(x, one)
    for bad in (lambda: ops.layer_norm_backward(y.half(), x, one, m, r),
                lambda: ops.layer_norm_backward(y[:3], x, one, m, r),
                lambda: ops.layer_norm_backward(y, x, one, m[:3], r)):
        with pytest.raises(ValueError):
            bad()
    assert np.isfinite(y.cpu().numpy()).all()


# (rows, d, stride - d, offset): rows of 16-bit elements that all start on 4-byte
# words, all between them, and alternately (odd strides, with even and odd
# starts), one row and fewer rows than a turn, each width class, a last row whose
# end is the tensor's.
@pytest.mark.gpu
@pytest.mark.parametrize("rows,d,gap,offset", [
    (1, 1, 0, 1), (3, 1, 0, 1), (5, 2, 0, 0), (5, 2, 1, 1), (7, 7, 0, 0), (70, 30, 0, 1), (301, 255, 0, 0),
    (301, 256, 0, 1), (90, 256, 1, 0), (77, 257, 0, 1), (700, 511, 2, 0), (150, 512, 0, 1), (333, 1023, 0, 1),
    (65, 4095, 0, 0), (66, 4096, 0, 1), (67, 4097, 0, 0), (130, 8192, 0, 1), (131, 8193, 0, 1), (3, 9001, 0, 0),
    (70, 32767, 0, 1), (66, 32768, 0, 1)])
@pytest.mark.parametrize("dtype,ptype", [("float16", "float16"), ("bfloat16", "float32")])
def test_rows_at_any_element(gpu, vc, rows, d, gap, offset, dtype, ptype):
    import torch
    t, p = getattr(torch, dtype), getattr(torch, ptype)
    code = {"float32": 0, "float16": 1, "bfloat16": 2}
    x, w, b, dy = _make(rows, d, t, p)
    stride = d + gap
    span = (rows - 1) * stride + d

    def inside(values=None):
        """rows x d within NaN, starting `offset` elements on."""
        whole = torch.full((span + 16,), float("nan"), dtype=t, device="cuda")
        part = torch.as_strided(whole, (rows, d), (stride, 1), 8 + offset)
        if values is not None:
            part.copy_(values)
        return whole, part

    def beside(whole, part):
        """Whether the elements around the rows are what they were."""
        seen = torch.isnan(whole)
        torch.as_strided(seen, (rows, d), (stride, 1), 8 + offset).fill_(True)
        return bool(seen.all())

    (xw, xp), (yw, yp), (gw, gp), (dw_, dp) = inside(x), inside(), inside(dy), inside()
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    dweight, dbias = torch.empty(d, dtype=p, device="cuda"), torch.empty(d, dtype=p, device="cuda")
    L, P, I = vc.lib(), ctypes.c_void_p, ctypes.c_int64
    n = ctypes.c_int64()
    assert L.vrs_layer_norm_backward_workspace(I(rows), I(d), ctypes.byref(n)) == 0
    ws = torch.empty(max(1, n.value), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    assert L.vrs_layer_norm_forward(P(xp.data_ptr()), I(stride), I(rows), I(d), code[dtype], P(w.data_ptr()),
                                    P(b.data_ptr()), code[ptype], ctypes.c_float(1e-5), P(yp.data_ptr()), I(stride),
                                    P(mean.data_ptr()), P(rstd.data_ptr()), None) == 0
    assert L.vrs_layer_norm_backward(P(gp.data_ptr()), I(stride), P(xp.data_ptr()), I(stride), I(rows), I(d),
                                     code[dtype], P(w.data_ptr()), code[ptype], P(mean.data_ptr()),
                                     P(rstd.data_ptr()), P(dp.data_ptr()), I(stride), P(dweight.data_ptr()),
                                     P(dbias.data_ptr()), P(ws.data_ptr()), I(n.value), None) == 0
    torch.cuda.synchronize()
    assert beside(yw, yp) and beside(dw_, dp)
    X, W, B, D = x.double(), w.double(), b.double(), dy.double()
    m = X.mean(1, keepdim=True)
    r = ((X - m).square().mean(1, keepdim=True) + 1e-5).rsqrt()
    xh, G = (X - m) * r, D * W
    e = 160 * U * (xh.abs() + r * X.abs().mean(1, keepdim=True) + 1.0)
    o = _half_ulp(t)
    want = xh * W + B
    _close(yp, want, e * W.abs() + 4 * U * want.abs() + o * want.abs() * 1.01 + _tiny(t), "y")
    want = r * (G - G.mean(1, keepdim=True) - xh * (G * xh).mean(1, keepdim=True))
    a0, a1 = G.abs().mean(1, keepdim=True), (G * xh).abs().mean(1, keepdim=True)
    er = 160 * U * (1 + r * X.abs().mean(1, keepdim=True)) * want.abs()
    tol = r * (8 * U * (G.abs() + a0 + xh.abs() * a1) + 48 * U * (a0 + xh.abs() * a1) + e * a1 +
               xh.abs() * e.amax(1, keepdim=True) * a0) + er
    _close(dp, want, tol + o * want.abs() * 1.01 + _tiny(t), "dx")
    sw, sb, q = (D * xh).sum(0), D.sum(0), _half_ulp(p)
    _close(dweight, sw, (rows + 64) * U * (D * xh).abs().sum(0) + (D.abs() * e).sum(0) + q * sw.abs() * 1.01 + _tiny(p),
           "dweight")
    _close(dbias, sb, (rows + 64) * U * D.abs().sum(0) + q * sb.abs() * 1.01 + _tiny(p), "dbias")


# Rows enough to fill the device: widths between powers of two, and odd ones.
@pytest.mark.gpu
@pytest.mark.parametrize("rows,d", [(12000, 96), (10001, 71), (6000, 136), (3000, 384), (3001, 383), (1300, 700),
                                    (700, 1500), (401, 3000), (333, 3071)])
@pytest.mark.parametrize("dtype,ptype", TYPES)
def test_many_rows(gpu, rows, d, dtype, ptype):
    import torch
    x, w, b, dy = _make(rows, d, getattr(torch, dtype), getattr(torch, ptype))
    _check(x, w, b, dy)


@pytest.mark.gpu
def test_workspace_grows_with_every_size(gpu, vc):
    """A workspace for the largest sizes serves every smaller call."""
    n = ctypes.c_int64(0)

    def size(rows, d):
        assert vc.lib().vrs_layer_norm_backward_workspace(rows, d, ctypes.byref(n)) == 0
        return n.value

    widths = sorted({w for k in range(16) for w in (2 ** k - 1, 2 ** k, 2 ** k + 1) if 1 <= w <= 32768} |
                    {4096 * k + o for k in range(1, 8) for o in (-1, 0, 1)} | {771, 6000, 20011, 32767, 32768})
    counts = [1, 2, 3, 17, 18, 19, 20, 36, 37, 38, 64, 65, 73, 74, 75, 98, 99, 148, 149, 200, 295, 296, 297, 1000, 10 ** 6]
    for rows in counts:
        for narrow, wide in zip(widths, widths[1:]):
            assert size(rows, narrow) <= size(rows, wide), (rows, narrow, wide)
    for d in widths:
        for few, many in zip(counts, counts[1:]):
            assert size(few, d) <= size(many, d), (few, many, d)


@pytest.mark.gpu
def test_gradients_have_their_parameters_shape(gpu):
    """Any shape of d values is taken for weight and bias; gradients come back in it."""
    import torch
    from vector_cuda import ops
    x, w, b, dy = _make(6, 40, torch.float32, torch.float32)
    flat = [t.clone().requires_grad_(True) for t in (x, w, b)]
    shaped = [x.clone().requires_grad_(True), w.view(1, 40).clone().requires_grad_(True),
              b.view(4, 10).clone().requires_grad_(True)]
    (ops.layer_norm(*flat) * dy).sum().backward()
    (ops.layer_norm(*shaped) * dy).sum().backward()
    for p, q in zip(flat, shaped):
        assert q.grad.shape == q.shape and torch.equal(q.grad.reshape(p.shape), p.grad)


@pytest.mark.gpu
@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("dtype,ptype", [("float32", "float32"), ("bfloat16", "float32"), ("float16", "float16")])
@pytest.mark.parametrize("wanted", ["x", "parameters", "all"])
def test_autograd_without_some(gpu, weight, bias, dtype, ptype, wanted):
    """Parameters that are missing, or whose gradient nobody asks for."""
    import torch
    from vector_cuda import ops
    x, w, b, dy = _make(30, 136, getattr(torch, dtype), getattr(torch, ptype))
    w, b = w if weight else None, b if bias else None
    if w is None and b is None and wanted == "parameters":
        pytest.skip("no gradient at all")
    y, m, r = ops.layer_norm_forward(x, w, b)
    want = ops.layer_norm_backward(dy, x, w, m, r, None if b is None else b.dtype)
    leaves = [None if t is None else t.clone().requires_grad_(wanted != ("parameters" if i == 0 else "x"))
              for i, t in enumerate((x, w, b))]
    ops.layer_norm(*leaves).backward(dy)
    for leaf, g in zip(leaves, want):
        if leaf is None:
            continue
        assert (leaf.grad is None) == (not leaf.requires_grad)
        assert leaf.grad is None or (leaf.grad.dtype == leaf.dtype and torch.equal(leaf.grad, g))
