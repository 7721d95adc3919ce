"""Attention over packed sequences (vrs_attention_*, vector_cuda.ops): output,
log-sum-exp and gradients against the formulas in 64 bits, differences, refusals.

Tolerances. Products of 16-bit operands are exact in 32 bits; a score is a sum of d
of them, off by at most (d + 2) 2^-22 scale sum|q k| (4 ulps a term, so that a
truncating accumulator is allowed), and 2^-22 |z| for its factor and shift before
the exponential. z_e, the largest such sum in a row, bounds the error of lse up to the
32-bit exponentials and sums: 2^-20 + 2^-22 |lse|. A weight is then off by the
factor 2 z_e + 2^-20, once more for the sum that divides it, and is rounded to 16
bits as an operand of the product with v (h = 2^-11 or 2^-8; f16 also 2^-32 of the
row's largest weight, where its range ends). With n keys
  |out - exact| <= (h + 4 z_e + 2^-18 + n 2^-22) sum p |v|, plus half an ulp of out.
Backward p is formed again from lse, off by w = 3 z_e + 2^-19 + 2^-21 |lse| of itself, and rounded
(h) for dv = p^T dout. delta = dout . out is that of the rounded out that the pass is
given, summed in 32 bits; ds = p (dp - delta) is off by w |ds| + p e, e = (d + 2) 2^-22
(sum |dout v| + sum |dout out|), and rounded (h; f16: relative to a bound B of all of them,
2^-38 of it) for dq = scale ds k and dk = scale ds^T q, whose sums
add n 2^-22 of their terms. Each result ends with half an ulp of its type."""
import ctypes
import math

import pytest

HALF = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float16": 2.0 ** -25, "bfloat16": 2.0 ** -133}


def _bounds(lengths):
    import torch
    ends = [0]
    for n in lengths:
        ends.append(ends[-1] + n)
    return torch.tensor(ends, dtype=torch.int32, device="cuda")


def _make(lengths, heads, kv, d, dtype, behind=0, seed=0, spread=1.5):
    import torch
    tokens = sum(lengths) + behind
    g = torch.Generator(device="cuda").manual_seed(seed + tokens * 7 + heads * 3 + d)

    def normal(n):
        return torch.randn(tokens, n, d, generator=g, device="cuda")

    dt = getattr(torch, dtype)
    return ((normal(heads) * spread).to(dt), normal(kv).to(dt), normal(kv).to(dt), normal(heads).to(dt))


def _seen(tokens, lengths, causal, device="cuda"):
    """Which keys each query sees."""
    import torch
    seq = torch.full((tokens,), -1, dtype=torch.long)
    at = 0
    for b, n in enumerate(lengths):
        seq[at:at + n] = b
        at += n
    seq = seq.to(device)
    i = torch.arange(tokens, device=device)
    m = (seq[:, None] == seq[None]) & (seq[:, None] >= 0)
    return m & (i[None] <= i[:, None]) if causal else m


def _off(got, want, lim, what):
    off = (got.double() - want).abs()
    assert (off <= lim).all(), f"{what}: {int((~(off <= lim)).sum())} of {off.numel()} off, worst {(off / lim).nan_to_num(9e9).max().item():.3g}x"


def _check(q, k, v, do, lengths, causal=True, scale=None, cu=True, back=True, call=None):
    """Every head's results against 64 bits; returns (out, lse, dq, dk, dv)."""
    import torch
    from vector_cuda import ops
    tokens, heads, d = q.shape[0], q.shape[1], q.shape[2]
    kv = k.shape[1]
    dtype = str(q.dtype).replace("torch.", "")
    h, tiny, f16 = HALF[dtype] * 1.01, TINY[dtype], dtype == "float16"
    bounds = _bounds(lengths) if cu else None
    out, lse = ops.attention_forward(q, k, v, bounds, causal, scale)
    assert out.dtype == q.dtype and out.shape == q.shape and lse.shape == (heads, tokens) and lse.dtype == torch.float32
    grads = ops.attention_backward(do, q, k, v, out, lse, bounds, causal, scale) if back else None
    seen = _seen(tokens, lengths, causal)
    some = seen.any(1)
    s = 1.0 / math.sqrt(d) if scale is None else scale
    for kh in range(kv):
        dk = dv = dk_e = dv_e = dk_t = dv_t = 0.0
        for qh in range(kh * heads // kv, (kh + 1) * heads // kv):
            Q, K, V = q[:, qh].double(), k[:, kh].double(), v[:, kh].double()
            z = torch.where(seen, s * (Q @ K.t()), -math.inf)
            size = torch.where(seen, s * (Q.abs() @ K.abs().t()), 0.0)
            ze = ((d + 2) * 2.0 ** -22 * size + 2.0 ** -22 * torch.where(seen, z.abs(), 0.0)).amax(1, keepdim=True)
            want = torch.logsumexp(z, 1)
            assert (lse[qh][~some] == -math.inf).all()
            _off(lse[qh][some], want[some], (ze[:, 0] + 2.0 ** -20 + 2.0 ** -22 * want.abs())[some], "lse")
            p = torch.where(seen, torch.exp(z - torch.where(some, want, 0.0)[:, None]), 0.0)
            n = seen.sum(1, keepdim=True)
            o = p @ V
            small = 2.0 ** -32 * p.amax(1, keepdim=True) * (seen.double() @ V.abs()) if f16 else 0.0
            _off(out[:, qh], o, (h + 4 * ze + 2.0 ** -18 + n * 2.0 ** -22) * (p @ V.abs()) + small + h * o.abs() + tiny, "out")
            assert not out[:, qh][~some].any()
            if not back:
                continue
            D, O = do[:, qh].double(), out[:, qh].double()
            dp, delta = D @ V.t(), (D * O).sum(1, keepdim=True)
            ds = p * (dp - delta)
            w = 3 * ze + 2.0 ** -19 + 2.0 ** -21 * torch.where(some, want, 0.0).abs()[:, None]
            e = (d + 2) * 2.0 ** -22 * (D.abs() @ V.abs().t() + (D * O).abs().sum(1, keepdim=True))
            ds_e = (h + w) * ds.abs() + p * e
            if f16:
                bound = 4 * max(do[:, x].double().square().sum(1).max() for x in range(heads)).sqrt() * max(
                    v[:, x].double().square().sum(1).max() for x in range(kv)).sqrt()
                ds_e = ds_e + 2.0 ** -38 * bound * seen
            p_e = (h + w) * p + (2.0 ** -38 * seen if f16 else 0.0)
            dq = s * (ds @ K)
            _off(grads[0][:, qh], dq, s * (ds_e @ K.abs() + n * 2.0 ** -22 * (ds.abs() @ K.abs())) + h * dq.abs() + tiny, "dq")
            assert not grads[0][:, qh][~some].any()
            m = seen.sum(0)[:, None] * (heads // kv)
            dk, dv = dk + s * (ds.t() @ Q), dv + p.t() @ D
            dk_e = dk_e + s * (ds_e.t() @ Q.abs() + m * 2.0 ** -22 * (ds.abs().t() @ Q.abs()))
            dv_e = dv_e + p_e.t() @ D.abs() + m * 2.0 ** -22 * (p.t() @ D.abs())
        if back:
            _off(grads[1][:, kh], dk, dk_e + h * dk.abs() + tiny, "dk")
            _off(grads[2][:, kh], dv, dv_e + h * dv.abs() + tiny, "dv")
            assert not grads[1][:, kh][~some].any() and not grads[2][:, kh][~some].any()
    return (out, lse, *grads) if back else (out, lse)


# Lengths: one token, both sides of a tile and of two, several in a tile, empty
# ones, tokens behind the last sequence.
CASES = [([1], 1, 1, 64, 0), ([2], 2, 1, 8, 0), ([127], 2, 2, 64, 0), ([128], 1, 1, 128, 0), ([129], 4, 2, 128, 3),
         ([256], 3, 1, 64, 0), ([257, 1], 2, 2, 128, 0), ([300], 6, 2, 96, 0), ([3, 0, 50, 1, 1, 0, 90], 4, 4, 64, 0),
         ([5] * 60, 2, 1, 32, 11), ([100, 28, 128, 7], 3, 3, 80, 0), ([1000], 2, 1, 128, 0), ([513, 700, 90], 5, 5, 72, 130),
         ([0, 0], 2, 2, 64, 20), ([640, 2, 600], 8, 2, 16, 0), ([1] * 200, 1, 1, 64, 100), ([2050], 2, 2, 48, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths,heads,kv,d,behind", CASES, ids=[str(i) for i in range(len(CASES))])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_forward_matches_formula(gpu, lengths, heads, kv, d, behind, causal, dtype):
    _check(*_make(lengths, heads, kv, d, dtype, behind), lengths, causal, back=False)


# Heads and tiles enough that items are pairs of heads (even groups), pairs of
# tiles, and more than one turn of the device.
@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths,heads,kv,d", [([900, 1300], 32, 4, 64), ([700, 31, 900], 27, 9, 128),
                                                ([1500], 40, 40, 32), ([60] * 30, 24, 12, 128)])
def test_forward_many_items(gpu, lengths, heads, kv, d, causal):
    _check(*_make(lengths, heads, kv, d, "bfloat16", 5), lengths, causal, back=False)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths,heads,kv,d,behind", CASES, ids=[str(i) for i in range(len(CASES))])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_gradients_match_formula(gpu, lengths, heads, kv, d, behind, causal, dtype):
    _check(*_make(lengths, heads, kv, d, dtype, behind, seed=1), lengths, causal)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths,heads,kv,d", [([900, 1300], 16, 4, 64), ([700, 31, 900], 27, 9, 128),
                                                ([1500], 14, 14, 32), ([60] * 30, 24, 12, 128)])
def test_gradients_many_items(gpu, lengths, heads, kv, d, causal):
    _check(*_make(lengths, heads, kv, d, "bfloat16", 5), lengths, causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("scale", [1e-3, 0.5, 3.0])
def test_scale(gpu, scale, dtype):
    """From nearly even weights to single keys whose scores are some hundreds: the running reference has to grow."""
    _check(*_make([300, 150], 2, 1, 64, dtype), [300, 150], True, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_growing_scores(gpu, dtype):
    """Each tile of keys has larger scores than all before it, and the other way round."""
    import torch
    q, k, v, do = _make([700], 2, 1, 64, dtype)
    steps = torch.linspace(0.05, 4.0, 700, device="cuda").to(q.dtype)[:, None, None]
    q = q.abs()
    _check(q, k.abs() * steps, v, do, [700], False)
    _check(q, k.abs() * steps.flip(0), v, do, [700], False)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [2.0 ** -20, 2.0 ** -12, 2.0 ** 8])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_gradients_of_any_size(gpu, size, dtype):
    """dout far from 1 (2^-20 is below float16's normal numbers)."""
    q, k, v, do = _make([260, 70], 4, 2, 64, dtype)
    _check(q, k, v, do * size, [260, 70])


@pytest.mark.gpu
def test_rows_of_very_different_weight(gpu):
    q, k, v, do = _make([200], 2, 2, 64, "float16")
    do[::2] *= 2.0 ** -10
    do[7] = 0.0
    _check(q, k, v, do, [200])


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
def test_batch_is_sequences_of_one_length(gpu, causal):
    import torch
    from vector_cuda import ops
    q, k, v, do = _make([150] * 5, 6, 3, 64, "bfloat16")
    want = _check(q, k, v, do, [150] * 5, causal)
    b = [t.view(5, 150, *t.shape[1:]) for t in (q, k, v, do)]
    out, lse = ops.attention_forward(*b[:3], causal=causal)
    grads = ops.attention_backward(b[3], *b[:3], out, lse, causal=causal)
    assert out.shape == b[0].shape and grads[1].shape == b[1].shape
    for a, w in zip((out, lse, *grads), want):
        assert torch.equal(a.reshape(w.shape), w)
    # one sequence without bounds
    want = _check(q, k, v, do, [750], causal)
    assert torch.equal(ops.attention_forward(q, k, v, causal=causal)[0], want[0])


@pytest.mark.gpu
@pytest.mark.parametrize("way", ["projection", "gaps", "odd", "heads first", "elements apart", "expanded"])
def test_views(gpu, way):
    import torch
    from vector_cuda import ops
    lengths, heads, kv, d = [130, 71], 4, 2, 64
    q, k, v, do = _make(lengths, heads, kv, d, "float16")
    want = _check(q, k, v, do, lengths)
    t = 201
    if way == "projection":
        w = torch.cat((q, k, v), 1)
        q, k, v = w[:, :4], w[:, 4:6], w[:, 6:]
    elif way in ("gaps", "odd"):
        pad = 16 if way == "gaps" else 3
        def inside(x):
            b = torch.full((t, x.shape[1] * d + pad), float("nan"), dtype=x.dtype, device="cuda")
            s = b[:, pad // 2:pad // 2 + x.shape[1] * d] if way == "odd" else b[:, :x.shape[1] * d]
            s = s.view(t, x.shape[1], d)
            s.copy_(x)
            return s
        q, k, v, do = (inside(x) for x in (q, k, v, do))
    elif way == "heads first":
        q, k, v, do = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v, do))
    elif way == "elements apart":
        q, k, v, do = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v, do))
    else:
        do = torch.ones((), dtype=q.dtype, device="cuda").expand(t, heads, d)
        want = _check(q, k, v, do.contiguous(), lengths)
    cu = _bounds(lengths)
    out, lse = ops.attention_forward(q, k, v, cu)
    got = (out, lse, *ops.attention_backward(do, q, k, v, out, lse, cu))
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.gpu
@pytest.mark.parametrize("d", [1, 7, 20, 33, 100, 127])
def test_widths_that_no_eight_divides(gpu, d):
    _check(*_make([140, 9], 2, 1, d, "bfloat16"), [140, 9])


@pytest.mark.gpu
def test_either_gradient_alone(gpu):
    import torch
    from vector_cuda import ops
    q, k, v, do = _make([200, 90], 4, 2, 64, "bfloat16")
    cu = _bounds([200, 90])
    out, lse = ops.attention_forward(q, k, v, cu)
    dq, dk, dv = ops.attention_backward(do, q, k, v, out, lse, cu)
    a = ops.attention_backward(do, q, k, v, out, lse, cu, need_dkv=False)
    b = ops.attention_backward(do, q, k, v, out, lse, cu, need_dq=False)
    assert torch.equal(a[0], dq) and a[1] is None and a[2] is None
    assert b[0] is None and torch.equal(b[1], dk) and torch.equal(b[2], dv)
    assert ops.attention_backward(do, q, k, v, out, lse, cu, need_dq=False, need_dkv=False) == (None, None, None)


@pytest.mark.gpu
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("causal,lengths,at", [(True, [300], 299), (True, [300], 140), (True, [90, 100, 60], 130),
                                               (False, [90, 100, 60], 130), (False, [200, 300, 7, 200], 505), (True, [40], 0)])
def test_not_finite_reaches_only_what_sees_it(gpu, causal, lengths, at, dtype, value):
    """A token whose key, value, query or output gradient is not finite: rows that
    do not see it keep their bits, rows that do say so."""
    import torch
    from vector_cuda import ops
    heads, kv, d = 4, 2, 64
    clean = list(_make(lengths, heads, kv, d, dtype, behind=9))
    tokens = clean[0].shape[0]
    cu = _bounds(lengths)

    def run(q, k, v, do):
        out, lse = ops.attention_forward(q, k, v, cu, causal)
        return (out, lse, *ops.attention_backward(do, q, k, v, out, lse, cu, causal))

    want = run(*clean)
    seen = _seen(tokens, lengths, causal)
    sees = seen[:, at]          # queries that see the token
    back = seen[sees].any(0)    # keys that those see
    own = seen[at]              # keys that the token sees
    for which in range(4):
        bad = [t.clone() for t in clean]
        bad[which][at, 1, 5] = value
        out, lse, dq, dk, dv = run(*bad)
        same = lambda a, b, rows: torch.equal(a[rows].view(torch.int16), b[rows].view(torch.int16))
        if which == 0:    # a query: its own row, and the keys it sees
            rows, keys = torch.arange(tokens, device="cuda") == at, own
        elif which == 3:
            rows, keys = torch.arange(tokens, device="cuda") == at, own
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        else:
            rows, keys = sees, back
        assert same(out, want[0], ~rows) and same(dq, want[2], ~rows)
        assert same(dk, want[3], ~keys) and same(dv, want[4], ~keys)
        assert torch.equal(lse[:, ~rows], want[1][:, ~rows])
        # the heads that do not use it keep everything
        group = slice(2, 4) if which in (1, 2) else slice(1, 2)
        others = [h for h in range(heads) if not (group.start <= h < group.stop)]
        assert same(out[:, others], want[0][:, others], torch.ones(tokens, dtype=torch.bool))
        if which == 3:
            # dout reaches dv of every key it sees (weights are above 0 here)
            assert not torch.isfinite(dv[own, 0, 5]).any()
        elif which == 2:
            assert not torch.isfinite(out[sees][:, 2:4, 5]).any()
        elif math.isnan(value):
            assert out[rows][:, group].isnan().all() and dq[rows][:, group].isnan().all()


@pytest.mark.gpu
def test_everything_not_finite(gpu):
    """A training run that has gone wrong ends with NaN, in a bounded time."""
    import torch
    from vector_cuda import ops
    q, k, v, do = (torch.full_like(t, float("nan")) for t in _make([700, 300, 90], 4, 2, 128, "bfloat16"))
    cu = _bounds([700, 300, 90])
    out, lse = ops.attention_forward(q, k, v, cu)
    grads = ops.attention_backward(do, q, k, v, out, lse, cu)
    assert all(t.isnan().all() for t in (out, lse, *grads))


@pytest.mark.gpu
def test_bounds_without_meaning_reach_no_other_memory(gpu):
    """cu_seqlens that fall, are negative or lie past the end: results without meaning, nothing else."""
    import torch
    from vector_cuda import ops
    q, k, v, do = _make([300], 2, 1, 64, "bfloat16")
    for bounds in ([0, 200, 100, 300], [-50, 100, 1000], [2 ** 31 - 1, -2 ** 31], [5, 5, 5], [300, 0], [7]):
        cu = torch.tensor(bounds, dtype=torch.int32, device="cuda")
        out, lse = ops.attention_forward(q, k, v, cu)
        ops.attention_backward(do, q, k, v, out, lse, cu)
    ops.check()
    _check(q, k, v, do, [300])


@pytest.mark.gpu
def test_rows_between_and_around_results_stay(gpu, vc):
    """C entry: results with strides of their own; what lies between is left alone."""
    import torch
    from vector_cuda import ops
    lengths, heads, kv, d = [150, 60], 4, 2, 72
    q, k, v, do = _make(lengths, heads, kv, d, "float16", behind=3)
    want = _check(q, k, v, do, lengths)
    L, i64, cu, t = vc.lib(), ctypes.c_int64, _bounds(lengths), 213

    class Heads(ctypes.Structure):
        _fields_ = [("data", ctypes.c_void_p), ("stride", i64), ("head", i64)]

    def of(x):
        return Heads(x.data_ptr(), x.stride(0), x.stride(1))

    def wide(n):
        b = torch.full((t + 2, n * 80 + 24), 7.0, dtype=q.dtype, device="cuda")
        return b, b[1:-1, 8:8 + n * 80].view(t, n, 80)[:, :, :72]

    rest = (i64(t), i64(heads), i64(kv), i64(d), 1, ctypes.c_void_p(cu.data_ptr()), i64(2), 1, ctypes.c_float(72 ** -0.5))
    n = i64(0)
    assert L.vrs_attention_forward_workspace(i64(t), ctypes.byref(n)) == 0
    ws = torch.empty(n.value, dtype=torch.uint8, device="cuda")
    bo, o = wide(heads)
    lse = torch.empty(heads, t, device="cuda")
    r = ctypes.byref
    assert L.vrs_attention_forward(r(of(q)), r(of(k)), r(of(v)), *rest, r(of(o)), ctypes.c_void_p(lse.data_ptr()),
                                   ctypes.c_void_p(ws.data_ptr()), n, None) == 0, L.vrs_last_error()
    torch.cuda.synchronize()
    assert L.vrs_attention_backward_workspace(i64(t), i64(heads), ctypes.byref(n)) == 0
    ws = torch.empty(n.value, dtype=torch.uint8, device="cuda")
    (bq, gq), (bk, gk), (bv, gv) = wide(heads), wide(kv), wide(kv)
    assert L.vrs_attention_backward(r(of(do)), r(of(q)), r(of(k)), r(of(v)), r(of(o)), ctypes.c_void_p(lse.data_ptr()), *rest,
                                    r(of(gq)), r(of(gk)), r(of(gv)), ctypes.c_void_p(ws.data_ptr()), n, None) == 0, L.vrs_last_error()
    torch.cuda.synchronize()
    assert torch.equal(lse, want[1])
    for b, x, w in ((bo, o, want[0]), (bq, gq, want[2]), (bk, gk, want[3]), (bv, gv, want[4])):
        assert torch.equal(x, w)
        x.fill_(7.0)
        assert (b == 7.0).all()


@pytest.mark.gpu
def test_same_bits_captured_and_on_another_stream(gpu):
    import torch
    from vector_cuda import ops
    lengths = [700, 33, 600]
    q, k, v, do = _make(lengths, 8, 2, 128, "float16", behind=40)
    cu = _bounds(lengths)

    def both():
        out, lse = ops.attention_forward(q, k, v, cu)
        return (out, lse, *ops.attention_backward(do, q, k, v, out, lse, cu))

    want = both()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(want, both()))
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for side in sides:  # two calls at once
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got.append(both())
    for side in sides:
        torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for g in got for a, b in zip(want, g))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for _ in range(2):
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    # other lengths in the captured call: the bounds are read by the device
    cu.copy_(_bounds([100, 1000, 10]))
    graph.replay()
    got = [t.clone() for t in got]
    assert all(torch.equal(a, b) for a, b in zip(both(), got))
    ops.check()


@pytest.mark.gpu
def test_autograd_against_differences(gpu):
    import torch
    from vector_cuda import ops
    g = torch.Generator(device="cuda").manual_seed(3)
    lengths, heads, kv, d = [9, 20], 2, 1, 16
    cu = _bounds(lengths)
    x = [(torch.randn(29, n, d, generator=g, device="cuda") * 0.5).half().requires_grad_(True) for n in (heads, kv, kv)]
    w = torch.randn(29, heads, d, generator=g, device="cuda").half()
    (ops.attention(*x, cu) * w).sum().backward()

    def f(q, k, v):
        z = torch.where(_seen(29, lengths, True)[None], torch.einsum("ihd,jhd->hij", q, k.expand(-1, heads, -1)) / 4.0, -math.inf)
        return (torch.einsum("hij,jhd->ihd", torch.softmax(z, 2), v.expand(-1, heads, -1)) * w.double()).sum().item()

    at = [t.detach().double() for t in x]
    for i, t in enumerate(x):
        u = torch.randn(t.shape, generator=g, device="cuda").double()
        step = 1e-4
        ends = [f(*[a + s * step * u if j == i else a for j, a in enumerate(at)]) for s in (1, -1)]
        want = (ends[0] - ends[1]) / (2 * step)
        # half ulps of the result, of p, ds and out: each at most 2^-11 of a term
        lim = 2.0 ** -8 * (t.grad.double().abs() * u.abs()).sum().item() + 1e-3
        assert abs((t.grad.double() * u).sum().item() - want) <= lim


@pytest.mark.gpu
def test_autograd_needs(gpu):
    """Leaves that want no gradient get none; the others' bits do not change."""
    import torch
    from vector_cuda import ops
    q, k, v, do = _make([70], 2, 1, 64, "bfloat16")
    cu = _bounds([70])
    out, lse = ops.attention_forward(q, k, v, cu)
    want = ops.attention_backward(do, q, k, v, out, lse, cu)
    for mask in range(1, 8):
        x = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((q, k, v))]
        ops.attention(*x, cu).backward(do)
        for i, t in enumerate(x):
            assert (t.grad is None) if not mask >> i & 1 else torch.equal(t.grad, want[i])


@pytest.mark.gpu
def test_no_tokens(gpu):
    import torch
    from vector_cuda import ops
    q, k, v, do = (torch.zeros(0, n, 64, dtype=torch.bfloat16, device="cuda") for n in (4, 2, 2, 4))
    for cu in (None, torch.zeros(3, dtype=torch.int32, device="cuda")):
        out, lse = ops.attention_forward(q, k, v, cu)
        assert out.shape == q.shape and lse.shape == (4, 0)
        assert [t.shape for t in ops.attention_backward(do, q, k, v, out, lse, cu)] == [q.shape, k.shape, v.shape]


@pytest.mark.gpu
def test_python_refusals(gpu):
    import torch
    from vector_cuda import ops
    q, k, v, do = _make([20], 4, 2, 64, "float16")
    cu = _bounds([20])
    for a in ((q.float(), k.float(), v.float(), cu), (q, k.bfloat16(), v, cu), (q, k[:, :1], v, cu), (q[:, :3], k, v, cu),
              (q, k[:19], v, cu), (q.cpu(), k.cpu(), v.cpu(), cu), (q, k, v, cu.long()), (q, k, v, cu.cpu()),
              (q, k, v, cu[:0]), (q, k, v, cu[None]), (q[None], k[None], v[None], cu), (q[0], k[0], v[0], cu),
              (q, k, v[..., :32], cu)):
        with pytest.raises(ValueError):
            ops.attention(*a)
    for scale in (0.0, -1.0, math.inf, math.nan, 1e-60):
        with pytest.raises(ValueError):
            ops.attention(q, k, v, cu, True, scale)
    wide = torch.zeros(5, 2, 136, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError, match="128"):
        ops.attention(wide, wide, wide)
    out, lse = ops.attention_forward(q, k, v, cu)
    for a in ((do[:19], q, k, v, out, lse), (do, q, k, v, out[:, :2], lse), (do, q, k, v, out, lse[:, :5]),
              (do.bfloat16(), q, k, v, out, lse), (do, q, k, v, out, lse.double())):
        with pytest.raises(ValueError):
            ops.attention_backward(*a, cu)


def test_c_refusals(vc):
    """Wrong arguments are told by status before anything is queued (no GPU needed)."""
    L, i64, r = vc.lib(), ctypes.c_int64, ctypes.byref

    class Heads(ctypes.Structure):
        _fields_ = [("data", ctypes.c_void_p), ("stride", i64), ("head", i64)]

    n = i64(0)
    assert L.vrs_attention_forward_workspace(i64(100), r(n)) == 0
    small = n.value
    assert L.vrs_attention_forward_workspace(i64(1000), r(n)) == 0 and n.value >= small > 0
    assert L.vrs_attention_forward_workspace(i64(-1), r(n)) == 5
    sizes = []
    for t, h in ((100, 2), (100, 4), (1000, 4)):
        assert L.vrs_attention_backward_workspace(i64(t), i64(h), r(n)) == 0
        sizes.append(n.value)
    assert sizes == sorted(sizes) and L.vrs_attention_backward_workspace(i64(5), i64(0), r(n)) == 5
    ok = Heads(256, 256, 64)

    def call(q=ok, k=ok, v=ok, o=ok, tokens=100, heads=4, kv=2, d=64, dtype=1, cu=256, sequences=2, scale=0.5, lse=256,
             ws=256, need=small, back=False, dq=ok, dk=ok, dv=ok):
        h = [r(x) if x else None for x in (q, k, v)]
        rest = (i64(tokens), i64(heads), i64(kv), i64(d), dtype, ctypes.c_void_p(cu), i64(sequences), 1, ctypes.c_float(scale))
        if back:
            g = [r(x) if x else None for x in (dq, dk, dv)]
            return L.vrs_attention_backward(r(ok), *h, r(o) if o else None, ctypes.c_void_p(lse), *rest, *g,
                                            ctypes.c_void_p(ws), i64(need), None)
        return L.vrs_attention_forward(*h, *rest, r(o) if o else None, ctypes.c_void_p(lse), ctypes.c_void_p(ws), i64(need), None)

    for bad in (dict(dtype=0), dict(dtype=3), dict(d=4), dict(d=60), dict(d=136), dict(heads=3), dict(heads=0), dict(kv=0),
                dict(tokens=-1), dict(tokens=2 ** 31), dict(scale=0.0), dict(scale=math.nan), dict(scale=math.inf),
                dict(sequences=-1), dict(cu=None, sequences=0), dict(cu=None, sequences=3), dict(q=None), dict(k=None),
                dict(o=None), dict(v=Heads(None, 256, 64)), dict(q=Heads(264, 256, 64)), dict(k=Heads(256, 260, 64)),
                dict(v=Heads(256, 256, 60)), dict(o=Heads(256, 256, 56)), dict(q=Heads(256, 56, 64)), dict(lse=None),
                dict(ws=None), dict(ws=264), dict(need=small - 1)):
        assert call(**bad) == 5, bad
    for bad in (dict(dk=None), dict(dv=None), dict(dq=None, dk=None, dv=None), dict(dq=Heads(264, 256, 64)), dict(ws=None),
                dict(need=sizes[1] - 1), dict(lse=None), dict(o=None)):
        assert call(**{"back": True, "need": sizes[1], **bad}) == 5, bad
    assert call(tokens=0) == 0 and call(tokens=0, back=True) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [64, 80])
@pytest.mark.parametrize("heads,kv", [(7, 7), (12, 3)])
def test_items_after_empty_ones(gpu, heads, kv, d, causal):
    """Tiles that no sequence touches come first and last in the order of work, others
    after them on the same SMs: results do not depend on how long anything takes."""
    import torch
    from vector_cuda import ops
    lengths = [700, 450, 0, 900, 129, 1000]
    q, k, v, do = _make(lengths, heads, kv, d, "float16", behind=700)
    want = _check(q, k, v, do, lengths, causal)
    cu = _bounds(lengths)
    for _ in range(100):
        out, lse = ops.attention_forward(q, k, v, cu, causal)
        got = (out, lse, *ops.attention_backward(do, q, k, v, out, lse, cu, causal))
        assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("first,last", [(0, 300), (5, 300), (130, 131), (100, 260), (128, 256), (0, 0), (299, 300), (256, 300)])
def test_one_sequence_within_the_tokens(gpu, first, last, causal):
    """A single sequence that starts and ends anywhere: the tokens before and behind it see nothing."""
    import torch
    from vector_cuda import ops
    q, k, v, do = _make([300], 4, 2, 64, "float16")
    cu = torch.tensor([first, last], dtype=torch.int32, device="cuda")
    out, lse = ops.attention_forward(q, k, v, cu, causal)
    got = (out, *ops.attention_backward(do, q, k, v, out, lse, cu, causal))
    part = slice(first, last)
    if last > first:
        # the same as three sequences, whose bounds are looked up the other way
        three = torch.tensor([0, first, last, 300], dtype=torch.int32, device="cuda")
        o3, l3 = ops.attention_forward(q, k, v, three, causal)
        want = (o3, *ops.attention_backward(do, q, k, v, o3, l3, three, causal))
        assert torch.equal(lse[:, part], l3[:, part])
        for a, b in zip(got, want):
            assert torch.equal(a[part], b[part])
        _check(q[part].contiguous(), k[part].contiguous(), v[part].contiguous(), do[part].contiguous(), [last - first], causal)
    outside = torch.ones(300, dtype=torch.bool)
    outside[part] = False
    assert all(not t[outside].any() for t in got) and (lse[:, outside] == -math.inf).all()


@pytest.mark.gpu
def test_offsets_beyond_32_bits(gpu):
    """Tokens so far apart that their elements' numbers pass 2^32."""
    import torch
    from vector_cuda import ops
    lengths, heads, kv, d = [1500, 600], 2, 1, 64
    q, k, v, do = _make(lengths, heads, kv, d, "bfloat16")
    cu = _bounds(lengths)
    want = _check(q, k, v, do, lengths)
    far = torch.empty(2100, 1 << 21, dtype=torch.bfloat16, device="cuda")  # 8.8 GB
    x = [far[:, i * 256:i * 256 + t.shape[1] * d].view(2100, t.shape[1], d) for i, t in enumerate((q, k, v, do))]
    for a, b in zip(x, (q, k, v, do)):
        a.copy_(b)
    x[1][1700, 0, 3] = float("nan")  # (the values that are read again, too)
    k = k.clone()
    k[1700, 0, 3] = float("nan")
    out, lse = ops.attention_forward(q, k, v, cu)
    near = (out, lse, *ops.attention_backward(do, q, k, v, out, lse, cu))
    out, lse = ops.attention_forward(*x[:3], cu)
    got = (out, lse, *ops.attention_backward(x[3], *x[:3], out, lse, cu))
    for a, b in zip(near, got):
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())
    assert torch.equal(got[0][:1500], want[0][:1500])


@pytest.mark.gpu
@pytest.mark.parametrize("value", [float("nan"), float("inf"), 60000.0, -3e4])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("first,lengths,behind", [(0, [100, 60], 40), (130, [90, 200], 0), (7, [1, 0, 250], 300), (9, [150], 5)])
def test_tokens_of_no_sequence_hold_anything(gpu, first, lengths, behind, dtype, value):
    """Queries, keys, values and output gradients before the first sequence and
    behind the last: the results are those of zeros there, bit for bit."""
    import torch
    from vector_cuda import ops
    tokens = first + sum(lengths) + behind
    cu = _bounds(lengths) + first
    arrays = list(_make([tokens], 4, 2, 64, dtype))
    none = torch.ones(tokens, dtype=torch.bool, device="cuda")
    none[first:first + sum(lengths)] = False

    def run(fill):
        q, k, v, do = (torch.where(none[:, None, None], torch.full_like(t, fill), t) for t in arrays)
        out, lse = ops.attention_forward(q, k, v, cu)
        return (out, lse, *ops.attention_backward(do, q, k, v, out, lse, cu))

    for a, b in zip(run(0.0), run(value)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_calls_on_two_streams_at_once(gpu):
    """Both passes of two calls, again and again on a stream each: every turn has
    the bits of a call by itself."""
    import torch
    from vector_cuda import ops
    calls = []
    for lengths, dtype in (([300, 1, 700, 64], "float16"), ([50] * 30, "bfloat16")):
        q, k, v, do = _make(lengths, 8, 2, 128, dtype)
        calls.append((q, k, v, do, _bounds(lengths), torch.cuda.Stream()))

    def run(q, k, v, do, cu, _):
        out, lse = ops.attention_forward(q, k, v, cu)
        return (out, lse, *ops.attention_backward(do, q, k, v, out, lse, cu))

    want = [run(*c) for c in calls]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for g, c in zip(got, calls):
            with torch.cuda.stream(c[5]):
                g.append(run(*c))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for turn in g for a, b in zip(turn, w))


def test_scales_whose_exponents_have_no_float(vc):
    """scale times log2 e is a factor of the scores."""
    L, i64 = vc.lib(), ctypes.c_int64
    p = ctypes.c_void_p(256)
    for scale in (2.4e38, 3.4e38):
        assert L.vrs_attention_forward(None, None, None, i64(4), i64(1), i64(1), i64(64), 1, None, i64(1), 0,
                                       ctypes.c_float(scale), None, p, p, i64(0), None) == 5
        assert b"scale" in L.vrs_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("lengths,heads,kv", [([1500], 2, 1), ([700, 20, 900], 12, 3), ([260] * 9, 8, 8)])
def test_calls_that_follow_each_other(gpu, lengths, heads, kv, dtype):
    """Calls queued one behind the other, whose workspaces are the same memory, and
    a copy of dk behind each: the bits of calls that wait for each other."""
    import torch
    from vector_cuda import ops
    cu = _bounds(lengths)
    inputs = [_make(lengths, heads, kv, 64, dtype, seed=s) for s in range(12)]
    passes = [ops.attention_forward(q, k, v, cu) for q, k, v, _ in inputs]

    def back(i):
        q, k, v, do = inputs[i]
        dq, dk, dv = ops.attention_backward(do, q, k, v, *passes[i], cu)
        return dk.clone(), dv.clone(), dq.clone()

    want = []
    for i in range(12):
        torch.cuda.synchronize()
        want.append(back(i))
    torch.cuda.synchronize()
    got = [back(i) for i in range(12)]
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
