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
