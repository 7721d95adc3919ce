"""The encoder operators together, as a text encoder uses them: norms and rotation
of queries and keys, attention over packed sequences, layer norm, the cross entropy
against a table, the gradients' norm and clipping; and the same encoder answering one
sequence at a time.

Tolerances. Everything is float16 (half an ulp h = 2^-11) but sums, the loss and the
clipping. Between the tokens and a gradient lie 14 tensors that are rounded to float16
(q k v, their norms, out, its projection, the layer norm, the pooled rows, the score
gradients, and each of these going back), each by at most h of its elements. The maps
between them are linear or normalise; with rows of unit size, weights of
orthogonal columns and scores of spread 1 none enlarges a relative error of the whole by
more than 2, and errors of different tensors add. So a gradient as a whole is off by
at most 14 x 2 x h x 2 = 2.8 % of its size."""
import math

import pytest

HEADS, KV, D, HIDDEN, CLASSES = 4, 2, 64, 256, 300
H = 2.0 ** -11


def _weights(g):
    import torch
    def square(rows, cols):
        return torch.linalg.qr(torch.randn(max(rows, cols), min(rows, cols), generator=g, device="cuda",
                                           dtype=torch.float64))[0][:rows, :cols]
    w = {"qkv": square(HIDDEN, HIDDEN), "qkv2": square(HIDDEN, HIDDEN), "out": square(HEADS * D, HIDDEN),
         "q_weight": 1 + 0.1 * torch.randn(D, generator=g, device="cuda", dtype=torch.float64),
         "k_weight": 1 + 0.1 * torch.randn(D, generator=g, device="cuda", dtype=torch.float64),
         "norm": 1 + 0.1 * torch.randn(HIDDEN, generator=g, device="cuda", dtype=torch.float64),
         "bias": 0.1 * torch.randn(HIDDEN, generator=g, device="cuda", dtype=torch.float64),
         "table": torch.randn(CLASSES, HIDDEN, generator=g, device="cuda", dtype=torch.float64) / HIDDEN ** 0.5}
    return {n: t.half() if n not in ("norm", "bias") else t.float() for n, t in w.items()}


def _encode(w, x, positions, cu, causal):
    """Tokens -> one row a token, with the framework's operators."""
    import torch
    from vector_cuda import ops
    q = (x @ w["qkv"]).view(-1, HEADS, D)
    k, v = (x @ w["qkv2"]).view(-1, 2 * KV, D).split(KV, 1)
    q, k = ops.qk_norm_rope(q, k, positions, w["q_weight"], w["k_weight"])
    out = ops.attention(q, k, v, cu, causal, scale=1.0 / 8.0)
    return ops.layer_norm(x + out.reshape(-1, HEADS * D) @ w["out"], w["norm"], w["bias"])


def _encode_plain(w, x, positions, lengths, causal):
    """The same in 64 bits, a sequence at a time."""
    import torch
    q = (x @ w["qkv"]).view(-1, HEADS, D)
    k, v = (x @ w["qkv2"]).view(-1, 2 * KV, D).split(KV, 1)
    angle = positions.double()[:, None, None] * 10000.0 ** (-torch.arange(0, D, 2, device="cuda").double() / D)
    c, s = torch.cos(angle), torch.sin(angle)

    def turn(t, weight):
        t = t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * weight
        a, b = t[..., :D // 2], t[..., D // 2:]
        return torch.cat((a * c - b * s, b * c + a * s), -1)

    q, k = turn(q, w["q_weight"]), turn(k, w["k_weight"])
    rows, at = [], 0
    for n in lengths:
        qs, ks, vs = (t[at:at + n].transpose(0, 1) for t in (q, k, v))
        z = qs @ ks.repeat_interleave(HEADS // KV, 0).transpose(1, 2) / 8.0
        if causal:
            z = z.masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -math.inf)
        rows.append((torch.softmax(z, 2) @ vs.repeat_interleave(HEADS // KV, 0)).transpose(0, 1).reshape(n, HEADS * D))
        at += n
    return torch.nn.functional.layer_norm(x + torch.cat(rows) @ w["out"], (HIDDEN,), w["norm"], w["bias"])


def _batch(seed, lengths):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    tokens = sum(lengths)
    w = _weights(g)
    x = torch.randn(tokens, HIDDEN, generator=g, device="cuda").half()
    ends = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    positions = torch.cat([torch.arange(n) for n in lengths]).cuda()
    targets = torch.randint(0, CLASSES, (len(lengths),), generator=g, device="cuda")
    return w, x, ends, positions, targets


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
def test_training_step(gpu, causal):
    import torch
    from vector_cuda import ops
    lengths = [5, 130, 1, 64, 300, 17]
    w, x, ends, positions, targets = _batch(11, lengths)
    last = ends[1:].long() - 1
    leaves = {n: t.clone().requires_grad_(True) for n, t in w.items()}
    rows = _encode(leaves, x, positions, ends, causal)
    pooled = rows[last] if causal else torch.segment_reduce(
        rows.float(), "mean", lengths=ends.diff().long(), axis=0).half()
    scale = 1024.0  # of the loss, as 16-bit training does
    loss = ops.linear_cross_entropy(pooled, leaves["table"], targets)
    (loss * scale).backward()

    exact = {n: t.double().requires_grad_(True) for n, t in w.items()}
    rows = _encode_plain(exact, x.double(), positions, lengths, causal)
    pooled = rows[last] if causal else torch.stack([r.mean(0) for r in rows.split(lengths)])
    want = torch.nn.functional.cross_entropy(pooled @ exact["table"].t(), targets)
    want.backward()
    assert abs(loss.item() - want.item()) <= 28 * H * want.item()
    for n in w:
        got, ref = leaves[n].grad.double() / scale, exact[n].grad
        assert (got - ref).norm() <= 28 * 2 * H * ref.norm(), (n, ((got - ref).norm() / ref.norm()).item())

    # The step's end: gradients to 32 bits, unscaled and clipped.
    names = list(w)
    grads = [leaves[n].grad for n in names]
    out = [torch.empty(t.shape, device="cuda") for t in grads]
    norm = ops.clip_grad_norm(grads, 0.05, out, 1.0 / scale)
    size = math.sqrt(sum((t.double() / scale).square().sum().item() for t in grads))
    assert abs(norm.item() - size) <= 6 * 2.0 ** -24 * size and size > 0.05
    total = math.sqrt(sum(t.double().square().sum().item() for t in out))
    assert abs(total - 0.05) <= 0.05 * (1e-6 / size + 2.0 ** -20)
    ops.check()


@pytest.mark.gpu
def test_step_in_a_graph(gpu):
    """Both passes and the clipping of a step, captured and replayed on other tokens."""
    import torch
    from vector_cuda import ops
    lengths = [70, 3, 200]
    w, x, ends, positions, targets = _batch(5, lengths)
    do = torch.randn(sum(lengths), HEADS, D, device="cuda").half()

    def step():
        q = (x @ w["qkv"]).view(-1, HEADS, D)
        k, v = (x @ w["qkv2"]).view(-1, 2 * KV, D).split(KV, 1)
        rest = (positions, w["q_weight"], w["k_weight"])
        qr, kr = ops.qk_norm_rope_forward(q, k, *rest)
        out, lse = ops.attention_forward(qr, kr, v, ends)
        dq, dk, dv = ops.attention_backward(do, qr, kr, v, out, lse, ends)
        dq, dk, dqw, dkw = ops.qk_norm_rope_backward(dq, dk, q, k, *rest)
        grads = [dq, dk, dv, dqw, dkw]
        return [ops.clip_grad_norm(grads, 1.0), *grads]

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (1, 2):
        x.copy_(torch.randn(x.shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda"))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip([t.clone() for t in got], step()))
    ops.check()


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
def test_one_at_a_time(gpu, causal):
    """A query encoded alone and the same one in a batch: each within the rounding of
    its own way (three tensors of float16 between them, the rows of size 1, as above)."""
    import torch
    lengths = [12, 1, 90, 33]
    w, x, ends, positions, _ = _batch(3, lengths)
    with torch.no_grad():
        rows = _encode(w, x, positions, ends, causal)
        for b, n in enumerate(lengths):
            part = slice(int(ends[b]), int(ends[b + 1]))
            alone = _encode(w, x[part], positions[part], None, causal)
            assert (alone.double() - rows[part].double()).norm() <= 2 * 6 * 2 * H * rows[part].double().norm()
