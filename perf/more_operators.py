"""The cases that the encoder operators are measured on, with their plain forms.

A text encoder turns the tokens of a query or a passage into the vector that an index holds: its blocks norm and rotate
the queries and keys of each head and attend over the sequence, and a training step ends with the norm of all gradients
and their clipping. Three operators:

* attention over packed sequences of different lengths (or a batch of equal ones), causal or over the whole sequence,
  with heads that share keys and values; forward alone and with its gradients. Tokens behind the last sequence have no
  keys: their output and gradients are 0.
* the RMS norm of each head's query and key with the rotation to its position, forward alone and with its gradients;
* the norm over a list of gradients, and the gradients times the factor that brings it below a limit (and times the
  inverse of a loss scale), in place or into tensors of 32 bits.

`run` computes them by elementary torch operations, or, where `own` is true, by `vector_cuda.ops`.
"""
import math
import os
import sys

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _attention(name, way, sequences, shortest, longest, heads, kv_heads, d, dtype, causal, behind=0):
    return {"name": name, "op": "attention", "way": way, "sequences": sequences, "shortest": shortest,
            "longest": longest, "heads": heads, "kv_heads": kv_heads, "d": d, "dtype": dtype, "causal": causal,
            "behind": behind}


def _rope(name, way, tokens, heads, kv_heads, d, rotary, interleaved, dtype, params, far):
    return {"name": name, "op": "qk_norm_rope", "way": way, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "d": d, "rotary": rotary, "interleaved": interleaved, "dtype": dtype, "params": params, "far": far}


def _clip(name, tensors, smallest, largest, dtype, out, limit, loss_scale, packed):
    return {"name": name, "op": "clip", "tensors": tensors, "smallest": smallest, "largest": largest, "dtype": dtype,
            "out": out, "limit": limit, "loss_scale": loss_scale, "packed": packed}


def listed():
    return [
        # One query on its way to a search: a dozen tokens, latency alone counts.
        _attention("attend one query", "forward", 1, 12, 12, 12, 12, 64, "bf16", False),
        # A batch of queries as a service encodes them: many sequences far shorter than a tile.
        _attention("attend queries", "forward", 512, 3, 48, 16, 16, 64, "f16", False),
        # A training step over passages of very different lengths, with shared keys and values.
        _attention("attend passages train", "train", 48, 20, 1500, 16, 4, 128, "bf16", True),
        # Sizes that no tile divides, an odd count of heads, empty sequences, rows behind the last sequence.
        _attention("attend odd train", "train", 9, 0, 700, 7, 7, 80, "f16", False, 57),
        # One long document, as it is encoded.
        _attention("attend long", "forward", 1, 32768, 32768, 8, 2, 128, "bf16", True),
        # The largest step: a batch of long passages, every head with keys of its own.
        _attention("attend largest train", "train", 4, 8192, 8192, 16, 16, 128, "bf16", True),
        # The same one query's norms and rotation.
        _rope("rotate one query", "forward", 12, 12, 12, 64, 64, False, "bf16", "bf16", False),
        # An ordinary training step's norms and rotations.
        _rope("rotate train", "train", 32768, 16, 4, 128, 128, False, "bf16", "bf16", False),
        # Half of an odd head rotated, neighbours as pairs, far positions, 32-bit weights.
        _rope("rotate odd train", "train", 2999, 7, 7, 80, 40, True, "f16", "f32", True),
        # The gradients of a small encoder, latency of the whole call.
        _clip("clip small", 30, 384, 589824, "f32", "f32", 1.0, 1.0, False),
        # Gradients in 16 bits with a loss scale, unscaled and clipped into 32 bits for the optimiser.
        _clip("clip large", 61, 1024, 33554432, "f16", "f32", 1.0, 1024.0, False),
        # Views at odd places of one flat buffer, in place, a norm below the limit: the ordinary late step.
        _clip("norm packed", 59, 1, 16000037, "f32", "", 1e6, 1.0, True),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.random()
    if kind < 0.5:
        d = rng.choice([16, 32, 48, 64, 64, 72, 80, 96, 128, 128, 128])
        kv = rng.choice([1, 2, 3, 4, 5, 8])
        heads = kv * rng.choice([1, 1, 2, 3, 4, 6])
        causal = rng.random() < 0.6
        longest = _log(rng, 1, 8192)
        shortest = rng.choice([longest, rng.randrange(longest + 1)])
        most = max(1, min(1024, 32768 // longest, (1 << 31) // (longest * longest * heads)))
        case = _attention("", rng.choice(["forward", "train"]), _log(rng, 1, most), shortest, longest, heads, kv, d,
                          rng.choice(["f16", "bf16"]), causal, rng.choice([0, 0, 0, rng.randrange(300)]))
    elif kind < 0.75:
        d = 2 * rng.randrange(8, 65) if rng.random() < 0.4 else rng.choice([32, 64, 80, 96, 128, 256])
        rotary = d if rng.random() < 0.6 else 2 * rng.randrange(1, d // 2 + 1)
        kv = rng.choice([1, 2, 4, 7, 8])
        heads = kv * rng.choice([1, 2, 3, 4])
        dtype = rng.choice(["f32", "f16", "bf16"])
        case = _rope("", rng.choice(["forward", "train"]), _log(rng, 1, min(65536, (1 << 27) // (heads * d))), heads, kv,
                     d, rotary, rng.random() < 0.5, dtype, rng.choice([dtype, "f32"]), rng.random() < 0.3)
    else:
        tensors = _log(rng, 1, 62)
        largest = _log(rng, 1, min(1 << 25, (1 << 29) // tensors))
        dtype = rng.choice(["f32", "f16", "bf16"])
        out = rng.choice(["", "f32", dtype])
        case = _clip("", tensors, _log(rng, 1, largest), largest, dtype, out,
                     1e6 if out == "" else rng.choice([0.1, 1.0, 1e6]), 1024.0 if dtype == "f16" and out else 1.0,
                     rng.random() < 0.4)
    del case["name"]
    return case


def _lengths(case):
    """The sequences' lengths: spread between the shortest and the longest, which the first one has."""
    n, low, high = case["sequences"], case["shortest"], case["longest"]
    if low == high:
        return [high] * n
    out = [high] + [low + (high - low) * ((i * 7919 + 104729) % 1009) // 1008 for i in range(1, n)]
    if low == 0 and n > 2:
        out[n // 2] = 0
    return out


def _numels(case):
    """The tensors' sizes, spread over the logarithm between the smallest and the largest."""
    n, low, high = case["tensors"], case["smallest"], case["largest"]
    steps = [((i * 7919 + 13) % 1009) / 1008 for i in range(n)]
    out = [round(low * (high / low) ** s) for s in steps]
    out[-1] = high
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = _TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "attention":
        lengths = _lengths(case)
        tokens, heads, kv, d = sum(lengths) + case["behind"], case["heads"], case["kv_heads"], case["d"]
        tokens = max(tokens, 1)
        # Queries, keys and values lie side by side, as one projection leaves them.
        qkv = normal(tokens, heads + 2 * kv, d)
        qkv[:, :heads] *= 1.5
        qkv = qkv.to(dt)
        ends = [0]
        for n in lengths:
            ends.append(ends[-1] + n)
        s = {"case": case, "q": qkv[:, :heads], "k": qkv[:, heads:heads + kv], "v": qkv[:, heads + kv:],
             "lengths": lengths, "cu_seqlens": torch.tensor(ends, dtype=torch.int32, device="cuda")}
        if case["way"] == "train":
            s["dout"] = normal(tokens, heads, d).to(dt)
        return s

    if case["op"] == "qk_norm_rope":
        tokens, heads, kv, d, pt = case["tokens"], case["heads"], case["kv_heads"], case["d"], _TYPES[case["params"]]
        qkv = (normal(tokens, heads + 2 * kv, d) * 1.3).to(dt)
        first = torch.randint(0, 1 << 20, (1,), generator=g, device="cuda") if case["far"] else 0
        s = {"case": case, "q": qkv[:, :heads], "k": qkv[:, heads:heads + kv], "base": 10000.0, "eps": 1e-6,
             "positions": torch.arange(tokens, device="cuda") % 8192 + first,
             "q_weight": (1.0 + 0.2 * normal(d)).to(pt), "k_weight": (1.0 + 0.2 * normal(d)).to(pt)}
        if case["way"] == "train":
            s["dq_out"] = normal(tokens, heads, d).to(dt)
            s["dk_out"] = normal(tokens, kv, d).to(dt)
        return s

    numels = _numels(case)
    # Gradients of a mean loss, of a size of its own per tensor.
    size = case["loss_scale"] * 1e-2 * torch.exp(normal(len(numels)))
    if case["packed"]:
        flat = torch.empty(sum(numels), dtype=dt, device="cuda")
        grads = list(flat.split(numels))
    else:
        grads = [torch.empty(n, dtype=dt, device="cuda") for n in numels]
    for t, f in zip(grads, size):
        t.normal_(generator=g)
        t *= f.to(dt)
    s = {"case": case, "grads": grads}
    if case["out"]:
        s["out"] = [torch.empty(n, dtype=_TYPES[case["out"]], device="cuda") for n in numels]
    return s


# ------------------------------------------------------------- plain forms


def _groups(case, length):
    """Heads of keys and values to take at once, so that a sequence's scores stay below 2^30 values."""
    per = case["heads"] // case["kv_heads"]
    return max(1, min(case["kv_heads"], (1 << 30) // max(1, length * length * per)))


def _plain_attention(s):
    case = s["case"]
    q, k, v, dt = s["q"], s["k"], s["v"], s["q"].dtype
    per, scale = case["heads"] // case["kv_heads"], 1.0 / math.sqrt(case["d"])
    train = case["way"] == "train"
    out = {"out": torch.zeros_like(q, memory_format=torch.contiguous_format),
           "lse": torch.full((q.shape[1], q.shape[0]), -math.inf, device=q.device)}
    if train:
        for name, like in (("dq", q), ("dk", k), ("dv", v)):
            out[name] = torch.zeros_like(like, memory_format=torch.contiguous_format)
    at = 0
    for n in s["lengths"]:
        rows = slice(at, at + n)
        at += n
        if n == 0:
            continue
        step = _groups(case, n)
        hidden = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1) if case["causal"] else None
        for h in range(0, case["kv_heads"], step):
            kv = slice(h, min(h + step, case["kv_heads"]))
            qs = slice(kv.start * per, kv.stop * per)
            qf = q[rows, qs].float().transpose(0, 1)
            kf = k[rows, kv].float().transpose(0, 1).repeat_interleave(per, 0)
            vf = v[rows, kv].float().transpose(0, 1).repeat_interleave(per, 0)
            z = qf @ kf.transpose(1, 2)
            z *= scale
            if hidden is not None:
                z.masked_fill_(hidden, -math.inf)
            top = z.amax(2, keepdim=True)
            z -= top
            p = z.exp_()
            total = p.sum(2, keepdim=True)
            p /= total
            o = p @ vf
            out["out"][rows, qs] = o.transpose(0, 1).to(dt)
            out["lse"][qs, rows] = (top + torch.log(total))[:, :, 0]
            if train:
                do = s["dout"][rows, qs].float().transpose(0, 1)
                # The pass back starts from the output as it was handed out.
                delta = (do * out["out"][rows, qs].float().transpose(0, 1)).sum(2, keepdim=True)
                dv = p.transpose(1, 2) @ do
                ds = do @ vf.transpose(1, 2)
                ds -= delta
                ds *= p
                ds *= scale
                del p, z
                out["dq"][rows, qs] = (ds @ kf).transpose(0, 1).to(dt)
                dk = ds.transpose(1, 2) @ qf
                shared = (kv.stop - kv.start, per, n, case["d"])
                out["dk"][rows, kv] = dk.view(shared).sum(1).transpose(0, 1).to(dt)
                out["dv"][rows, kv] = dv.view(shared).sum(1).transpose(0, 1).to(dt)
    return out


def _turn(case, x, cos, sin):
    """The pairs of x's first `rotary` elements turned by their angles."""
    r = case["rotary"]
    if case["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., r:]), -1)


def _plain_rope(s):
    case, dt = s["case"], s["q"].dtype
    # Angles of far positions: in 64 bits.
    power = torch.arange(0, case["rotary"], 2, device="cuda").double() / case["rotary"]
    angle = s["positions"].double()[:, None, None] / s["base"] ** power
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    out = {}
    for name in ("q", "k"):
        x, w = s[name].float(), s[name + "_weight"].float()
        rstd = 1.0 / torch.sqrt((x * x).sum(2, keepdim=True) / case["d"] + s["eps"])
        xhat = x * rstd
        out[name] = _turn(case, xhat * w, cos, sin).to(dt)
        if case["way"] == "train":
            grad = _turn(case, s[f"d{name}_out"].float(), cos, -sin)
            out[f"d{name}_weight"] = (grad * xhat).double().sum((0, 1)).to(s[name + "_weight"].dtype)
            grad = grad * w
            out["d" + name] = ((grad - xhat * ((grad * xhat).sum(2, keepdim=True) / case["d"])) * rstd).to(dt)
    return out


def _plain_clip(s):
    case = s["case"]
    unscale = 1.0 / case["loss_scale"]
    total = torch.zeros((), dtype=torch.float64, device="cuda")
    for t in s["grads"]:
        f = t.float()
        total += (f * f).sum(dtype=torch.float64)
    norm = (torch.sqrt(total) * unscale).float()
    factor = torch.clamp(case["limit"] / (norm + 1e-6), max=1.0) * unscale
    if case["out"]:
        for t, o in zip(s["grads"], s["out"]):
            o.copy_(t.float() * factor)
        return [norm, *s["out"]]
    for t in s["grads"]:
        t.copy_(t.float() * factor)
    return [norm, *s["grads"]]


# ----------------------------------------------------- the framework's calls

_ops = None


def _vector_cuda():
    global _ops
    if _ops is None:
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vector-rs_b200", "python")
        if at not in sys.path:
            sys.path.insert(0, at)
        import vector_cuda.ops
        _ops = vector_cuda.ops
    return _ops


def _own_attention(s):
    ops, causal, cu = _vector_cuda(), s["case"]["causal"], s["cu_seqlens"]
    out, lse = ops.attention_forward(s["q"], s["k"], s["v"], cu, causal)
    r = {"out": out, "lse": lse}
    if s["case"]["way"] == "train":
        r["dq"], r["dk"], r["dv"] = ops.attention_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, cu, causal)
    return r


def _own_rope(s):
    ops, case = _vector_cuda(), s["case"]
    rest = (s["positions"], s["q_weight"], s["k_weight"], s["base"], case["rotary"], case["interleaved"], s["eps"])
    r = {}
    r["q"], r["k"] = ops.qk_norm_rope_forward(s["q"], s["k"], *rest)
    if case["way"] == "train":
        r["dq"], r["dk"], r["dq_weight"], r["dk_weight"] = ops.qk_norm_rope_backward(s["dq_out"], s["dk_out"], s["q"],
                                                                                     s["k"], *rest)
    return r


def _own_clip(s):
    ops, case = _vector_cuda(), s["case"]
    if case["out"]:
        norm = ops.clip_grad_norm(s["grads"], case["limit"], s["out"], 1.0 / case["loss_scale"])
        return [norm, *s["out"]]
    return [ops.clip_grad_norm(s["grads"], case["limit"]), *s["grads"]]


def run(state):
    op = state["case"]["op"]
    if op == "attention":
        return _own_attention(state) if own else _plain_attention(state)
    if op == "qk_norm_rope":
        return _own_rope(state) if own else _plain_rope(state)
    return _own_clip(state) if own else _plain_clip(state)


def work(case):
    """Inputs once, outputs once. Attention: two products over the pairs of a query and a key that it sees forward, five
    backward (the scores again, and four for the gradients)."""
    e = _BYTES[case["dtype"]]
    if case["op"] == "attention":
        lengths, heads, kv, d = _lengths(case), case["heads"], case["kv_heads"], case["d"]
        tokens = max(1, sum(lengths) + case["behind"])
        train = case["way"] == "train"
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lengths) * heads
        one = tokens * d * e
        moved = (heads + 2 * kv) * one + heads * one + 4 * heads * tokens
        if train:
            moved += heads * one + (heads + 2 * kv) * one
        return {"bytes": moved, "flops": (14 if train else 4) * pairs * d}
    if case["op"] == "qk_norm_rope":
        one = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["d"]
        train = case["way"] == "train"
        return {"bytes": (4 if train else 2) * one * e + 8 * case["tokens"], "flops": (26 if train else 8) * one}
    n = sum(_numels(case))
    return {"bytes": n * (e + (_BYTES[case["out"]] if case["out"] else 0)), "flops": (3 if case["out"] else 2) * n}


# ------------------------------------------------------------------- exact


def _exact_attention(case, s):
    train = case["way"] == "train"
    per = case["heads"] // case["kv_heads"]
    parts = {name: [] for name in ("out", "lse") + (("dq", "dk", "dv") if train else ())}
    begin = 0
    for n in s["lengths"] + [s["q"].shape[0] - sum(s["lengths"])]:
        inside = len(parts["out"]) < len(s["lengths"])
        part = {name: [] for name in parts}
        for h in range(case["kv_heads"]):
            for i in range(per):  # a head at a time; the gradients of shared ones add up
                at = h * per + i
                q, k, v = (s[x][begin:begin + n, y].double().requires_grad_(train)
                           for x, y in (("q", at), ("k", h), ("v", h)))
                if not inside or n == 0:
                    o, lse = torch.zeros_like(q), torch.full((n,), -math.inf, dtype=torch.float64, device="cuda")
                    grads = tuple(torch.zeros_like(x) for x in (q, k, v))
                else:
                    z = torch.einsum("id,jd->ij", q, k) / math.sqrt(case["d"])
                    if case["causal"]:
                        seen = torch.arange(n, device="cuda")
                        z = torch.where(seen[None, :] <= seen[:, None], z, -math.inf)
                    o = torch.softmax(z, 1) @ v
                    lse = torch.logsumexp(z, 1).detach()
                    del z
                    if train:
                        grads = torch.autograd.grad(o, (q, k, v), s["dout"][begin:begin + n, at].double())
                part["out"].append(o.detach())
                part["lse"].append(lse)
                if train:
                    part["dq"].append(grads[0])
                    for name, x in (("dk", grads[1]), ("dv", grads[2])):
                        if i == 0:
                            part[name].append(x)
                        else:
                            part[name][-1] = part[name][-1] + x
        for name in parts:
            parts[name].append(torch.stack(part[name], 0 if name == "lse" else 1))
        begin += n
    return {name: torch.cat(p, 1 if name == "lse" else 0) for name, p in parts.items()}


def _exact_rope(case, s):
    r, d = case["rotary"], case["d"]
    out = {}
    # The rotation as a matrix for each position: the product of the pair (a, b) as a complex number with e^(i angle).
    turns = torch.exp(-math.log(s["base"]) * torch.arange(r // 2, device="cuda", dtype=torch.float64) * 2 / r)
    phase = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["positions"].double()[:, None] * turns)
    first = torch.arange(r // 2, device="cuda") * (2 if case["interleaved"] else 1)
    second = first + (1 if case["interleaved"] else r // 2)
    for name in ("q", "k"):
        x, w = (t.double().requires_grad_(True) for t in (s[name], s[name + "_weight"]))
        u = torch.nn.functional.rms_norm(x, (d,), w, s["eps"])
        z = torch.complex(u[..., first], u[..., second]) * phase[:, None]
        y = u.index_copy(2, first, z.real).index_copy(2, second, z.imag)
        out[name] = y.detach()
        if case["way"] == "train":
            dx, dw = torch.autograd.grad(y, (x, w), s[f"d{name}_out"].double())
            out[f"d{name}_weight"], out["d" + name] = dw, dx
    return out


def _exact_clip(case, s):
    norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(t.double())) ** 2 for t in s["grads"])) / case["loss_scale"]
    factor = min(1.0, case["limit"] / (norm + 1e-6)) / case["loss_scale"]
    return [torch.tensor(norm, dtype=torch.float64, device="cuda"), *(t.double() * factor for t in s["grads"])]


def exact(case, seed):
    """The operators by their definition in 64 bits, the gradients by automatic differentiation."""
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    return _exact_rope(case, s) if case["op"] == "qk_norm_rope" else _exact_clip(case, s)
