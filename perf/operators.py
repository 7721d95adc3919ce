"""The cases that the framework's training and scoring operators are measured on, with their plain forms.

An embedding that an index holds comes out of an encoder whose last steps are a layer norm and the product with a
table of vectors (classes, catalogue items, passages), and which is trained by the softmax cross entropy of those
scores. Two operators, each forward alone and with its gradients:

* layer norm of rows, with the reduction of the weight's and the bias's gradient over all rows;
* linear cross entropy: loss and log-sum-exp of `scale * x @ table.T` against one target a row, without keeping the
  scores, and the gradients of the rows and of the table. Rows whose target lies outside the table take no part.

`run` computes them by elementary torch operations in 32 bits, or, where `own` is true, by `vector_cuda.ops`.
"""
import math
import os
import sys

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _norm(name, way, rows, d, dtype, params):
    return {"name": name, "op": "layer_norm", "way": way, "rows": rows, "d": d, "dtype": dtype, "params": params}


def _loss(name, way, rows, classes, d, dtype, scale, unit, ignored):
    return {"name": name, "op": "linear_cross_entropy", "way": way, "rows": rows, "classes": classes, "d": d,
            "dtype": dtype, "scale": scale, "unit": unit, "ignored": ignored}


def listed():
    return [
        # One query's vector on its way to a search: latency alone counts.
        _norm("norm one query", "forward", 1, 384, "f32", "f32"),
        # A batch of token vectors of an encoder, inference.
        _norm("norm batch forward", "forward", 8192, 1024, "bf16", "bf16"),
        # A training step's norm at an odd width (rows that no vector load divides), weights kept in 32 bits.
        _norm("norm train odd", "train", 2999, 771, "f16", "f32"),
        # The backward pass of a long batch: bandwidth, and the weights' gradient over many rows.
        _norm("norm backward large", "backward", 65536, 2048, "bf16", "bf16"),
        # Few rows, very wide (a concatenation of features): little parallelism over rows.
        _norm("norm backward few wide", "backward", 37, 20011, "f32", "f32"),
        # One query's log likelihood under a whole catalogue, as served: reading the table is all there is.
        _loss("score one", "forward", 1, 100000, 768, "bf16", 1.0, False, 0.0),
        # A few queries at a time, sizes that nothing divides.
        _loss("score few ragged", "forward", 19, 30011, 500, "f16", 1.0, False, 0.0),
        # A small contrastive step: latency of the whole chain of both passes.
        _loss("train small", "train", 128, 8192, 256, "bf16", 20.0, True, 0.0),
        # An ordinary training step over a catalogue.
        _loss("train ordinary", "train", 4096, 48000, 1024, "bf16", 1.0, False, 0.0),
        # Sizes that no tile and no aligned load divides, and rows without a target.
        _loss("train odd", "train", 1999, 30011, 501, "f16", 1.0, False, 0.4),
        # A contrastive step against every row of the benchmark's index (1,000,000 x 128, unit rows).
        _loss("train whole index", "train", 1024, 1000000, 128, "bf16", 20.0, True, 0.0),
        # The largest step: a wide encoder and a large table.
        _loss("train largest", "train", 8192, 131072, 2048, "bf16", 1.0, False, 0.1),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    if rng.random() < 0.4:
        d = _log(rng, 8, 20011)
        rows = _log(rng, 1, min(65536, (1 << 27) // d))
        dtype = rng.choice(["f32", "f16", "bf16"])
        params = rng.choice([dtype, "f32"])
        case = _norm("", rng.choice(["forward", "backward", "train"]), rows, d, dtype, params)
    else:
        d = _log(rng, 16, 2048)
        classes = _log(rng, 2, min(1000000, (1 << 28) // d))
        most = min(8192, (1 << 30) // classes, (1 << 41) // (classes * d))
        rows = _log(rng, 1, max(1, most))
        unit = rng.random() < 0.4
        case = _loss("", rng.choice(["forward", "train", "train"]), rows, classes, d, rng.choice(["f16", "bf16"]),
                     20.0 if unit else 1.0, unit, rng.choice([0.0, 0.0, 0.25, 0.7]))
    del case["name"]
    return case


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = _TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "layer_norm":
        rows, d, pt = case["rows"], case["d"], _TYPES[case["params"]]
        s = {"case": case, "eps": 1e-5}
        s["x"] = (normal(rows, d) * 1.7 + normal(rows, 1)).to(dt)  # activations with a mean of their own per row
        s["weight"] = (1.0 + 0.2 * normal(d)).to(pt)
        s["bias"] = (0.1 * normal(d)).to(pt)
        if case["way"] != "forward":
            s["dy"] = normal(rows, d).to(dt)
        if case["way"] == "backward":  # what the forward pass left behind
            x = s["x"].float()
            mean = x.mean(1)
            s["mean"] = mean
            s["rstd"] = torch.rsqrt((x - mean[:, None]).square().mean(1) + s["eps"])
        return s

    rows, classes, d = case["rows"], case["classes"], case["d"]
    targets = torch.randint(0, classes, (rows,), generator=g, device="cuda")
    if case["unit"]:  # vectors of a contrastive encoder: unit rows, a query near its passage
        table = normal(classes, d)
        table /= table.norm(dim=1, keepdim=True)
        x = table[targets] + normal(rows, d) * (1.5 / math.sqrt(d))
        x /= x.norm(dim=1, keepdim=True)
    else:  # scores of spread 1.5, the target's raised by some 4
        table = normal(classes, d) * (1.5 / math.sqrt(d))
        x = normal(rows, d) + table[targets] * (4.0 / 2.25)
    if case["ignored"]:
        drop = torch.rand(rows, generator=g, device="cuda") < case["ignored"]
        targets = torch.where(drop, torch.full_like(targets, -1), targets)
    s = {"case": case, "x": x.to(dt), "table": table.to(dt), "targets": targets}
    if case["way"] == "train":  # the gradient of the mean loss; in 16-bit floats times a loss scale, as such training does
        n = (targets >= 0).sum().clamp(min=1).float()
        s["dloss"] = ((1024.0 if dt == torch.float16 else 1.0) / n).repeat(rows)
    return s


# ------------------------------------------------------------- plain forms


def _plain_norm(s):
    case, way, dt = s["case"], s["case"]["way"], s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    out = {}
    if way == "backward":
        mean, rstd = s["mean"], s["rstd"]
        xhat = (x - mean[:, None]) * rstd[:, None]
    else:
        mean = x.sum(1) / case["d"]
        xc = x - mean[:, None]
        rstd = 1.0 / torch.sqrt((xc * xc).sum(1) / case["d"] + s["eps"])
        xhat = xc * rstd[:, None]
        out = {"y": (xhat * w + s["bias"].float()).to(dt), "mean": mean, "rstd": rstd}
    if way != "forward":
        dy = s["dy"].float()
        gy = dy * w
        a = gy.sum(1, keepdim=True) / case["d"]
        b = (gy * xhat).sum(1, keepdim=True) / case["d"]
        out["dx"] = ((gy - a - xhat * b) * rstd[:, None]).to(dt)
        out["dweight"] = (dy * xhat).sum(0).to(s["weight"].dtype)
        out["dbias"] = dy.sum(0).to(s["bias"].dtype)
    return out


def _plain_loss(s):
    case = s["case"]
    valid = (s["targets"] >= 0) & (s["targets"] < case["classes"])
    at = s["targets"].clamp(0, case["classes"] - 1)[:, None]
    x = torch.where(valid[:, None], s["x"].float(), 0.0)
    table = s["table"].float()
    z = x @ table.t()
    z *= case["scale"]
    top = z.amax(1, keepdim=True)
    zt = z.gather(1, at)
    z -= top
    p = z.exp_()
    total = p.sum(1, keepdim=True)
    lse = top + torch.log(total)
    out = {"loss": torch.where(valid, (lse - zt)[:, 0], 0.0), "lse": torch.where(valid, lse[:, 0], 0.0)}
    if case["way"] == "train":
        p /= total
        p.scatter_add_(1, at, torch.full_like(zt, -1.0))
        p *= torch.where(valid, s["dloss"] * case["scale"], 0.0)[:, None]
        out["dx"] = (p @ table).to(s["x"].dtype)
        out["dtable"] = (p.t() @ x).to(s["table"].dtype)
    return out


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


def _own_norm(s):
    ops, way, out = _vector_cuda(), s["case"]["way"], {}
    if way == "backward":
        mean, rstd = s["mean"], s["rstd"]
    else:
        y, mean, rstd = ops.layer_norm_forward(s["x"], s["weight"], s["bias"], s["eps"])
        out = {"y": y, "mean": mean, "rstd": rstd}
    if way != "forward":
        out["dx"], out["dweight"], out["dbias"] = ops.layer_norm_backward(s["dy"], s["x"], s["weight"], mean, rstd)
    return out


def _own_loss(s):
    ops, scale = _vector_cuda(), s["case"]["scale"]
    loss, lse = ops.linear_cross_entropy_forward(s["x"], s["table"], s["targets"], scale)
    out = {"loss": loss, "lse": lse}
    if s["case"]["way"] == "train":
        out["dx"], out["dtable"] = ops.linear_cross_entropy_backward(s["dloss"], s["x"], s["table"], s["targets"], lse,
                                                                     scale)
    return out


def run(state):
    if state["case"]["op"] == "layer_norm":
        return _own_norm(state) if own else _plain_norm(state)
    return _own_loss(state) if own else _plain_loss(state)


def work(case):
    """Inputs once, outputs once. Without keeping the scores a training step has four products of rows x classes x d:
    the scores for the loss, the scores again, and one for each gradient."""
    e, d, rows = _BYTES[case["dtype"]], case["d"], case["rows"]
    if case["op"] == "layer_norm":
        one, p = rows * d * e, d * _BYTES[case["params"]]
        n = {"forward": 2, "backward": 3, "train": 4}[case["way"]]
        params = {"forward": 2, "backward": 3, "train": 4}[case["way"]] * p
        return {"bytes": n * one + params + 8 * rows, "flops": {"forward": 8, "backward": 14, "train": 20}[case["way"]] * rows * d}
    train = case["way"] == "train"
    taken = rows * (1.0 - case["ignored"])
    return {"bytes": (2 if train else 1) * (rows + case["classes"]) * d * e + (20 if train else 16) * rows,
            "flops": (8 if train else 2) * taken * case["classes"] * d}


def exact(case, seed):
    """The operators by their definition in 64 bits, the gradients by automatic differentiation."""
    s = prepare(case, seed)
    if case["op"] == "layer_norm":
        x, w, b = (s[k].double().requires_grad_(True) for k in ("x", "weight", "bias"))
        out = {}
        if case["way"] == "backward":  # differentiated at the statistics that x has
            y = torch.nn.functional.layer_norm(x, (case["d"],), w, b, s["eps"])
        else:
            y = torch.nn.functional.layer_norm(x, (case["d"],), w, b, s["eps"])
            var, mean = torch.var_mean(x.detach(), 1, correction=0)
            out = {"y": y.detach(), "mean": mean, "rstd": (var + s["eps"]).rsqrt()}
        if case["way"] != "forward":
            out["dx"], out["dweight"], out["dbias"] = torch.autograd.grad(y, (x, w, b), s["dy"].double())
        return out
    x, table = s["x"].double(), s["table"].double()
    train = case["way"] == "train"
    x.requires_grad_(train)
    table.requires_grad_(train)
    z = torch.nn.functional.linear(x, table) * case["scale"]
    taken = s["targets"] >= 0
    loss = torch.nn.functional.cross_entropy(z, s["targets"], ignore_index=-1, reduction="none")
    out = {"loss": loss.detach(), "lse": torch.where(taken, torch.logsumexp(z.detach(), 1), 0.0)}
    if train:
        out["dx"], out["dtable"] = torch.autograd.grad(loss, (x, table), s["dloss"].double())
    return out
