"""vector_cuda.ops -- training operators over libvrs, on torch CUDA tensors.

What produces and trains the vectors that an index holds: the layer norm at
an encoder's end, and the softmax cross entropy of a row's scores against
every row of a table of vectors (the inner products that a dot-product search
ranks), without keeping the scores. Neither has a counterpart in the
reference, whose vectors come from outside.

``layer_norm`` and ``linear_cross_entropy`` take part in autograd; the
``*_forward`` and ``*_backward`` functions are the passes by themselves.
Every call queues its work on torch's current stream of the tensors' device
and returns without waiting. There is no CPU fallback.
"""
from __future__ import annotations

import ctypes
import functools
from typing import Optional, Tuple

import torch

from . import _check, lib

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # vrs_dtype


def _rows(t: torch.Tensor, name: str, d: Optional[int] = None) -> Tuple[torch.Tensor, int, int]:
    """t as rows of its last dimension: (tensor, rows, row stride). Rows that
    are contiguous and evenly spaced are used where they are."""
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (there is no CPU fallback)")
    if t.dim() < 1 or t.dtype not in _DTYPES:
        raise ValueError(f"{name} must have rows of float32, float16 or bfloat16, got {t.dtype}")
    have = t.shape[-1]
    if d is not None and have != d:
        raise ValueError(f"{name} has rows of {have} elements, expected {d}")
    if have < 1:
        raise ValueError(f"{name} has rows of no elements")
    if t.dim() != 2:
        t = t.reshape(-1, have)
    n = t.shape[0]
    stride, one = t.stride()
    if (have > 1 and one != 1) or (n > 1 and stride < have):
        t = t.contiguous()
        stride = have
    return t, n, stride if stride > have else have


def _same(t: torch.Tensor, like: torch.Tensor, name: str, n: int, dtype: torch.dtype) -> torch.Tensor:
    """A tensor of n values beside `like`, contiguous."""
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.numel() != n:
        raise ValueError(f"{name} holds {t.numel()} values, expected {n}")
    if t.get_device() != like.get_device():
        raise ValueError(f"{name} is on {t.device}, expected {like.device}")
    return t if t.is_contiguous() else t.contiguous()


def _params(weight, bias, x, d: int):
    """The parameters' type (the rows', or float32) and the checked tensors."""
    pt = x.dtype
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None:
            if p.dtype != x.dtype and p.dtype != torch.float32:
                raise ValueError(f"{name} must be {x.dtype} or float32, got {p.dtype}")
            pt = p.dtype
    if weight is not None:
        weight = _same(weight, x, "weight", d, pt)
    if bias is not None:
        bias = _same(bias, x, "bias", d, pt)
    return weight, bias, pt


def _like(t: torch.Tensor, rows: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of t's shape and type (rows: t seen as rows)."""
    return torch.empty_like(t) if t is rows and t.is_contiguous() else t.new_empty(t.shape)


def _column(t: torch.Tensor, n: int) -> torch.Tensor:
    """An f32 value for each of t's n rows."""
    v = torch.empty(n, dtype=torch.float32, device=t.device)
    return v if t.dim() == 2 else v.view(t.shape[:-1])


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _call(f, device: int, *args):
    """f(*args, stream) on the device's current stream, with the device current."""
    stream = torch.cuda.current_stream(device).cuda_stream
    if device == torch.cuda.current_device():
        status = f(*args, stream)
    else:
        with torch.cuda.device(device):
            status = f(*args, stream)
    if status:
        _check(status)


@functools.lru_cache(maxsize=1024)
def _norm_workspace(device: int, rows: int, d: int) -> int:
    n = ctypes.c_int64(0)
    with torch.cuda.device(device):
        _check(lib().vrs_layer_norm_backward_workspace(rows, d, ctypes.byref(n)))
    return n.value


@functools.lru_cache(maxsize=1024)
def _loss_workspace(rows: int, classes: int, d: int, dtype: int, backward: bool, aligned: bool) -> int:
    n = ctypes.c_int64(0)
    _check(lib().vrs_linear_cross_entropy_workspace(rows, classes, d, dtype, int(backward), int(aligned),
                                                    ctypes.byref(n)))
    return n.value


# ---------------------------------------------------------------- layer norm


def layer_norm_forward(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                       eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, mean, rstd): the norm of x's last dimension, y in x's type and
    shape, mean and rstd float32 of x's leading shape."""
    xr, n, xs = _rows(x, "x")
    d = xr.shape[1]
    weight, bias, pt = _params(weight, bias, xr, d)
    y = _like(x, xr)
    mean = _column(x, n)
    rstd = torch.empty_like(mean)
    _call(lib().vrs_layer_norm_forward, xr.get_device(), xr.data_ptr(), xs, n, d, _DTYPES[xr.dtype], _p(weight),
          _p(bias), _DTYPES[pt], eps, y.data_ptr(), d, mean.data_ptr(), rstd.data_ptr())
    return y, mean, rstd


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], mean: torch.Tensor,
                        rstd: torch.Tensor, param_dtype: Optional[torch.dtype] = None, params: bool = True):
    """(dx, dweight, dbias) from the forward pass's mean and rstd; dweight and
    dbias in weight's type (param_dtype where there is no weight), or None
    each with params false."""
    xr, n, xs = _rows(x, "x")
    d = xr.shape[1]
    if dy.shape != x.shape or dy.dtype != xr.dtype or dy.get_device() != xr.get_device():
        raise ValueError(f"dy must be like x ({tuple(x.shape)}, {xr.dtype}), got {tuple(dy.shape)}, {dy.dtype}")
    yr, _, ys = _rows(dy, "dy", d)
    weight, _, pt = _params(weight, None, xr, d)
    if weight is None and param_dtype is not None:
        pt = param_dtype
        if pt not in (xr.dtype, torch.float32):
            raise ValueError(f"param_dtype must be {xr.dtype} or float32, got {pt}")
    mean = _same(mean, xr, "mean", n, torch.float32)
    rstd = _same(rstd, xr, "rstd", n, torch.float32)
    device = xr.get_device()
    dx = _like(x, xr)
    dw = db = ws = None
    need = 0
    if params:
        dw = torch.empty(d, dtype=pt, device=xr.device)
        db = torch.empty_like(dw)
        need = _norm_workspace(device, n, d)
        ws = torch.empty(need, dtype=torch.uint8, device=xr.device)
    _call(lib().vrs_layer_norm_backward, device, yr.data_ptr(), ys, xr.data_ptr(), xs, n, d, _DTYPES[xr.dtype],
          _p(weight), _DTYPES[pt], mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), d, _p(dw), _p(db), _p(ws), need)
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        want = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        dx, dw, db = layer_norm_backward(dy, x, weight, mean, rstd, ctx.bias_dtype, want)
        return dx, dw if ctx.needs_input_grad[1] else None, db if ctx.needs_input_grad[2] else None, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over x's last dimension
    (at most 32,768 elements). weight and bias are in x's type or float32."""
    return _LayerNorm.apply(x, weight, bias, eps)


# ------------------------------------------------------ linear cross entropy


def _loss_args(x, table, targets, scale):
    xr, n, xs = _rows(x, "x")
    if table.dim() != 2:
        raise ValueError(f"table must be classes x d, got {tuple(table.shape)}")
    d = xr.shape[1]
    tr, classes, ts = _rows(table, "table", d)
    if tr.dtype != xr.dtype or tr.get_device() != xr.get_device():
        raise ValueError(f"table must be {xr.dtype} on {xr.device}, got {tr.dtype} on {tr.device}")
    if xr.dtype == torch.float32:
        raise ValueError("x and table must be float16 or bfloat16 (operands of the tensor cores)")
    if classes < 1:
        raise ValueError("table has no rows")
    if targets.shape != x.shape[:-1]:
        raise ValueError(f"targets have shape {tuple(targets.shape)}, expected {tuple(x.shape[:-1])}")
    targets = _same(targets, xr, "targets", n, torch.int64)
    if not 0.0 < scale < float("inf"):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    return xr, n, xs, tr, classes, ts, d, targets


def _aligned(t: torch.Tensor, stride: int) -> bool:
    return t.data_ptr() % 16 == 0 and stride % 8 == 0


def linear_cross_entropy_forward(x: torch.Tensor, table: torch.Tensor, targets: torch.Tensor,
                                 scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss, lse), float32 of targets' shape: lse = log sum_v exp(scale x .
    table[v]) and loss = lse - scale x . table[target]. Rows whose target is
    not a row of the table take no part: loss 0, lse 0."""
    xr, n, xs, tr, classes, ts, d, tg = _loss_args(x, table, targets, scale)
    dt = _DTYPES[xr.dtype]
    loss = _column(x, n)
    lse = torch.empty_like(loss)
    need = _loss_workspace(n, classes, d, dt, False, _aligned(tr, ts))
    ws = torch.empty(need, dtype=torch.uint8, device=xr.device)
    _call(lib().vrs_linear_cross_entropy_forward, xr.get_device(), xr.data_ptr(), xs, n, tr.data_ptr(), ts, classes, d,
          dt, tg.data_ptr(), scale, loss.data_ptr(), lse.data_ptr(), ws.data_ptr(), need)
    return loss, lse


def linear_cross_entropy_backward(dloss: torch.Tensor, x: torch.Tensor, table: torch.Tensor, targets: torch.Tensor,
                                  lse: torch.Tensor, scale: float = 1.0, need_dx: bool = True,
                                  need_dtable: bool = True):
    """(dx, dtable): gradients of sum(dloss * loss), in x's and table's type;
    None for one that is not needed. lse is the forward pass's."""
    xr, n, xs, tr, classes, ts, d, tg = _loss_args(x, table, targets, scale)
    dt = _DTYPES[xr.dtype]
    dloss = _same(dloss, xr, "dloss", n, torch.float32)
    lse = _same(lse, xr, "lse", n, torch.float32)
    dx = _like(x, xr) if need_dx else None
    dtable = _like(table, tr) if need_dtable else None
    need = _loss_workspace(n, classes, d, dt, True, _aligned(tr, ts))
    ws = torch.empty(need, dtype=torch.uint8, device=xr.device)
    _call(lib().vrs_linear_cross_entropy_backward, xr.get_device(), dloss.data_ptr(), xr.data_ptr(), xs, n,
          tr.data_ptr(), ts, classes, d, dt, tg.data_ptr(), scale, lse.data_ptr(), _p(dx), d, _p(dtable), d,
          ws.data_ptr(), need)
    return dx, dtable


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, table, targets, scale):
        loss, lse = linear_cross_entropy_forward(x, table, targets, scale)
        ctx.save_for_backward(x, table, targets, lse)
        ctx.scale = scale
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        x, table, targets, lse = ctx.saved_tensors
        dx, dtable = linear_cross_entropy_backward(dloss, x, table, targets, lse, ctx.scale,
                                                   ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        return dx, dtable, None, None


def linear_cross_entropy(x: torch.Tensor, table: torch.Tensor, targets: torch.Tensor, scale: float = 1.0,
                         reduction: str = "mean") -> torch.Tensor:
    """Softmax cross entropy of scale * x @ table.T against targets (int64),
    without keeping the scores. Rows whose target is not a row of the table
    (any negative number, say) take no part. reduction: "mean" over the rows
    that take part (0 where there are none), "sum" or "none"."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"unknown reduction {reduction!r}")
    loss = _LinearCrossEntropy.apply(x, table, targets, scale)
    if reduction == "none":
        return loss
    total = loss.sum()
    if reduction == "sum":
        return total
    taken = ((targets >= 0) & (targets < table.shape[0])).sum()
    return total / taken.clamp(min=1)


__all__ = ["layer_norm", "layer_norm_forward", "layer_norm_backward", "linear_cross_entropy",
           "linear_cross_entropy_forward", "linear_cross_entropy_backward"]
