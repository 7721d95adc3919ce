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
from typing import Optional, Tuple

import torch

from . import _check, lib

try:
    from . import _ops
except ImportError as e:
    raise ImportError("vector_cuda._ops is missing or was built for another torch; build it with "
                      "`python vector-rs_b200/build.py` (there is no fallback)") from e


def _bind():
    L = lib()
    names = ("layer_norm_forward", "layer_norm_backward", "layer_norm_backward_workspace",
             "linear_cross_entropy_forward", "linear_cross_entropy_backward_with_loss",
             "linear_cross_entropy_workspace")
    _ops.bind(*(ctypes.cast(getattr(L, "vrs_" + n), ctypes.c_void_p).value for n in names), _check)


_bind()


def check() -> None:
    """Waits for the current device and raises CudaError where a device wait of an
    earlier call gave up, whose results are then not valid. (No correct launch
    does that. Without this the next call raises it, a program's last none.)"""
    torch.cuda.synchronize()
    _check(lib().vrs_operators_status())


# ---------------------------------------------------------------- layer norm


def layer_norm_forward(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                       eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, mean, rstd): the norm of x's last dimension, y in x's type and
    shape, mean and rstd float32 of x's leading shape."""
    return _ops.layer_norm_forward(x, weight, bias, eps)


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], mean: torch.Tensor,
                        rstd: torch.Tensor, param_dtype: Optional[torch.dtype] = None, params: bool = True):
    """(dx, dweight, dbias) from the forward pass's mean and rstd; dweight and
    dbias in weight's type (param_dtype where there is no weight), or None
    each with params false."""
    if param_dtype is not None and param_dtype not in (x.dtype, torch.float32):
        raise ValueError(f"param_dtype must be {x.dtype} or float32, got {param_dtype}")
    return _ops.layer_norm_backward(dy, x, weight, mean, rstd, param_dtype == torch.float32, params)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.bias_shape = None if bias is None else bias.shape
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        want = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        dx, dw, db = layer_norm_backward(dy, x, weight, mean, rstd, ctx.bias_dtype, want)
        return (dx, dw.view(weight.shape) if ctx.needs_input_grad[1] else None,
                db.view(ctx.bias_shape) if ctx.needs_input_grad[2] else None, None)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over x's last dimension
    (at most 32,768 elements). weight and bias hold one value a column, both in
    x's type or both in float32."""
    return _LayerNorm.apply(x, weight, bias, eps)


# ------------------------------------------------------ linear cross entropy


def linear_cross_entropy_forward(x: torch.Tensor, table: torch.Tensor, targets: torch.Tensor,
                                 scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss, lse), float32 of targets' shape: lse = log sum_v exp(scale x .
    table[v]) and loss = lse - scale x . table[target]. Rows whose target is
    not a row of the table take no part: loss 0, lse 0."""
    return _ops.linear_cross_entropy_forward(x, table, targets, scale)


def linear_cross_entropy_backward(dloss: torch.Tensor, x: torch.Tensor, table: torch.Tensor, targets: torch.Tensor,
                                  lse: torch.Tensor, scale: float = 1.0, need_dx: bool = True,
                                  need_dtable: bool = True, loss: Optional[torch.Tensor] = None):
    """(dx, dtable): gradients of sum(dloss * loss), in x's and table's type;
    None for one that is not needed. lse is the forward pass's, and so is loss:
    with it the gradient of the target's score is exact for rows whose loss is
    small; without it, it is off by up to half of lse's last place."""
    return _ops.linear_cross_entropy_backward(dloss, x, table, targets, lse, scale, need_dx, need_dtable, loss)


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, table, targets, scale, handed_out):
        loss, lse = linear_cross_entropy_forward(x, table, targets, scale)
        # Losses that the caller gets may change in place.
        ctx.save_for_backward(x, table, targets, lse, loss.clone() if handed_out else loss)
        ctx.scale = scale
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss):
        x, table, targets, lse, loss = ctx.saved_tensors
        dx, dtable = linear_cross_entropy_backward(dloss, x, table, targets, lse, ctx.scale,
                                                   ctx.needs_input_grad[0], ctx.needs_input_grad[1], loss)
        return dx, dtable, None, None, None


def linear_cross_entropy(x: torch.Tensor, table: torch.Tensor, targets: torch.Tensor, scale: float = 1.0,
                         reduction: str = "mean") -> torch.Tensor:
    """Softmax cross entropy of scale * x @ table.T against targets (int64),
    without keeping the scores. Rows whose target is not a row of the table
    (any negative number, say) take no part. reduction: "mean" over the rows
    that take part (0 where there are none), "sum" or "none"."""
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"unknown reduction {reduction!r}")
    loss = _LinearCrossEntropy.apply(x, table, targets, scale, reduction == "none")
    if reduction == "none":
        return loss
    total = loss.sum()
    if reduction == "sum":
        return total
    taken = ((targets >= 0) & (targets < table.shape[0])).sum()
    return total / taken.clamp(min=1)


__all__ = ["check", "layer_norm", "layer_norm_forward", "layer_norm_backward", "linear_cross_entropy",
           "linear_cross_entropy_forward", "linear_cross_entropy_backward"]
