"""Layer norm and its gradients."""
from __future__ import annotations

import functools
import math
import struct

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L
from ._device import as_float32, dtype_code, empty_as, on_device, raw_stream, refuse_tangents, rows_of, saved

# advopt_layer_norm_args, advopt_layer_norm_grad_args
_FORWARD = struct.Struct("<QQQQQqqqfiii")
_GRAD = struct.Struct("<QQQQQQQQqqqqii")


@functools.lru_cache(maxsize=1024)
def _work_bytes(rows, cols):
    return L.lib().advopt_layer_norm_grad_work(rows, cols)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _forward(x, weight, bias, eps, keep):
    """(y, {mean, rstd} of the rows if `keep`) of a matrix x."""
    R, C = x.shape
    x, ld = rows_of(x)
    y = empty_as(x)
    stats = x.new_empty(R, 2, dtype=torch.float32) if keep else None
    affine = weight if weight is not None else bias
    with on_device(x.device):
        rc = L.lib().advopt_layer_norm(_FORWARD.pack(
            y.data_ptr(), x.data_ptr(), _ptr(weight), _ptr(bias), _ptr(stats), ld, R, C, eps, dtype_code(x.dtype),
            0 if affine is None else dtype_code(affine.dtype), 0), raw_stream(x.device))
    if rc:
        L.check(rc, "advopt_layer_norm")
    return y, stats


def _backward(ctx, dy):
    x, stats, *rest = ctx.saved_tensors
    need_x, need_w, need_b = ctx.needs_input_grad[:3]
    dev, w_dtype = dy.device, ctx.w_dtype
    R, C = dy.shape
    if x.dtype is not dy.dtype or x.shape != dy.shape or x.device != dev:
        saved(x, "input", dy.dtype, dy.shape, dev)   # raises
    x, ldx = rows_of(x)
    dy, lddy = rows_of(dy)
    stats = saved(stats, "rows' statistics", torch.float32, (R, 2), dev)
    weight = saved(rest[0], "weight", w_dtype, (C,), dev) if rest else None
    dx = empty_as(dy) if need_x else None
    dw = dy.new_empty(C, dtype=w_dtype) if need_w else None
    db = dy.new_empty(C, dtype=w_dtype) if need_b else None
    work = dy.new_empty(_work_bytes(R, C), dtype=torch.uint8) if need_w or need_b else None
    with on_device(dev):
        rc = L.lib().advopt_layer_norm_grad(_GRAD.pack(
            _ptr(dx), _ptr(dw), _ptr(db), dy.data_ptr(), x.data_ptr(), _ptr(weight), stats.data_ptr(), _ptr(work), lddy, ldx, R, C,
            dtype_code(dy.dtype), dtype_code(w_dtype)), raw_stream(dev))
    if rc:
        L.check(rc, "advopt_layer_norm_grad")
    return dx, dw, db, None


_backward_once = once_differentiable(_backward)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _forward(x, weight, bias, eps, True)
        affine = weight if weight is not None else bias
        ctx.w_dtype = x.dtype if affine is None else affine.dtype
        ctx.save_for_backward(x, stats, *([] if weight is None else [weight]))
        return y

    @staticmethod
    def backward(ctx, dy):
        # a second derivative is refused, without the wrapper's cost where none can be asked for
        return _backward_once(ctx, dy) if torch.is_grad_enabled() else _backward(ctx, dy)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """y = (x - mean) / sqrt(var + eps) * weight + bias over the last dimension,
    in float32 and rounded once to x's dtype; var is the mean square of the
    differences from the mean, found from them.

    x [..., C]; weight and bias [C], either of them optional, of one dtype,
    which may be another one than x's (float32 or bfloat16 each), on one CUDA
    device.  Rows of a matrix may have any pitch; other strides are copied
    first.  Gradients of all three, in the dtype of each; those of weight and
    bias are summed over the rows in float32 in a fixed order (they repeat bit
    for bit) and rounded once.  x, two floats a row and the weight are kept.
    Second and forward-mode derivatives are refused."""
    if x.dim() < 1:
        raise ValueError("layer_norm: x has at least one dimension")
    C = x.shape[-1]
    dev = x.device
    if not x.is_cuda or (weight is not None and weight.device != dev) or (bias is not None and bias.device != dev):
        raise NotImplementedError("layer_norm: tensors must live on one CUDA device (no CPU fallback)")
    dtype_code(x.dtype)
    for t in (weight, bias):
        if t is not None:
            dtype_code(t.dtype)
            if t.dim() != 1 or t.shape[0] != C:
                raise ValueError(f"layer_norm: weight and bias are [{C}], got {tuple(t.shape)}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"layer_norm: weight and bias share a dtype, got {weight.dtype} and {bias.dtype}")
    eps = float(eps)
    eps32 = as_float32(eps)
    if not (eps >= 0 and math.isfinite(eps32) and (eps32 > 0 or eps == 0)):
        raise ValueError(f"layer_norm: eps must be 0 or a positive number of float32, got {eps}")
    if C == 0 or C >= 1 << 31:
        raise ValueError(f"layer_norm: rows of 1 to 2^31 - 1 elements, got {C}")
    refuse_tangents("layer_norm", x, weight, bias)
    if weight is not None and not weight.is_contiguous():
        weight = weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    flat = x.dim() == 2
    x2 = x if flat else x.reshape(-1, C)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or (
            bias is not None and bias.requires_grad)):
        y = _LayerNorm.apply(x2, weight, bias, eps)
    else:
        y = _forward(x2, weight, bias, eps, False)[0]
    return y if flat else y.view(x.shape)
