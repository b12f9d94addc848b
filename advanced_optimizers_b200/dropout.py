"""Dropout from the library's counter-based generator.

The mask is a pure function of (seed, site, step, element index), so it is
stored nowhere: the backward pass, the fp8 quantiser and the fp8 product's
epilogue each draw it again.  The generator is the one the optimizer steps
round stochastically with (Philox4x32-10, key = seed), on a stream of its own.
"""
from __future__ import annotations

import struct

import torch

from . import _lib as L
from ._device import dtype_code, on_device, raw_stream, refuse_tangents

# advopt_dropout_spec: seed, step_dev, site, step, threshold, scale
SPEC = struct.Struct("<QQIIIf")
NO_DROP = (0, 0, 0, 0, 0, 1.0)


def drop_fields(p, seed, site, step, device):
    """advopt_dropout_spec's fields (a tuple) after the argument checks."""
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability must be between 0 and 1, got {p}")
    if not 0 <= seed < 1 << 64:
        raise ValueError("seed must fit 64 unsigned bits")
    if not 0 <= site < 1 << 32:
        raise ValueError("site must fit 32 unsigned bits")
    step_ptr = 0
    if isinstance(step, torch.Tensor):
        if step.dtype != torch.int64 or step.numel() != 1 or step.device != device:
            raise ValueError(f"a step tensor is one int64 value on the input's device ({device})")
        step_ptr, step = step.data_ptr(), 0
    elif not 0 <= step < 1 << 32:
        raise ValueError("step must fit 32 unsigned bits")
    threshold = round(p * 65536)
    scale = 65536 / (65536 - threshold) if threshold < 65536 else 0.0
    if threshold in (0, 65536):
        step_ptr = 0   # all or nothing is kept at every step: none is read, and it may be written at any time
    return seed, step_ptr, site, step, threshold, scale


def with_saved_step(fields, step, device):
    """`fields` with the step where the unpacked saved tensor `step` holds it: a hook on saved tensors gives another
    tensor than the caller's, which may have been advanced or freed since the forward pass."""
    if step.dtype != torch.int64 or step.numel() != 1 or step.device != device:
        raise RuntimeError(f"a hook on saved tensors gave {step.dtype} {tuple(step.shape)} on {step.device} for the step, "
                           f"one int64 value on {device} was saved")
    return fields[0], step.data_ptr(), *fields[2:]


def _launch(x, residual, fields):
    y = torch.empty_like(x)
    with on_device(x.device):
        rc = L.lib().advopt_dropout(y.data_ptr(), x.data_ptr(), 0 if residual is None else residual.data_ptr(), x.numel(),
                                    dtype_code(x.dtype), SPEC.pack(*fields), raw_stream(x.device))
    if rc:
        L.check(rc, "advopt_dropout")
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, step_tensor, fields):
        ctx.fields, ctx.stepped = fields, step_tensor is not None and ctx.needs_input_grad[0]   # the residual's needs no mask
        if ctx.stepped:
            ctx.save_for_backward(step_tensor)
        return _launch(x, residual, fields)

    @staticmethod
    def backward(ctx, dy):
        dx = step = None
        fields = ctx.fields
        if ctx.stepped:
            step, = ctx.saved_tensors   # raises if the step tensor was written since the forward pass
            fields = with_saved_step(fields, step, dy.device)
        if ctx.needs_input_grad[0]:
            g = dy.contiguous()
            # the gradient's own gradient is the same mask again
            dx = (_Dropout.apply(g, None, step, fields) if torch.is_grad_enabled() and g.requires_grad
                  else _launch(g, None, fields))
        return dx, (dy if ctx.needs_input_grad[1] else None), None, None


def philox_dropout(x: torch.Tensor, p: float, *, seed: int = 42, site: int = 0, step=0,
                   residual: torch.Tensor | None = None) -> torch.Tensor:
    """y = residual + keep * x / q, in float32 and rounded once to x's dtype.

    Element k of the flattened tensor is kept iff its 16-bit value r_k of the
    generator (`advopt_noise_fill` with tensor_id = `site`, stream 4) is at
    least T = round(65536 p); q = 1 - T / 65536.  A dropped element is exactly
    0 (or the residual), whatever x holds there.  `site` tells the dropouts of
    one model apart, `step` the training steps: an int, or a one-element int64
    tensor on x's device, which is read when the kernel runs, so that each
    replay of a captured graph draws another mask.  It may be advanced only
    after the backward pass, which reads it again: a write between the two
    raises.  Hooks on saved tensors that keep a copy (`save_on_cpu`) keep the
    forward pass's value with it.  A checkpointed region runs its forward pass
    again and reads the step as it is then; pass it as an argument of
    `checkpoint`, which raises if it was written, not through a closure.

    x and residual (of x's shape and dtype): float32 or bfloat16 on one CUDA
    device; other strides than contiguous ones are copied first.  Forward-mode
    derivatives are refused."""
    if not x.is_cuda:
        raise NotImplementedError("philox_dropout: tensors must live on a CUDA device (no CPU fallback)")
    dtype_code(x.dtype)
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError("philox_dropout: the residual must have x's shape, dtype and device")
    fields = drop_fields(p, seed, site, step, x.device)
    refuse_tangents("philox_dropout", x, residual)
    x = x.contiguous()
    if residual is not None:
        residual = residual.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        return _Dropout.apply(x, residual, step if fields[1] else None, fields)
    return _launch(x, residual, fields)
