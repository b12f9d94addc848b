"""Token embedding with scaling, and its gradient by sorted tokens."""
from __future__ import annotations

import functools
import math
import struct

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L
from ._device import ErrorWord, as_float32, dtype_code, on_device, raw_stream, refuse_tangents, rows_of, saved

# advopt_embedding_args, advopt_embedding_grad_args
_FORWARD = struct.Struct("<QQQQqqqqiifi")
_GRAD = struct.Struct("<QQQQqqqqiifi")

INDEX_ERRORS = ErrorWord("an earlier embedding or token_logprobs call met an index outside its table; that row of its result is NaN")


def check_index_errors():
    """Waits for the GPUs of earlier calls and raises if an `embedding` or `token_logprobs` call
    met an index outside its table (otherwise the process's next such call
    raises, on whichever thread or device).  Calls captured before the
    process's first eager one have no word to report to."""
    INDEX_ERRORS.check()


def index_bytes(what, t):
    if t.dtype not in (torch.int32, torch.int64):
        raise NotImplementedError(f"{what} are int32 or int64, got {t.dtype}")
    return t.element_size()


@functools.lru_cache(maxsize=1024)
def _work_bytes(tokens, width, dtype):
    return L.lib().advopt_embedding_grad_work(tokens, width, dtype)


def _gather(ids, weight, scale, dtype):
    w, ld = rows_of(weight)
    V, C = weight.shape
    y = weight.new_empty(*ids.shape, C)
    with on_device(weight.device):
        rc = L.lib().advopt_embedding(_FORWARD.pack(
            y.data_ptr(), w.data_ptr(), ids.data_ptr(), INDEX_ERRORS.pointer(weight.device), ld, ids.numel(), V, C, dtype, ids.element_size(), scale, 0),
            raw_stream(weight.device))
    if rc:
        L.check(rc, "advopt_embedding")
    return y


def _backward(ctx, dy):
    id_dtype, id_shape, V, C, scale, padding, dtype = ctx.call
    dev = dy.device
    ids = saved(ctx.saved_tensors[0], "ids", id_dtype, id_shape, dev)
    dy = dy.contiguous()
    T = ids.numel()
    dw = dy.new_empty(V, C)
    size = _work_bytes(T, C, dtype)
    work = dy.new_empty(size, dtype=torch.uint8) if size else None
    with on_device(dev):
        rc = L.lib().advopt_embedding_grad(_GRAD.pack(
            dw.data_ptr(), dy.data_ptr(), ids.data_ptr(), 0 if work is None else work.data_ptr(), T, V, C, padding, dtype, ids.element_size(), scale, 0),
            raw_stream(dev))
    if rc:
        L.check(rc, "advopt_embedding_grad")
    return dw, None


_backward_once = once_differentiable(_backward)


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, call):   # a tuple: torch looks at every argument of its own
        ids, scale, padding, dtype = call
        ctx.call = ids.dtype, ids.shape, *weight.shape, scale, padding, dtype
        ctx.save_for_backward(ids)
        return _gather(ids, weight, scale, dtype)

    @staticmethod
    def backward(ctx, dy):
        # a second derivative is refused, without the wrapper's cost where none can be asked for
        return _backward_once(ctx, dy) if torch.is_grad_enabled() else _backward(ctx, dy)


def embedding(ids: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0, padding_idx: int | None = None) -> torch.Tensor:
    """y[..., :] = scale * weight[ids[...]], in float32 and rounded once to the
    weight's dtype.

    ids: int32 or int64 of any shape; weight [V][C]: float32 or bfloat16, rows
    of any pitch, both on one CUDA device.  The gradient is dense: dweight[v] =
    scale * the sum of dy over the tokens of id v, in float32 in an order that
    the ids alone decide (results repeat bit for bit), rounded once; rows
    without a token are zeros, and so is row `padding_idx` (negative: from the
    end), which is looked up like any other.

    An id outside the table gives a row of NaN and no gradient, and the next
    `embedding` or `token_logprobs` call raises (`check_index_errors()` waits
    and raises).  Second and forward-mode derivatives are refused."""
    if weight.dim() != 2:
        raise ValueError(f"embedding: the weight is a matrix [V, C], got {tuple(weight.shape)}")
    index_bytes("embedding: ids", ids)
    if not weight.is_cuda or ids.device != weight.device:
        raise NotImplementedError("embedding: ids and weight must live on one CUDA device (no CPU fallback)")
    dtype = dtype_code(weight.dtype)
    V, C = weight.shape
    scale = float(scale)
    if not math.isfinite(as_float32(scale)):
        raise ValueError(f"embedding: the scale must be finite in float32, got {scale}")
    if max(V, C, ids.numel()) >= 1 << 31:
        raise ValueError("embedding: fewer than 2^31 ids, rows and columns")
    padding = -1
    if padding_idx is not None:
        if not -V <= padding_idx < V:
            raise ValueError(f"embedding: padding_idx {padding_idx} is outside a table of {V} rows")
        padding = int(padding_idx) % V
    refuse_tangents("embedding", weight)
    if not ids.is_contiguous():
        ids = ids.contiguous()
    if torch.is_grad_enabled() and weight.requires_grad:
        return _Embedding.apply(weight, (ids, scale, padding, dtype))
    return _gather(ids, weight, scale, dtype)
