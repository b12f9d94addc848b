"""Matrix products in 8-bit floating point with a scale for each block of 128.

A block is 1 x 128 along the contraction (activations, gradients) or
128 x 128 (weights); its scale is a power of two, so quantising rounds each
value once, a 128 x 128 block may be read in both directions, and the tensor
cores apply the scales themselves.  `quantize_fp8` makes the operands,
`fp8_matmul` multiplies them, `fp8_linear` is a training layer of both with
its gradients, optional bias, residual and dropout.
"""
from __future__ import annotations

import functools
import struct
import threading

import torch

from . import _lib as L
from ._device import dtype_code, on_device, raw_stream, refuse_tangents
from .dropout import NO_DROP, drop_fields, with_saved_step

_CODE = {torch.float8_e4m3fn: 0, torch.float8_e5m2: 1}
_E8M0 = torch.float8_e8m0fnu

# advopt_fp8_quant_args, advopt_fp8_gemm_args (each ends in an advopt_dropout_spec)
_QUANT = struct.Struct("<QqqqQqQqQqQqQiiiiQQIIIf")
_GEMM = struct.Struct("<QqQqQqQqQqQQqqqqiiiiiiQQQIIIf")


class _ErrorWord:
    """The word that a kernel's bounded wait sets when it gives up: pinned host
    memory that the kernels write directly, so that every call can look at it
    without waiting for the GPU.  One for the process: whichever thread's call
    comes next reports it, for whichever device."""

    def __init__(self):
        self.word = self.view = None
        self.lock = threading.Lock()

    def pointer(self) -> int:
        if self.word is None:
            if torch.cuda.is_current_stream_capturing():
                return 0   # no allocation of pinned memory during a capture
            with self.lock:
                if self.word is None:
                    word = torch.zeros(1, dtype=torch.int32, pin_memory=True)
                    self.view = word.numpy()   # before the word, which other threads find without the lock
                    self.word = word
        if self.view[0]:
            self.raise_()
        return self.word.data_ptr()

    def raise_(self):
        self.view[0] = 0
        raise L.AdvOptError("an earlier fp8 product gave up waiting for its copies (bounded wait); its result is not valid")


_ERR = _ErrorWord()


def check_fp8_errors():
    """Waits for the GPU and raises if an fp8 product's bounded wait gave up (a
    guard that is not expected to fire; otherwise the process's next product
    raises, on whichever thread or device).  Products captured before the
    process's first eager one have no word to report to."""
    torch.cuda.synchronize()
    if _ERR.word is not None and _ERR.view[0]:
        _ERR.raise_()


def _round_up(n, to):
    return (n + to - 1) // to * to


def _pitch(k):
    """The codes' row pitch: whole 16 bytes, which the product needs, and whole 128-byte lines where a row has
    several, so that its loads do not straddle them (4096 x 4096 x 4097: 83 us with rows of 4112 bytes)."""
    return _round_up(k, 128 if k > 128 else 16)


def _empty_codes(rows, k, dtype, like):
    ld = _pitch(k)
    return like.new_empty((rows, k), dtype=dtype) if k == ld else like.new_empty_strided((rows, k), (ld, 1), dtype=dtype)


def _empty_scales(rows, nb, like):
    t = like.new_empty((rows, _round_up(nb, 4)), dtype=_E8M0)
    return t if nb % 4 == 0 else t.narrow(1, 0, nb)


class Fp8Blocks:
    """A matrix [rows][k] quantised along k.

    codes   [rows][k], torch.float8_e4m3fn or torch.float8_e5m2
    scales  torch.float8_e8m0fnu, [rows][ceil(k / 128)] (1 x 128 blocks) or
            [ceil(rows / 128)][ceil(k / 128)] (128 x 128 blocks)

    Element (i, j) stands for codes[i, j] * scales[i or i // 128, j // 128].
    Codes whose rows do not start at whole 16 bytes, and scales whose rows do
    not hold whole 4 bytes, are copied once into such a layout here."""

    __slots__ = ("codes", "scales", "rows", "k", "square", "ld", "lds", "codes_ptr", "scales_ptr", "code")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        code = _CODE.get(codes.dtype)
        if code is None or scales.dtype is not _E8M0:
            raise NotImplementedError("Fp8Blocks: codes are float8_e4m3fn or float8_e5m2, scales float8_e8m0fnu "
                                      f"(got {codes.dtype}, {scales.dtype})")
        if not codes.is_cuda or scales.device != codes.device:
            raise NotImplementedError("Fp8Blocks: codes and scales must live on one CUDA device (no CPU fallback)")
        shape, of_scales = codes.shape, scales.shape
        if len(shape) != 2 or len(of_scales) != 2:
            raise ValueError("Fp8Blocks: codes and scales are matrices")
        rows, k = shape
        srows, nb = of_scales
        square = srows != rows
        if nb != (k + 127) // 128 or square and srows != (rows + 127) // 128:
            nb = (k + 127) // 128
            raise ValueError(f"Fp8Blocks: codes {rows} x {k} need scales {rows} x {nb} or {(rows + 127) // 128} x {nb}, "
                             f"got {tuple(of_scales)}")
        codes_ptr, scales_ptr = codes.data_ptr(), scales.data_ptr()
        if rows and k:
            (ld, one), (lds, sone) = codes.stride(), scales.stride()
            if rows == 1:
                ld = _round_up(k, 16)
            if codes_ptr % 16 or ld % 16 or ld < k or (one != 1 and k > 1):
                own = _empty_codes(rows, k, codes.dtype, codes)
                own.view(torch.uint8).copy_(codes.view(torch.uint8))
                codes, ld, codes_ptr = own, _pitch(k), own.data_ptr()
            if srows == 1:
                lds = _round_up(nb, 4)
            if scales_ptr % 4 or lds % 4 or lds < nb or (sone != 1 and nb > 1) or (
                    nb % 4 and scales.untyped_storage().nbytes() <
                    scales.storage_offset() + (srows - 1) * lds + _round_up(nb, 4)):
                own = _empty_scales(srows, nb, scales)
                own.view(torch.uint8).copy_(scales.view(torch.uint8))
                scales, lds, scales_ptr = own, _round_up(nb, 4), own.data_ptr()
        else:
            ld, lds = _pitch(k), _round_up(nb, 4)
        self.codes, self.scales, self.rows, self.k, self.square, self.code = codes, scales, rows, k, square, code
        self.ld, self.lds, self.codes_ptr, self.scales_ptr = ld, lds, codes_ptr, scales_ptr

    @property
    def operand(self):
        return self.codes_ptr, self.ld, self.scales_ptr, self.lds

    @property
    def block(self):
        return (128, 128) if self.square else (1, 128)

    @property
    def device(self):
        return self.codes.device


def _owned(rows, k, square, dtype, like):
    """An Fp8Blocks of new tensors."""
    b = object.__new__(Fp8Blocks)
    b.codes = _empty_codes(rows, k, dtype, like)
    b.scales = _empty_scales((rows + 127) // 128 if square else rows, (k + 127) // 128, like)
    b.rows, b.k, b.square, b.code = rows, k, square, _CODE[dtype]
    b.ld, b.lds = _pitch(k), _round_up((k + 127) // 128, 4)
    b.codes_ptr, b.scales_ptr = b.codes.data_ptr(), b.scales.data_ptr()
    return b


def _quantize(x, by_row, by_col, square, code, partial=0, drop=NO_DROP):
    """Fills by_row (blocks of x), by_col (blocks of x^T), each (codes pointer, pitch, scales pointer, pitch) or
    _NONE, and partial (column sums of 128-row slabs, a pointer or 0).  x's device is the current one."""
    R, C = x.shape
    rs, cs = x.stride()
    if C > 1 and cs != 1 or R > 1 and rs < C:
        x = x.contiguous()
        rs = C
    rc = L.lib().advopt_fp8_quantize(_QUANT.pack(x.data_ptr(), rs if R > 1 else C, R, C, *by_row, *by_col, partial,
                                                 dtype_code(x.dtype), square, code, 0, *drop), raw_stream(x.device))
    if rc:
        L.check(rc, "advopt_fp8_quantize")


_NONE = _ZERO = (0, 0, 0, 0)


@functools.lru_cache(maxsize=4096)
def _layout(rows, k, square):
    """(codes' pitch, scales' offset, scales' pitch, bytes) of blocks kept in a buffer of their own."""
    ld, lds = _pitch(k), _round_up((k + 127) // 128, 4)
    size = rows * ld                          # whole 16 bytes, so the scales behind are aligned
    return ld, size, lds, _round_up(size + ((rows + 127) // 128 if square else rows) * lds, 16)


def _at(base, layout):
    return base, layout[0], base + layout[1], layout[2]


def quantize_fp8(x: torch.Tensor, block=(1, 128), dtype: torch.dtype = torch.float8_e4m3fn, layout: str = "rows"):
    """Quantises a matrix [R][C] (float32 or bfloat16, rows of any pitch).

    For each block the scale is the least power of two that brings the largest
    finite magnitude into the type's range (1 for a block of zeros, never below
    2^-127), and a code is the nearest value of the type, ties to even.
    Infinities and NaN become NaN codes and do not enter a scale.  Codes carry
    no derivative, in either mode; `fp8_linear` is the differentiable layer.

    layout  "rows": Fp8Blocks of x, quantised along its columns' index
            "cols": Fp8Blocks of x^T [C][R], quantised along the rows' index
            "both": the pair, from one pass over x
    block   (1, 128), or (128, 128): then both layouts hold the same codes"""
    if block not in ((1, 128), (128, 128)):
        raise NotImplementedError(f"quantize_fp8: blocks of (1, 128) and (128, 128) are supported, got {block}")
    if dtype not in _CODE:
        raise NotImplementedError(f"quantize_fp8: codes are float8_e4m3fn or float8_e5m2, got {dtype}")
    if layout not in ("rows", "cols", "both"):
        raise ValueError(f"quantize_fp8: layout is 'rows', 'cols' or 'both', got {layout!r}")
    if x.dim() != 2:
        raise ValueError("quantize_fp8 takes a matrix")
    if not x.is_cuda:
        raise NotImplementedError("quantize_fp8: tensors must live on a CUDA device (no CPU fallback)")
    dtype_code(x.dtype)
    (R, C), square = x.shape, block[0] == 128
    r = _owned(R, C, square, dtype, x) if layout != "cols" else None
    c = _owned(C, R, square, dtype, x) if layout != "rows" else None
    with on_device(x.device):
        _quantize(x, _NONE if r is None else r.operand, _NONE if c is None else c.operand, square, _CODE[dtype])
    return (r, c) if layout == "both" else r if layout == "rows" else c


def _product(a, b, k, a_code, b_code, a_square, b_square, out, bias=None, residual=None, drop=NO_DROP, variant=0):
    """out = epilogue(A B^T) of two operands (codes pointer, pitch, scales pointer, pitch).  out's device is the current one."""
    m, n = out.shape
    rc = L.lib().advopt_fp8_gemm(_GEMM.pack(
        *a, *b, out.data_ptr(), n, 0 if bias is None else bias.data_ptr(), 0 if residual is None else residual.data_ptr(), n,
        m, n, k, a_code, b_code, a_square, b_square, dtype_code(out.dtype), variant, _ERR.pointer(), *drop),
        raw_stream(out.device))
    if rc:
        L.check(rc, "advopt_fp8_gemm")
    return out


def _gemm(a, b, out, bias=None, residual=None, drop=NO_DROP, variant=0):
    with on_device(out.device):
        return _product(a.operand, b.operand, a.k, a.code, b.code, a.square, b.square, out, bias, residual, drop, variant)


def fp8_matmul(a: Fp8Blocks, b: Fp8Blocks, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a @ b^T [a.rows][b.rows]: products of the values that the codes and
    scales stand for, summed in the tensor cores' float32 accumulators and
    rounded once to `out_dtype` (bfloat16 or float32).  These accumulators
    truncate: a sum of up to 8192 elements is low by up to 5e-7 to 7e-7 of the
    result (Frobenius norm, K = 8192; a float32 product that rounds is off by
    1.5e-7).  Longer float32 results are float32 sums of such sums, so that the
    error does not grow with the length; longer bfloat16 ones are one such sum
    (2e-5 at 10^6 elements, where half a step of bfloat16 is 4e-3).  The operands
    may differ in code type and block shape.  Its gradients are products of the
    same kind (see `fp8_linear`)."""
    codes = a.codes
    if a.k != b.k:
        raise ValueError(f"fp8_matmul: the operands are quantised along {a.k} and {b.k} elements")
    if codes.device != b.codes.device:
        raise ValueError(f"fp8_matmul: operands on {a.device} and {b.device}")
    dtype_code(out_dtype)
    if a.k == 0:
        return torch.zeros((a.rows, b.rows), dtype=out_dtype, device=a.device)
    return _gemm(a, b, codes.new_empty((a.rows, b.rows), dtype=out_dtype))


def _kept_at(base, T, N, K, need_x, need_w, own_w):
    """The operands x^T and weight^T in the buffer kept for the gradients, and its size."""
    lx = _layout(K, T, False) if need_w else _ZERO
    lw = _layout(K, N, True) if need_x and own_w else _ZERO
    return _at(base, lx), _at(base + lx[3], lw), lx[3] + lw[3]


def _linear(x, weight, bias, residual, blocks, drop, need_x, need_w):
    """(y, the buffer of x^T's and the weight^T's blocks that the gradients need, or None).

    The blocks of one pass lie in two buffers, one that ends with it and one
    that is kept: an allocation for each, and tensor views of them, cost the
    host as much as the kernel launches."""
    T, K = x.shape
    N = weight.shape[0]
    with on_device(x.device):
        own_w = blocks is None
        lx, lw = _layout(T, K, False), _layout(N, K, True) if own_w else _ZERO
        passing = x.new_empty(lx[3] + lw[3], dtype=torch.uint8)
        xr, wr = _at(passing.data_ptr(), lx), _at(passing.data_ptr() + lx[3], lw)
        size = _kept_at(0, T, N, K, need_x, need_w, own_w)[2]
        kept = x.new_empty(size, dtype=torch.uint8) if size else None
        xc, wc, _ = _kept_at(kept.data_ptr() if size else 0, T, N, K, need_x, need_w, own_w)
        _quantize(x, xr, xc if need_w else _NONE, False, 0)
        if own_w:
            _quantize(weight, wr, wc if need_x else _NONE, True, 0)
        else:
            wr = blocks[0].operand
        y = _product(xr, wr, K, 0, 0 if own_w else blocks[0].code, False, True, x.new_empty((T, N)), bias, residual, drop)
    return y, kept


def _linear_backward(ctx, dy):
    saved = ctx.saved_tensors   # raises if the step tensor was written since the forward pass
    need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
    dx = dw = db = None
    if need_x or need_w or need_b:
        T, N = dy.shape
        K, blocks = ctx.K, ctx.blocks
        drop = with_saved_step(ctx.drop, saved[-1], dy.device) if ctx.stepped else ctx.drop
        # by offset from where the buffer is now: a hook on saved tensors may have moved it
        xc, wc, size = _kept_at(saved[0].data_ptr() if ctx.keeps else 0, T, N, K, need_x, need_w, blocks is None)
        if ctx.keeps:
            kept = saved[0]
            if kept.dtype is not torch.uint8 or kept.device != dy.device or kept.numel() != size or not kept.is_contiguous():
                raise RuntimeError(f"a hook on saved tensors gave {kept.dtype} {tuple(kept.shape)} on {kept.device} for the kept "
                                   f"blocks, {size} bytes on {dy.device} were saved")
        with on_device(dy.device):
            # g = mask * dy / q once, for every gradient that reads it
            by_row = need_x or not need_w
            lr, lc = _layout(T, N, False) if by_row else _ZERO, _layout(N, T, False) if need_w else _ZERO
            slabs = (T + 127) // 128
            passing = dy.new_empty(lr[3] + lc[3] + (4 * slabs * N if need_b else 0), dtype=torch.uint8)
            at = passing.data_ptr()
            gr, gc, partial = _at(at, lr), _at(at + lr[3], lc), at + lr[3] + lc[3]
            _quantize(dy, gr if by_row else _NONE, gc if need_w else _NONE, False, 0, partial if need_b else 0, drop)
            if need_x:
                w_code = 0
                if blocks is not None:
                    wc, w_code = blocks[1].operand, blocks[1].code
                dx = _product(gr, wc, N, 0, w_code, False, True, dy.new_empty((T, K)))
            if need_w:
                dw = _product(gc, xc, T, 0, 0, False, False, dy.new_empty((N, K), dtype=ctx.w_dtype))
            if need_b:
                db = dy.new_empty((N,))
                L.check(L.lib().advopt_col_sum(db.data_ptr(), partial, slabs, N, dtype_code(db.dtype),
                                               raw_stream(dy.device)), "advopt_col_sum")
    return dx, dw, db, (dy if need_r else None), None, None, None


_linear_backward_once = torch.autograd.function.once_differentiable(_linear_backward)


class _Fp8Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, blocks, step_tensor, drop):
        y, kept = _linear(x, weight, bias, residual, blocks, drop, *ctx.needs_input_grad[:2])
        ctx.drop, ctx.w_dtype, ctx.K, ctx.blocks, ctx.keeps = drop, weight.dtype, x.shape[1], blocks, kept is not None
        ctx.stepped = step_tensor is not None and any(ctx.needs_input_grad[:3])   # the residual's gradient needs no mask
        ctx.save_for_backward(*[t for t in (kept, step_tensor if ctx.stepped else None) if t is not None])
        return y

    @staticmethod
    def backward(ctx, dy):
        # a second derivative is refused, without the wrapper's cost where none can be asked for
        return _linear_backward_once(ctx, dy) if torch.is_grad_enabled() else _linear_backward(ctx, dy)


def fp8_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
               residual: torch.Tensor | None = None, dropout_p: float = 0.0, seed: int = 42, site: int = 0, step=0,
               weight_blocks=None) -> torch.Tensor:
    """y = residual + dropout(x @ weight^T + bias), the products in block-scaled
    e4m3 with float32 accumulation, bias, dropout and residual in the product's
    epilogue (float32, one rounding to x's dtype).

    x [..., K] and weight [N][K] are quantised in the call: x in 1 x 128
    blocks, the weight in 128 x 128 ones.  Gradients: with g = dropout's mask and
    scale applied to dy (the mask of `philox_dropout` with these `seed`,
    `site`, `step`, over y's elements; it is drawn again, never stored),
      dx = Q(g) Q(weight),  dweight = Q(g^T) Q(x^T)^T,  dbias = sum of g,
      dresidual = dy,
    where Q quantises along the contraction (g in 1 x 128 blocks of its rows
    for dx, of its columns for dweight; x in blocks of its columns).  What is
    kept for the backward pass is x's and the weight's transposed codes, one
    byte per element, not x.

    x, bias and residual share a dtype (float32 or bfloat16), the weight may
    have the other one; dweight has the weight's.  `weight_blocks` takes
    quantize_fp8(weight, (128, 128), layout="both") made before, for weights
    that do not change between calls (accumulation, evaluation).  Second and
    forward-mode derivatives are refused."""
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"fp8_linear: x [..., K] and weight [N, K], got {tuple(x.shape)} and {tuple(weight.shape)}")
    dev = x.device
    if not x.is_cuda or weight.device != dev or (bias is not None and bias.device != dev) or (
            residual is not None and residual.device != dev):
        raise NotImplementedError("fp8_linear: tensors must live on one CUDA device (no CPU fallback)")
    dtype_code(x.dtype), dtype_code(weight.dtype)
    N, K = weight.shape
    if bias is not None and (bias.shape != (N,) or bias.dtype != x.dtype):
        raise ValueError(f"fp8_linear: bias must be [{N}] in x's dtype")
    if residual is not None and (residual.shape != (*x.shape[:-1], N) or residual.dtype != x.dtype):
        raise ValueError("fp8_linear: the residual must have the result's shape and dtype")
    if N == 0 or K == 0:
        raise ValueError("fp8_linear: the weight is empty")
    drop = NO_DROP if dropout_p == 0 else drop_fields(dropout_p, seed, site, step, dev)
    if weight_blocks is not None:
        r, c = weight_blocks
        # of a single row, 1 x 128 and 128 x 128 blocks are the same
        if not ((r.square or r.rows == 1) and (c.square or c.rows == 1) and (r.rows, r.k) == (N, K) == (c.k, c.rows) and
                r.device == dev == c.device):
            raise ValueError("fp8_linear: weight_blocks is quantize_fp8(weight, (128, 128), layout='both')")
    if x.numel() == 0:   # no tokens: no products, and gradients of zeros
        y = x.new_zeros((*x.shape[:-1], N)) if residual is None else residual.clone()
        return y + 0.0 * (x.sum() + weight.sum(dtype=x.dtype) + (0.0 if bias is None else bias.sum()))
    refuse_tangents("fp8_linear", x, weight, bias, residual)
    flat = x.dim() == 2
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    if residual is not None:
        residual = (residual if flat else residual.reshape(-1, N)).contiguous()
    x2 = x if flat else x.reshape(-1, K)
    if torch.is_grad_enabled():
        y = _Fp8Linear.apply(x2, weight, bias, residual, weight_blocks, step if drop[1] else None, drop)
    else:   # no transposed codes, whatever the parameters' requires_grad
        y = _linear(x2, weight, bias, residual, weight_blocks, drop, False, False)[0]
    return y if flat else y.view(*x.shape[:-1], N)
