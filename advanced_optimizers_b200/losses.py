"""Log-probabilities of tokens under logits, and losses over them: a clipped
policy loss with a KL term and a preference loss of paired log ratios."""
from __future__ import annotations

import functools
import math
import struct
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L
from ._device import dtype_code, empty_as, on_device, raw_stream, refuse_tangents, rows_of, saved
from .embeddings import INDEX_ERRORS, index_bytes

# advopt_token_logprobs_args, advopt_policy_loss_args, advopt_preference_loss_args
_LOGPROBS = struct.Struct("<QQQQQQqqqqqqiifi")
_POLICY = struct.Struct("<QQQQQQQQQQQqqqqqqqddfffiii")
_PREFERENCE = struct.Struct("<QQQQQQQqqqqqffii")


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _round_up(n, to):
    return (n + to - 1) // to * to


# ---- log-probabilities ----
def _strided(logits):
    """(logits, inner, outer pitch, inner pitch) of rows that the kernels read as they lie."""
    V = logits.shape[-1]
    if V > 1 and logits.stride(-1) != 1:
        logits = logits.contiguous()
    if logits.dim() > 3 or logits.dim() < 2:
        logits = logits.reshape(-1, V)
    if logits.dim() == 2:
        return logits, max(1, logits.shape[0]), 0, logits.stride(0)
    return logits, max(1, logits.shape[1]), logits.stride(0), logits.stride(1)


@functools.lru_cache(maxsize=1024)
def _logprobs_work(rows, vocab, dtype):
    return L.lib().advopt_token_logprobs_work(rows, vocab, dtype)


def _logprobs_args(out, stats, work, logits, tokens, temperature, ignore, dtype, err):
    x, inner, outer_pitch, pitch = _strided(logits)
    # x is returned too: a copy must outlive the launch
    return x, _LOGPROBS.pack(out, stats, x.data_ptr(), tokens.data_ptr(), err, work, inner, outer_pitch, pitch, tokens.numel(),
                             logits.shape[-1], ignore, dtype, tokens.element_size(), temperature, 0)


def _token_logprobs(logits, tokens, temperature, ignore, dtype, keep):
    """(log-probabilities, {m, 1 / s} of the rows if `keep`)"""
    R = tokens.numel()
    out = logits.new_empty(tokens.shape, dtype=torch.float32)
    stats = logits.new_empty(R, 2, dtype=torch.float32) if keep else None
    size = _logprobs_work(R, logits.shape[-1], dtype)
    work = logits.new_empty(size, dtype=torch.uint8) if size else None
    with on_device(logits.device):
        x, args = _logprobs_args(out.data_ptr(), _ptr(stats), _ptr(work), logits, tokens, temperature, ignore, dtype, INDEX_ERRORS.pointer(logits.device))
        rc = L.lib().advopt_token_logprobs(args, raw_stream(logits.device))
    if rc:
        L.check(rc, "advopt_token_logprobs")
    return out, stats


def _logprobs_backward(ctx, dlp):
    logits, tokens, stats = ctx.saved_tensors
    x_dtype, x_shape, t_dtype, temperature, ignore, dtype = ctx.call
    dev = dlp.device
    if logits.dtype is not x_dtype or logits.shape != x_shape or logits.device != dev:
        saved(logits, "logits", x_dtype, x_shape, dev)   # raises
    tokens = saved(tokens, "tokens", t_dtype, dlp.shape, dev)
    stats = saved(stats, "rows' statistics", torch.float32, (tokens.numel(), 2), dev)
    dlp = dlp.contiguous()
    dx = empty_as(logits)
    with on_device(dev):
        x, args = _logprobs_args(0, stats.data_ptr(), 0, logits, tokens, temperature, ignore, dtype, 0)
        rc = L.lib().advopt_token_logprobs_grad(dx.data_ptr(), dlp.data_ptr(), args, raw_stream(dev))
    if rc:
        L.check(rc, "advopt_token_logprobs_grad")
    return dx, None


_logprobs_backward_once = once_differentiable(_logprobs_backward)


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, call):   # a tuple: torch looks at every argument of its own
        tokens, temperature, ignore, dtype = call
        out, stats = _token_logprobs(logits, tokens, temperature, ignore, dtype, True)
        ctx.call = logits.dtype, logits.shape, tokens.dtype, temperature, ignore, dtype
        ctx.save_for_backward(logits, tokens, stats)
        return out

    @staticmethod
    def backward(ctx, dlp):
        # a second derivative is refused, without the wrapper's cost where none can be asked for
        return _logprobs_backward_once(ctx, dlp) if torch.is_grad_enabled() else _logprobs_backward(ctx, dlp)


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, temperature: float = 1.0, ignore_index: int = -100) -> torch.Tensor:
    """log softmax(logits / temperature)[..., tokens], float32, of tokens' shape:
    the input of the losses below, and with a minus sign and a mean the
    cross-entropy.

    logits [..., V] float32 or bfloat16, tokens [...] int32 or int64, on one
    CUDA device.  Logits with up to two leading dimensions are read as they lie
    where a row's elements are consecutive (so `logits[:, :-1]` is not copied;
    torch's gradient of that slice is, and shifted tokens with the last place
    ignored need neither).
    Sums are float32; infinities and NaN act as in the formula (a logit of -inf
    has probability 0).  A token `ignore_index` gives 0 and its row is neither
    read nor given a gradient.  In the backward pass rows whose incoming
    gradient is 0 get zeros and are not read either.

    Any other token outside [0, V) gives NaN (and a gradient of NaN), and the
    next `embedding` or `token_logprobs` call raises (`check_index_errors()`
    waits and raises).  Second and forward-mode derivatives are refused."""
    if logits.dim() < 1 or tokens.shape != logits.shape[:-1]:
        raise ValueError(f"token_logprobs: logits [..., V] and tokens [...], got {tuple(logits.shape)} and {tuple(tokens.shape)}")
    index_bytes("token_logprobs: tokens", tokens)
    if not logits.is_cuda or tokens.device != logits.device:
        raise NotImplementedError("token_logprobs: tensors must live on one CUDA device (no CPU fallback)")
    dtype = dtype_code(logits.dtype)
    temperature = float(temperature)
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError(f"token_logprobs: the temperature must be between 1e-30 and 1e30, got {temperature}")
    if not 0 < logits.shape[-1] < 1 << 31 or tokens.numel() >= 1 << 31:
        raise ValueError("token_logprobs: fewer than 2^31 tokens, rows of 1 to 2^31 - 1 logits")
    ignore_index = int(ignore_index)
    if not -(1 << 63) <= ignore_index < 1 << 63:
        raise ValueError(f"token_logprobs: ignore_index must fit 64 bits, got {ignore_index}")
    refuse_tangents("token_logprobs", logits)
    if not tokens.is_contiguous():
        tokens = tokens.contiguous()
    if torch.is_grad_enabled() and logits.requires_grad:
        return _TokenLogprobs.apply(logits, (tokens, temperature, ignore_index, dtype))
    return _token_logprobs(logits, tokens, temperature, ignore_index, dtype, False)[0]


# ---- losses ----
def _check_rows(what, logprobs, mask, **constants):
    """logprobs [rows, tokens] and what is compared with it: one shape, dtype and CUDA device, gradients to logprobs alone."""
    shape, dtype, dev = logprobs.shape, logprobs.dtype, logprobs.device
    if len(shape) != 2:
        raise ValueError(f"{what}: log-probabilities are [sequences, tokens], got {tuple(shape)}")
    grad = torch.is_grad_enabled()
    for name, t in constants.items():
        if t is None:
            continue
        if t.device != dev:
            break
        if t.dtype is not dtype:
            raise ValueError(f"{what}: {name} must have the log-probabilities' dtype {dtype}, got {t.dtype}")
        if name != "advantages" and t.shape != shape:
            raise ValueError(f"{what}: {name} must have the log-probabilities' shape {tuple(shape)}, got {tuple(t.shape)}")
        if grad and t.requires_grad:
            raise ValueError(f"{what}: {name} is a constant of the loss: detach it")
    else:
        if logprobs.is_cuda and (mask is None or mask.device == dev):
            dev = None
    if dev is not None:
        raise NotImplementedError(f"{what}: tensors must live on one CUDA device (no CPU fallback)")
    if mask is not None and (mask.dtype is not torch.bool or mask.shape != shape):
        raise ValueError(f"{what}: the mask is bool of the log-probabilities' shape {tuple(shape)}, got {mask.dtype} {tuple(mask.shape)}")
    refuse_tangents(what, logprobs, *constants.values())
    return dtype_code(dtype)


def _rows(t):
    return (None, 0) if t is None else rows_of(t)


def _floats(like, n):
    return like.new_empty(n) if like.dtype is torch.float32 else like.new_empty(n, dtype=torch.float32)


class PolicyLoss(NamedTuple):
    loss: torch.Tensor            # differentiable in the log-probabilities
    kl: torch.Tensor              # mean over the tokens (0 without a reference)
    clip_fraction: torch.Tensor   # share of the tokens whose ratio is clipped


@functools.lru_cache(maxsize=1024)
def _policy_layout(rows, cols, keep):
    """Floats of the kept buffer {slope [rows][cols], scale [rows], work}, where its parts begin (bytes), and its size (floats)."""
    slope = _round_up(rows * cols, 4) if keep else 0
    scale = slope + _round_up(rows, 4)
    return 4 * slope, 4 * scale, scale + L.lib().advopt_policy_loss_work(rows, cols) // 4


def _policy(logprobs, old, advantages, mask, ref, clip, kl_weight, by_rows, dtype, keep):
    """(loss, kl, clip fraction, kept buffer): one buffer, since an allocation costs the host as much as a launch."""
    R, C = logprobs.shape
    p, ld_p = rows_of(logprobs)
    old, ld_old = rows_of(old)
    ref, ld_ref = _rows(ref)
    mask, ld_mask = _rows(mask)
    advantages, ld_adv = (advantages.contiguous(), -1) if advantages.dim() == 1 else rows_of(advantages)
    loss, kl, clipped = _floats(p, ()), _floats(p, ()), _floats(p, ())
    scale, work, size = _policy_layout(R, C, keep)
    kept = _floats(p, size)
    at = kept.data_ptr()
    with on_device(p.device):
        rc = L.lib().advopt_policy_loss(_POLICY.pack(
            loss.data_ptr(), kl.data_ptr(), clipped.data_ptr(), at if keep else 0, at + scale, p.data_ptr(), old.data_ptr(), _ptr(ref),
            advantages.data_ptr(), _ptr(mask), at + work, ld_p, ld_old, ld_ref, ld_adv, ld_mask, R, C, math.log1p(clip[1]),
            math.log1p(-clip[0]) if clip[0] < 1 else -math.inf, *clip, kl_weight, by_rows, dtype, 0), raw_stream(p.device))
    if rc:
        L.check(rc, "advopt_policy_loss")
    return loss, kl, clipped, kept


def _policy_backward(ctx, dloss):
    R, C, x_dtype, dtype = ctx.call
    dev = dloss.device
    scale, _, size = _policy_layout(R, C, True)
    kept = saved(ctx.saved_tensors[0], "slopes", torch.float32, (size,), dev)
    dx = kept.new_empty(R, C) if dtype == 0 else kept.new_empty(R, C, dtype=x_dtype)
    at = kept.data_ptr()
    with on_device(dev):
        rc = L.lib().advopt_policy_loss_grad(dx.data_ptr(), dloss.data_ptr(), at, at + scale, R, C, dtype, raw_stream(dev))
    if rc:
        L.check(rc, "advopt_policy_loss_grad")
    return dx, None


_policy_backward_once = once_differentiable(_policy_backward)


class _Policy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logprobs, made):   # a tuple: torch looks at every argument of its own
        loss, kept, ctx.call = made
        ctx.save_for_backward(kept)
        return loss

    @staticmethod
    def backward(ctx, dloss):
        # a second derivative is refused, without the wrapper's cost where none can be asked for
        return _policy_backward_once(ctx, dloss) if torch.is_grad_enabled() else _policy_backward(ctx, dloss)


def policy_loss(logprobs: torch.Tensor, old_logprobs: torch.Tensor, advantages: torch.Tensor, mask: torch.Tensor | None = None, *,
                ref_logprobs: torch.Tensor | None = None, clip=(0.2, 0.2), kl_weight: float = 0.0, average: str = "tokens") -> PolicyLoss:
    """The clipped policy loss with a KL term: over the tokens with mask (None:
    all), with r = exp(logprobs - old), q = ref - logprobs,

      loss = mean of -min(r A, clamp(r, 1 - clip[0], 1 + clip[1]) A) + kl_weight (exp(q) - q - 1)

    kl_weight   0: the KL term is only reported, whatever its size
    average     "tokens": the mean over all tokens; "sequences": the mean over
                the sequences with a token of the means over their tokens.  With
                no token at all the loss is 0.
    logprobs, old_logprobs, ref_logprobs (None: no KL term)  [sequences, tokens]
    advantages  [sequences] or [sequences, tokens]
    mask        bool [sequences, tokens]; what masked places hold is not looked at

    All of one dtype (float32 or bfloat16) on one CUDA device, rows of any
    pitch.  Whether a ratio is clipped is decided in float64; the rest is
    float32, sums over sequences are float64, and the loss is float32.  The
    gradient goes to `logprobs` alone, in their dtype (old, reference and
    advantages must not require one), is 0 at masked and, but for the KL term,
    at clipped tokens, and repeats bit for bit.  Second and forward-mode
    derivatives are refused."""
    dtype = _check_rows("policy_loss", logprobs, mask, old_logprobs=old_logprobs, ref_logprobs=ref_logprobs, advantages=advantages)
    R, C = logprobs.shape
    if advantages.shape != (R,) and advantages.shape != (R, C):
        raise ValueError(f"policy_loss: advantages are [sequences] or [sequences, tokens], got {tuple(advantages.shape)}")
    clip = tuple(map(float, clip))
    kl_weight = float(kl_weight)
    if len(clip) != 2 or not 0 <= clip[0] <= 1 or not 0 <= clip[1] < 1e30:
        raise ValueError(f"policy_loss: clip is (low in [0, 1], high >= 0), got {clip}")
    if not abs(kl_weight) < 1e30:
        raise ValueError(f"policy_loss: kl_weight must be finite, got {kl_weight}")
    if kl_weight and ref_logprobs is None:
        raise ValueError("policy_loss: a KL term needs ref_logprobs")
    if average not in ("tokens", "sequences"):
        raise ValueError(f"policy_loss: average is 'tokens' or 'sequences', got {average!r}")
    keep = logprobs.requires_grad and torch.is_grad_enabled()
    loss, kl, clipped, kept = _policy(logprobs, old_logprobs, advantages, mask, ref_logprobs, clip, kl_weight,
                                      average == "sequences", dtype, keep)
    if keep:
        loss = _Policy.apply(logprobs, (loss, kept, (R, C, logprobs.dtype, dtype)))
    return PolicyLoss(loss, kl, clipped)


class PreferenceLoss(NamedTuple):
    loss: torch.Tensor              # differentiable in the log-probabilities
    chosen_rewards: torch.Tensor    # [pairs], beta times the chosen rows' log ratios
    rejected_rewards: torch.Tensor


@functools.lru_cache(maxsize=1024)
def _preference_layout(rows, cols):
    """Of the buffer {slope [rows], work}: where work begins (bytes), and its size (floats)."""
    work = _round_up(rows, 4)
    return 4 * work, work + L.lib().advopt_preference_loss_work(rows // 2, cols) // 4


def _preference(logprobs, ref, mask, beta, smoothing, average, dtype):
    """(loss, rewards, kept buffer)"""
    R, C = logprobs.shape
    p, ld_p = rows_of(logprobs)
    ref, ld_ref = _rows(ref)
    mask, ld_mask = _rows(mask)
    loss, rewards = _floats(p, ()), _floats(p, R)
    work, size = _preference_layout(R, C)
    kept = _floats(p, size)
    at = kept.data_ptr()
    with on_device(p.device):
        rc = L.lib().advopt_preference_loss(_PREFERENCE.pack(
            loss.data_ptr(), rewards.data_ptr(), at, p.data_ptr(), _ptr(ref), _ptr(mask), at + work, ld_p, ld_ref, ld_mask, R // 2, C, beta,
            smoothing, average, dtype), raw_stream(p.device))
    if rc:
        L.check(rc, "advopt_preference_loss")
    return loss, rewards, kept


def _preference_backward(ctx, dloss):
    R, C, x_dtype, dtype = ctx.call
    dev = dloss.device
    kept, *rest = ctx.saved_tensors
    kept = saved(kept, "rows' slopes", torch.float32, (_preference_layout(R, C)[1],), dev)
    mask, ld_mask = None, 0
    if rest:
        mask = rest[0]
        if mask.dtype is not torch.bool or mask.shape != (R, C) or mask.device != dev:
            saved(mask, "mask", torch.bool, (R, C), dev)   # raises
        mask, ld_mask = rows_of(mask)
    dx = kept.new_empty(R, C) if dtype == 0 else kept.new_empty(R, C, dtype=x_dtype)
    with on_device(dev):
        rc = L.lib().advopt_preference_loss_grad(dx.data_ptr(), dloss.data_ptr(), kept.data_ptr(), _ptr(mask), ld_mask, R // 2, C, dtype,
                                                 raw_stream(dev))
    if rc:
        L.check(rc, "advopt_preference_loss_grad")
    return dx, None


_preference_backward_once = once_differentiable(_preference_backward)


class _Preference(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logprobs, made):   # a tuple: torch looks at every argument of its own
        loss, kept, mask, ctx.call = made
        if mask is None:
            ctx.save_for_backward(kept)
        else:
            ctx.save_for_backward(kept, mask)
        return loss

    @staticmethod
    def backward(ctx, dloss):
        # a second derivative is refused, without the wrapper's cost where none can be asked for
        return _preference_backward_once(ctx, dloss) if torch.is_grad_enabled() else _preference_backward(ctx, dloss)


def preference_loss(logprobs: torch.Tensor, ref_logprobs: torch.Tensor | None = None, mask: torch.Tensor | None = None, *, beta: float = 0.1,
                    label_smoothing: float = 0.0, average: bool = False) -> PreferenceLoss:
    """The loss of pairs of a chosen and a rejected sequence: with s the sum of
    logprobs - ref_logprobs (None: of logprobs) over a sequence's tokens with
    mask (None: all), or their mean if `average`, and h = beta (s_chosen -
    s_rejected),

      loss = mean over the pairs of -(1 - e) log sigmoid(h) - e log sigmoid(-h),  e = label_smoothing.

    logprobs, ref_logprobs [2 pairs, tokens]: the chosen sequences first, then
    the rejected ones in the same order; mask bool of that shape: what masked
    places hold is not looked at.  A sequence without a token has s = 0.

    float32 or bfloat16 (both the same) on one CUDA device, rows of any pitch;
    a row's sum is float32 and float64, the loss and the rewards beta s are
    float32.  The gradient goes to `logprobs` alone, in their dtype, and
    repeats bit for bit.  Second and forward-mode derivatives are refused."""
    dtype = _check_rows("preference_loss", logprobs, mask, ref_logprobs=ref_logprobs)
    R, C = logprobs.shape
    if R == 0 or R % 2:
        raise ValueError(f"preference_loss: an even number of rows, the chosen and then the rejected sequences, got {R}")
    beta, label_smoothing = float(beta), float(label_smoothing)
    if not abs(beta) < 1e30:
        raise ValueError(f"preference_loss: beta must be finite, got {beta}")
    if not 0 <= label_smoothing <= 1:
        raise ValueError(f"preference_loss: label_smoothing is between 0 and 1, got {label_smoothing}")
    keep = logprobs.requires_grad and torch.is_grad_enabled()
    loss, rewards, kept = _preference(logprobs, ref_logprobs, mask, beta, label_smoothing, bool(average), dtype)
    if keep:
        loss = _Preference.apply(logprobs, (loss, kept, mask, (R, C, logprobs.dtype, dtype)))
    return PreferenceLoss(loss, rewards[: R // 2], rewards[R // 2 :])
