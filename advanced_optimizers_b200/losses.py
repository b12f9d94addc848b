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
from ._device import dtype_code, on_device, raw_stream, refuse_tangents, rows_of, saved
from .embeddings import INDEX_ERRORS, index_bytes

# advopt_token_logprobs_args, advopt_policy_loss_args, advopt_preference_loss_args
_LOGPROBS = struct.Struct("<QQQQQqqqqqqiifi")
_POLICY = struct.Struct("<QQQQQQQQQQqqqqqqqddfffiii")
_PREFERENCE = struct.Struct("<QQQQQQQqqqqqffii")


def _ptr(t):
    return 0 if t is None else t.data_ptr()


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


def _logprobs_args(out, stats, logits, tokens, temperature, ignore, err):
    x, inner, outer_pitch, pitch = _strided(logits)
    # x is returned too: a copy must outlive the launch
    return x, _LOGPROBS.pack(_ptr(out), _ptr(stats), x.data_ptr(), tokens.data_ptr(), err, inner, outer_pitch, pitch, tokens.numel(),
                             logits.shape[-1], ignore, dtype_code(logits.dtype), tokens.element_size(), temperature, 0)


def _token_logprobs(logits, tokens, temperature, ignore, keep):
    out = logits.new_empty(tokens.shape, dtype=torch.float32)
    stats = logits.new_empty((tokens.numel(), 2), dtype=torch.float32) if keep else None
    with on_device(logits.device):
        x, args = _logprobs_args(out, stats, logits, tokens, temperature, ignore, INDEX_ERRORS.pointer())
        rc = L.lib().advopt_token_logprobs(args, raw_stream(logits.device))
    if rc:
        L.check(rc, "advopt_token_logprobs")
    return out, stats


def _logprobs_backward(ctx, dlp):
    logits, tokens, stats = ctx.saved_tensors
    if logits.dtype is not ctx.x_dtype or logits.shape != ctx.x_shape or logits.device != dlp.device:
        saved(logits, "logits", ctx.x_dtype, ctx.x_shape, dlp.device)   # raises
    tokens = saved(tokens, "tokens", ctx.t_dtype, dlp.shape, dlp.device)
    stats = saved(stats, "rows' statistics", torch.float32, (tokens.numel(), 2), dlp.device)
    dlp = dlp.contiguous()
    dx = torch.empty(ctx.x_shape, dtype=ctx.x_dtype, device=dlp.device)
    with on_device(dlp.device):
        x, args = _logprobs_args(None, stats, logits, tokens, ctx.temperature, ctx.ignore, 0)
        rc = L.lib().advopt_token_logprobs_grad(dx.data_ptr(), dlp.data_ptr(), args, raw_stream(dlp.device))
    if rc:
        L.check(rc, "advopt_token_logprobs_grad")
    return dx, None, None, None


_logprobs_backward_once = once_differentiable(_logprobs_backward)


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, temperature, ignore):
        out, stats = _token_logprobs(logits, tokens, temperature, ignore, True)
        ctx.x_dtype, ctx.x_shape, ctx.t_dtype, ctx.temperature, ctx.ignore = logits.dtype, logits.shape, tokens.dtype, temperature, ignore
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
    where a row's elements are consecutive (so `logits[:, :-1]` is not copied).
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
    dtype_code(logits.dtype)
    temperature = float(temperature)
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError(f"token_logprobs: the temperature must be between 1e-30 and 1e30, got {temperature}")
    if not 0 < logits.shape[-1] < 1 << 31:
        raise ValueError("token_logprobs: rows of 1 to 2^31 - 1 logits")
    refuse_tangents("token_logprobs", logits)
    if not tokens.is_contiguous():
        tokens = tokens.contiguous()
    if torch.is_grad_enabled() and logits.requires_grad:
        return _TokenLogprobs.apply(logits, tokens, temperature, int(ignore_index))
    return _token_logprobs(logits, tokens, temperature, int(ignore_index), False)[0]


# ---- losses ----
def _check_rows(what, logprobs, constants, mask):
    """logprobs [rows, tokens] and what is compared with it: one shape, dtype and CUDA device, gradients to logprobs alone."""
    if logprobs.dim() != 2:
        raise ValueError(f"{what}: log-probabilities are [sequences, tokens], got {tuple(logprobs.shape)}")
    if not logprobs.is_cuda or any(t is not None and t.device != logprobs.device for t in (*constants.values(), mask)):
        raise NotImplementedError(f"{what}: tensors must live on one CUDA device (no CPU fallback)")
    dtype_code(logprobs.dtype)
    for name, t in constants.items():
        if t is None:
            continue
        if t.dtype != logprobs.dtype:
            raise ValueError(f"{what}: {name} must have the log-probabilities' dtype {logprobs.dtype}, got {t.dtype}")
        if t.shape != logprobs.shape and name != "advantages":
            raise ValueError(f"{what}: {name} must have the log-probabilities' shape {tuple(logprobs.shape)}, got {tuple(t.shape)}")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{what}: {name} is a constant of the loss: detach it")
    if mask is not None and (mask.dtype != torch.bool or mask.shape != logprobs.shape):
        raise ValueError(f"{what}: the mask is bool of the log-probabilities' shape {tuple(logprobs.shape)}, got {mask.dtype} {tuple(mask.shape)}")
    refuse_tangents(what, logprobs, *constants.values())


def _rows(t):
    return (None, 0) if t is None else rows_of(t)


class PolicyLoss(NamedTuple):
    loss: torch.Tensor            # differentiable in the log-probabilities
    kl: torch.Tensor              # mean over the tokens (0 without a reference)
    clip_fraction: torch.Tensor   # share of the tokens whose ratio is clipped


@functools.lru_cache(maxsize=1024)
def _policy_work(rows, cols):
    return L.lib().advopt_policy_loss_work(rows, cols)


def _policy(logprobs, old, advantages, mask, ref, clip, kl_weight, by_rows, keep):
    R, C = logprobs.shape
    p, ld_p = rows_of(logprobs)
    old, ld_old = rows_of(old)
    ref, ld_ref = _rows(ref)
    mask, ld_mask = _rows(mask)
    advantages, ld_adv = (advantages.contiguous(), -1) if advantages.dim() == 1 else rows_of(advantages)
    new = lambda *shape, dtype=torch.float32: p.new_empty(shape, dtype=dtype)  # noqa: E731
    loss, stats, scale = new(), new(2), new(R)
    slope = new(R, C) if keep else None
    work = new(_policy_work(R, C), dtype=torch.uint8)
    with on_device(p.device):
        rc = L.lib().advopt_policy_loss(_POLICY.pack(
            loss.data_ptr(), stats.data_ptr(), _ptr(slope), scale.data_ptr(), p.data_ptr(), old.data_ptr(), _ptr(ref), advantages.data_ptr(),
            _ptr(mask), work.data_ptr(), ld_p, ld_old, ld_ref, ld_adv, ld_mask, R, C, math.log1p(clip[1]),
            math.log1p(-clip[0]) if clip[0] < 1 else -math.inf, *clip, kl_weight, by_rows, dtype_code(p.dtype), 0), raw_stream(p.device))
    if rc:
        L.check(rc, "advopt_policy_loss")
    return loss, stats, slope, scale


def _policy_backward(ctx, dloss, _):
    slope, scale = ctx.saved_tensors
    (R, C), dev = ctx.x_shape, dloss.device
    slope, scale = saved(slope, "slopes", torch.float32, (R, C), dev), saved(scale, "rows' weights", torch.float32, (R,), dev)
    dx = torch.empty((R, C), dtype=ctx.x_dtype, device=dev)
    with on_device(dev):
        rc = L.lib().advopt_policy_loss_grad(dx.data_ptr(), dloss.data_ptr(), slope.data_ptr(), scale.data_ptr(), R, C,
                                             dtype_code(ctx.x_dtype), raw_stream(dev))
    if rc:
        L.check(rc, "advopt_policy_loss_grad")
    return dx, *[None] * 7


_policy_backward_once = once_differentiable(_policy_backward)


class _Policy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logprobs, old, advantages, mask, ref, clip, kl_weight, by_rows):
        loss, stats, slope, scale = _policy(logprobs, old, advantages, mask, ref, clip, kl_weight, by_rows, True)
        ctx.x_shape, ctx.x_dtype = logprobs.shape, logprobs.dtype
        ctx.save_for_backward(slope, scale)
        ctx.mark_non_differentiable(stats)
        ctx.set_materialize_grads(False)
        return loss, stats

    @staticmethod
    def backward(ctx, dloss, dstats):
        # a second derivative is refused, without the wrapper's cost where none can be asked for
        return _policy_backward_once(ctx, dloss, dstats) if torch.is_grad_enabled() else _policy_backward(ctx, dloss, dstats)


def policy_loss(logprobs: torch.Tensor, old_logprobs: torch.Tensor, advantages: torch.Tensor, mask: torch.Tensor | None = None, *,
                ref_logprobs: torch.Tensor | None = None, clip=(0.2, 0.2), kl_weight: float = 0.0, average: str = "tokens") -> PolicyLoss:
    """The clipped policy loss with a KL term: over the tokens with mask (None:
    all), with r = exp(logprobs - old), q = ref - logprobs,

      loss = mean of -min(r A, clamp(r, 1 - clip[0], 1 + clip[1]) A) + kl_weight (exp(q) - q - 1)

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
    _check_rows("policy_loss", logprobs, dict(old_logprobs=old_logprobs, ref_logprobs=ref_logprobs, advantages=advantages), mask)
    if advantages.shape != logprobs.shape and advantages.shape != logprobs.shape[:1]:
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
    args = logprobs, old_logprobs, advantages, mask, ref_logprobs, clip, kl_weight, average == "sequences"
    if torch.is_grad_enabled() and logprobs.requires_grad:
        loss, stats = _Policy.apply(*args)
    else:
        loss, stats, _, _ = _policy(*args, False)
    return PolicyLoss(loss, stats[0], stats[1])


class PreferenceLoss(NamedTuple):
    loss: torch.Tensor              # differentiable in the log-probabilities
    chosen_rewards: torch.Tensor    # [pairs], beta times the chosen rows' log ratios
    rejected_rewards: torch.Tensor


@functools.lru_cache(maxsize=1024)
def _preference_work(pairs, cols):
    return L.lib().advopt_preference_loss_work(pairs, cols)


def _preference(logprobs, ref, mask, beta, smoothing, average, keep):
    """(loss, rewards, slope, mask as it was read)."""
    R, C = logprobs.shape
    p, ld_p = rows_of(logprobs)
    ref, ld_ref = _rows(ref)
    mask, ld_mask = _rows(mask)
    new = lambda *shape, dtype=torch.float32: p.new_empty(shape, dtype=dtype)  # noqa: E731
    loss, rewards = new(), new(R)
    slope = new(R) if keep else None
    work = new(_preference_work(R // 2, C), dtype=torch.uint8)
    with on_device(p.device):
        rc = L.lib().advopt_preference_loss(_PREFERENCE.pack(
            loss.data_ptr(), rewards.data_ptr(), _ptr(slope), p.data_ptr(), _ptr(ref), _ptr(mask), work.data_ptr(), ld_p, ld_ref, ld_mask,
            R // 2, C, beta, smoothing, average, dtype_code(p.dtype)), raw_stream(p.device))
    if rc:
        L.check(rc, "advopt_preference_loss")
    return loss, rewards, slope


def _preference_backward(ctx, dloss, _):
    slope, *rest = ctx.saved_tensors
    (R, C), dev = ctx.x_shape, dloss.device
    slope = saved(slope, "rows' slopes", torch.float32, (R,), dev)
    mask, ld_mask = None, 0
    if rest:
        mask = rest[0]
        if mask.dtype is not torch.bool or mask.shape != ctx.x_shape or mask.device != dev:
            saved(mask, "mask", torch.bool, ctx.x_shape, dev)   # raises
        mask, ld_mask = rows_of(mask)
    dx = torch.empty((R, C), dtype=ctx.x_dtype, device=dev)
    with on_device(dev):
        rc = L.lib().advopt_preference_loss_grad(dx.data_ptr(), dloss.data_ptr(), slope.data_ptr(), _ptr(mask), ld_mask, R // 2, C,
                                                 dtype_code(ctx.x_dtype), raw_stream(dev))
    if rc:
        L.check(rc, "advopt_preference_loss_grad")
    return dx, *[None] * 5


_preference_backward_once = once_differentiable(_preference_backward)


class _Preference(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logprobs, ref, mask, beta, smoothing, average):
        loss, rewards, slope = _preference(logprobs, ref, mask, beta, smoothing, average, True)
        ctx.x_shape, ctx.x_dtype = logprobs.shape, logprobs.dtype
        ctx.save_for_backward(slope, *([] if mask is None else [mask]))
        ctx.mark_non_differentiable(rewards)
        ctx.set_materialize_grads(False)
        return loss, rewards

    @staticmethod
    def backward(ctx, dloss, drewards):
        # a second derivative is refused, without the wrapper's cost where none can be asked for
        return _preference_backward_once(ctx, dloss, drewards) if torch.is_grad_enabled() else _preference_backward(ctx, dloss, drewards)


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
    _check_rows("preference_loss", logprobs, dict(ref_logprobs=ref_logprobs), mask)
    R = logprobs.shape[0]
    if R == 0 or R % 2:
        raise ValueError(f"preference_loss: an even number of rows, the chosen and then the rejected sequences, got {R}")
    beta, label_smoothing = float(beta), float(label_smoothing)
    if not abs(beta) < 1e30:
        raise ValueError(f"preference_loss: beta must be finite, got {beta}")
    if not 0 <= label_smoothing <= 1:
        raise ValueError(f"preference_loss: label_smoothing is between 0 and 1, got {label_smoothing}")
    args = logprobs, ref_logprobs, mask, beta, label_smoothing, bool(average)
    if torch.is_grad_enabled() and logprobs.requires_grad:
        loss, rewards = _Preference.apply(*args)
    else:
        loss, rewards, _ = _preference(*args, False)
    return PreferenceLoss(loss, rewards[: R // 2], rewards[R // 2 :])
