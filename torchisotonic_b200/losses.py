"""Losses that a language model is trained on, in front of the calibration of its answers: token
log-probabilities, the preference loss over paired log ratios, and the clipped policy loss with a
KL term, each forward and backward in this library's kernels. The margins that a preference-trained
model gives held-out pairs are what ``fit_calibration`` turns into probabilities.

The reference has no such operators; the conventions are those of the rest of this package: CUDA
tensors only, float16 and bfloat16 computed in float32, float64 kept, rows packed with offsets.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor

from torchisotonic_b200 import _ext, ops


def _need_cuda(t: Tensor, name: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(
            "torchisotonic_b200 runs on CUDA tensors only (no CPU fallback); "
            f"move {name} to a CUDA device"
        )


def _as(t: Tensor, dtype: torch.dtype) -> Tensor:
    return t if t.dtype == dtype and t.is_contiguous() else t.to(dtype).contiguous()


def _check_logits(logits: Tensor, targets: Tensor, temperature: float) -> None:
    if not isinstance(logits, Tensor) or not isinstance(targets, Tensor):
        raise TypeError("logits and targets must be torch.Tensors")
    if not logits.is_floating_point() or logits.dtype not in _ext._DTYPES:
        raise TypeError("logits must be float16, bfloat16, float32 or float64")
    if targets.is_floating_point() or targets.is_complex() or targets.dtype == torch.bool:
        raise TypeError("targets must be an integer tensor")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError("logits must have a last dimension of at least one element")
    if targets.shape != logits.shape[:-1]:
        raise ValueError(f"targets of shape {tuple(targets.shape)} do not fit logits of shape "
                         f"{tuple(logits.shape)}")
    if not temperature > 0:
        raise ValueError("temperature must be > 0")
    _need_cuda(logits, "logits")
    if targets.device != logits.device:
        raise ValueError("targets must be on logits' device")


def token_logprobs(logits: Tensor, targets: Tensor, *, temperature: float = 1.0,
                   ignore_index: int = -100) -> Tensor:
    """Log-probability of one token per row: ``log softmax(logits / temperature)`` ([..., vocab],
    CUDA) at ``targets`` ([...], integers), without the softmax in memory. Returns ``targets``'
    shape in float32 (float64 for float64 logits). Differentiable in ``logits`` (once).

    Where a target is ``ignore_index`` the result and its gradient are 0 and the row of logits is
    not read; any other target outside ``[0, vocab)`` gives NaN. Logits may be -inf or the type's
    lowest value (a masked vocabulary); a row with nothing but -inf, or with NaN or +inf, gives NaN.
    A cut along the length (``logits[:, :-1]``) or a padded vocabulary (``logits[..., :v]``) is
    read in place; in the backward the cut's own gradient is torch's, which fills a tensor of the
    whole logits' size and copies this one's gradient into it.
    """
    traced = torch.compiler.is_compiling()
    settings = float(temperature), int(ignore_index)
    if not traced:
        got = _ext.native().token_logprobs(logits, targets, *settings)
        if got is not None:
            return got
    _check_logits(logits, targets, temperature)
    targets = _as(targets, torch.int64)
    if traced:  # the operators, which the compiler keeps whole
        return ops.token_logprobs(logits, targets, *settings)[0]
    return _ext.native().token_logprobs(logits, targets, *settings)


def preference_loss(
    logps: Tensor,
    ref_logps: Tensor | None,
    offsets: Tensor,
    *,
    beta: float = 0.1,
    kind: str = "logistic",
    label_smoothing: float = 0.0,
    margin: float = 0.0,
    mask: Tensor | None = None,
    average: bool = False,
) -> tuple[Tensor, Tensor]:
    """Preference loss over pairs of answers from their token log-probabilities.

    ``logps`` (and ``ref_logps``, the frozen reference's, or None for none): 1-D CUDA tensors of
    token log-probabilities (``token_logprobs``), the answers packed back to back; ``offsets``: 1-D
    integer tensor of ``2 pairs + 1`` non-decreasing positions on their device, answer k being
    ``logps[offsets[k]:offsets[k + 1]]``: first every pair's chosen answer, then every pair's
    rejected one. ``mask``: bool, which tokens count (a token that does not may hold anything).

    With ``s`` an answer's sum (``average=True``: its mean, 0 for an empty one) of ``logps -
    ref_logps``, and ``u = beta (s_chosen - s_rejected) - margin``, the loss is the mean over the
    pairs of, by ``kind``: "logistic" ``(1 - e) log(1 + exp(-u)) + e log(1 + exp(u))`` with ``e =
    label_smoothing``, "hinge" ``max(0, 1 - u)``, "square" ``(u - 1/2)^2 / beta^2``.

    Returns ``(loss, rewards)``: the scalar loss, differentiable (once) in ``logps`` and
    ``ref_logps``, and ``beta s`` of every answer, ``[2, pairs]`` (chosen, rejected), without
    gradient: ``rewards[0] - rewards[1]`` are the margins that a calibration curve is fitted on.
    float32 (float64 for float64 logps); sums are float64 in a fixed order.
    """
    traced = torch.compiler.is_compiling()
    settings = (_ext.PREFERENCE_KINDS.get(kind, -1), bool(average), float(beta),
                float(label_smoothing), float(margin))
    if not traced:
        got = _ext.native().preference_loss(logps, ref_logps, mask, offsets, *settings)
        if got is not None:
            return got
    if not isinstance(logps, Tensor) or not isinstance(offsets, Tensor):
        raise TypeError("logps and offsets must be torch.Tensors")
    if not logps.is_floating_point():
        raise TypeError("logps must be a floating-point tensor")
    if offsets.is_floating_point() or offsets.is_complex() or offsets.dtype == torch.bool:
        raise TypeError("offsets must be an integer tensor")
    if logps.dim() != 1:
        raise ValueError("logps must be 1-D")
    if offsets.dim() != 1 or offsets.numel() < 3 or offsets.numel() % 2 == 0:
        raise ValueError("offsets must be 1-D with 2 * pairs + 1 entries, pairs >= 1")
    if kind not in _ext.PREFERENCE_KINDS:
        raise ValueError(f"kind must be one of {', '.join(_ext.PREFERENCE_KINDS)}, got {kind!r}")
    if not beta > 0:
        raise ValueError("beta must be > 0")
    if not 0 <= label_smoothing < 0.5:
        raise ValueError("label_smoothing must be in [0, 0.5)")
    _need_cuda(logps, "logps")
    dev = logps.device
    dtype = torch.float64 if logps.dtype == torch.float64 else torch.float32
    if ref_logps is not None:
        if not isinstance(ref_logps, Tensor) or not ref_logps.is_floating_point():
            raise TypeError("ref_logps must be a floating-point torch.Tensor")
        if ref_logps.shape != logps.shape or ref_logps.device != dev:
            raise ValueError("ref_logps must be shaped like logps and on its device")
        ref_logps = _as(ref_logps, dtype)
    if mask is not None:
        if not isinstance(mask, Tensor) or mask.dtype != torch.bool:
            raise TypeError("mask must be a bool torch.Tensor")
        if mask.shape != logps.shape or mask.device != dev:
            raise ValueError("mask must be shaped like logps and on its device")
        mask = mask.contiguous()
    if offsets.device != dev:
        raise ValueError("offsets must be on logps' device")
    logps, offsets = _as(logps, dtype), _as(offsets, torch.int64)
    if traced:
        loss, rewards, _ = ops.preference(logps, ref_logps, mask, offsets, *settings)
        return loss, rewards.detach()
    return _ext.native().preference_loss(logps, ref_logps, mask, offsets, *settings)


class PolicyLoss(NamedTuple):
    """What ``policy_loss`` returns; only ``loss`` has a gradient."""

    loss: Tensor
    logps: Tensor
    kl: Tensor
    clip_fraction: Tensor


def policy_loss(
    logits: Tensor,
    targets: Tensor,
    old_logps: Tensor,
    advantages: Tensor,
    *,
    ref_logps: Tensor | None = None,
    weight: Tensor | None = None,
    clip_low: float = 0.2,
    clip_high: float = 0.2,
    kl_coef: float = 0.0,
    temperature: float = 1.0,
    ignore_index: int = -100,
) -> PolicyLoss:
    """Clipped policy loss with a KL term, from the policy's logits, with its gradient in one pass
    over them.

    For every token, ``lp`` its log-probability (``token_logprobs(logits, targets)``), ``rho =
    exp(lp - old_logps)`` and ``d = ref_logps - lp``: ``l = -min(rho A, clip(rho, 1 - clip_low, 1 +
    clip_high) A) + kl_coef (exp(d) - d - 1)``, A the advantage, the last term only with
    ``ref_logps``. The loss is ``sum(weight l) / sum(weight)`` (0 if the weights sum to 0).

    ``logits``: [..., vocab]; every other tensor has the targets' shape [...]. ``weight``: numbers,
    or a bool mask; None for 1. A token of weight 0 (or with target ``ignore_index``) is left out:
    nothing else of it is read, its gradient is 0. Where both sides of the minimum are equal the
    gradient is the unclipped side's. A ratio or a ``kl_coef`` term beyond the type's range is
    infinite; a factor of 0 (the advantage, ``kl_coef``) leaves its term out also there.

    The gradient is written with the loss, for an upstream gradient of exactly 1; any other one
    (``loss / n``, a scaled loss) takes another pass over the logits in the backward.

    Returns ``PolicyLoss(loss, logps, kl, clip_fraction)``: the loss, differentiable (once) in
    ``logits`` alone; the tokens' log-probabilities (0 where left out); the weighted means of
    ``exp(d) - d - 1`` and of where the clip holds. float32 (float64 for float64 logits).
    """
    traced = torch.compiler.is_compiling()
    rows = int(ignore_index), float(temperature)
    clip = float(clip_low), float(clip_high), float(kl_coef)
    if not traced:
        got = _ext.native().policy_loss(logits, targets, *rows, old_logps, advantages, ref_logps,
                                        weight, *clip)
        if got is not None:
            return PolicyLoss(*got)
    if not (clip_low >= 0 and clip_high >= 0):
        raise ValueError("clip_low and clip_high must not be negative")
    _check_logits(logits, targets, temperature)
    acc, shape, device = _ext.acc_dtype(logits.dtype), targets.shape, logits.device

    def constant(name: str, t: Tensor | None) -> Tensor:
        if not isinstance(t, Tensor) or t.is_complex():
            raise TypeError(f"{name} must be a real torch.Tensor")
        if t.shape != shape or t.device != device:
            raise ValueError(f"{name} must be shaped like targets and on logits' device")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} is a constant of the loss: detach it")
        return _as(t, torch.bool if name == "weight" and t.dtype == torch.bool else acc)

    old_logps = constant("old_logps", old_logps)
    advantages = constant("advantages", advantages)
    ref_logps = None if ref_logps is None else constant("ref_logps", ref_logps)
    weight = None if weight is None else constant("weight", weight)
    targets = _as(targets, torch.int64)
    constants = old_logps, advantages, ref_logps, weight
    if traced:
        out, logps, _ = ops.policy(logits, targets, *rows, *constants, *clip)
        rest = out.detach()
        return PolicyLoss(out[0], logps.detach(), rest[1], rest[2])
    return PolicyLoss(*_ext.native().policy_loss(logits, targets, *rows, *constants, *clip))
